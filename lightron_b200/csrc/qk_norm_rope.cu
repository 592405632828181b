// Norms of queries and keys for each head, with the position rotation in the same pass:
//     xhat = x / sqrt(mean(x^2) + eps)     y = R(position) (w * xhat)
// over the d columns of every head of q (weight wq) and of k (weight wk).  Backward, with g = R(-position) dy:
//     dw = sum over tokens and heads of g * xhat       dx = rstd (g w - xhat mean(g w xhat))
// x is read in the backward anyway and rstd is made anew from it, so that nothing but x is kept.  Memory bound: x in, y out; x and dy in, dx out.
// Sums of a head are over the lanes that have it, in 32 bits; dw is added up in 32 bits by every thread over its tokens, then over the CTA's threads and over the CTAs, in
// their order: the same bits in every run.  y, dx and dw are rounded once.
#include "tcgen05.cuh"

namespace {
using namespace bw;

constexpr int MAX_AXES = 8, MAX_PAIRS = 128;

struct NormRopeHeads { long long b, s, h; };      // strides in elements; the columns of a head are contiguous
struct NormRopeParams {
  const bf16 *q, *k, *wq, *wk;
  bf16 *oq, *ok;                 // y, or dx
  const bf16 *dq, *dk;           // backward: dy
  NormRopeHeads qs, ks, oqs, oks, dqs, dks;
  const float *cosT, *sinT;
  const int* positions;          // null: a token's place in its sequence; else axis a of token (b, s) at a * pos_a + b * pos_b + s
  long long pos_a, pos_b;
  float* partial;                // backward, null or [CTAs][2][d]
  int B, S, hq, hkv, d, rows;
  float eps;
  int of_q, groups, share, items;      // groups of q, of a token, of a warp; warps' shares of all tokens
  FastDiv by_parts, by_S;
  int plain;                     // one axis, and tables on 16 bytes: a lane's angles are two vectors
  unsigned char axis[MAX_PAIRS];
};

// A head is P2 lanes', 8 columns each (d / 8 of them, up to the next power of two, work); a warp takes 32 / P2 heads of q or of k at a time, a group: what is decided for a group is decided
// for the warp.  Two groups make a round, and the next round (of the next token, behind a token's last) is on its way while one is worked on.
// The first columns of a lane's four pairs are two pairs of numbers, the second ones two more: everything but sums over lanes is done two numbers at a time.  (One at a time the
// backward took 305 instructions a group and was bound by them: 16384 tokens, 36 heads of 64 61 us.)
template <int P2>
struct Lanes {
  static constexpr int G = 32 / P2;
  int mine, v;                   // which of the G heads, which vector of it
  bool works;
  __device__ Lanes(int d) {
    const int lane = threadIdx.x & 31;
    mine = lane / P2;
    v = lane % P2;
    works = v * 8 < d;
  }
};
template <int P2>
__device__ __forceinline__ float head_sum(float x) {
#pragma unroll
  for (int o = P2 / 2; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

struct Pairs { f32x2 a[2], b[2]; };      // first and second columns of four pairs
__device__ __forceinline__ Pairs pairs_of(const uint4& u) {
  auto lo = [](uint32_t w) { return __uint_as_float(w << 16); };
  auto hi = [](uint32_t w) { return __uint_as_float(w & 0xffff0000u); };
  return Pairs{{pack2(lo(u.x), lo(u.y)), pack2(lo(u.z), lo(u.w))}, {pack2(hi(u.x), hi(u.y)), pack2(hi(u.z), hi(u.w))}};
}
__device__ __forceinline__ uint4 packed(const Pairs& p) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 2; i++) {
    float a0, a1, b0, b1;
    unpack2(p.a[i], a0, a1);
    unpack2(p.b[i], b0, b1);
    const bf162 x = __floats2bfloat162_rn(a0, b0), y = __floats2bfloat162_rn(a1, b1);
    w[2 * i] = *reinterpret_cast<const uint32_t*>(&x);
    w[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&y);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ Pairs times(const Pairs& x, const Pairs& y) { return Pairs{{mul2(x.a[0], y.a[0]), mul2(x.a[1], y.a[1])}, {mul2(x.b[0], y.b[0]), mul2(x.b[1], y.b[1])}}; }
__device__ __forceinline__ Pairs times(const Pairs& x, float y) {
  const f32x2 t = pack2(y, y);
  return Pairs{{mul2(x.a[0], t), mul2(x.a[1], t)}, {mul2(x.b[0], t), mul2(x.b[1], t)}};
}
__device__ __forceinline__ Pairs plus(const Pairs& x, const Pairs& y, const Pairs& z) {      // x y + z
  return Pairs{{fma2(x.a[0], y.a[0], z.a[0]), fma2(x.a[1], y.a[1], z.a[1])}, {fma2(x.b[0], y.b[0], z.b[0]), fma2(x.b[1], y.b[1], z.b[1])}};
}
__device__ __forceinline__ float dot(const Pairs& x, const Pairs& y) {
  float a, b;
  unpack2(add2(fma2(x.a[0], y.a[0], mul2(x.b[0], y.b[0])), fma2(x.a[1], y.a[1], mul2(x.b[1], y.b[1]))), a, b);
  return a + b;
}
// Turned by the angles, whose sines are in minus with the other sign; back: the two in each other's place.
struct Angles { f32x2 c[2], s[2], minus[2]; };
__device__ __forceinline__ Pairs turned(const Pairs& x, const Angles& t, bool back) {
  Pairs y;
#pragma unroll
  for (int i = 0; i < 2; i++) {
    y.a[i] = fma2(x.a[i], t.c[i], mul2(x.b[i], back ? t.s[i] : t.minus[i]));
    y.b[i] = fma2(x.b[i], t.c[i], mul2(x.a[i], back ? t.minus[i] : t.s[i]));
  }
  return y;
}
// Of the lane's four pairs of a token; a position outside of the tables gives NaN, no access.
__device__ __forceinline__ Angles angles(const NormRopeParams& p, int b, int s, int v, bool works) {
  float4 c, n;
  if (p.plain) {
    const int pos = p.positions ? p.positions[b * p.pos_b + s] : s;
    c = n = make_float4(__int_as_float(0x7fffffff), __int_as_float(0x7fffffff), __int_as_float(0x7fffffff), __int_as_float(0x7fffffff));
    if ((unsigned)pos < (unsigned)p.rows) {
      const long long at = (long long)pos * (p.d >> 1) + (works ? v * 4 : 0);
      c = *reinterpret_cast<const float4*>(p.cosT + at);
      n = *reinterpret_cast<const float4*>(p.sinT + at);
    }
  } else {
    float cs[8];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int pair = works ? v * 4 + i : 0;
      const int pos = p.positions ? p.positions[p.axis[pair] * p.pos_a + b * p.pos_b + s] : s;
      const bool there = (unsigned)pos < (unsigned)p.rows;
      const long long at = (long long)pos * (p.d >> 1) + pair;
      cs[i] = there ? p.cosT[at] : __int_as_float(0x7fffffff);
      cs[4 + i] = there ? p.sinT[at] : __int_as_float(0x7fffffff);
    }
    c = make_float4(cs[0], cs[1], cs[2], cs[3]);
    n = make_float4(cs[4], cs[5], cs[6], cs[7]);
  }
  return Angles{{pack2(c.x, c.y), pack2(c.z, c.w)}, {pack2(n.x, n.y), pack2(n.z, n.w)}, {pack2(-n.x, -n.y), pack2(-n.z, -n.w)}};
}

// Groups [g0, g1) of a token: those of q, then those of k.
struct Item { int b, s, g0, g1; };
__device__ __forceinline__ Item item_of(const NormRopeParams& p, int i) {
  Item t;
  const int tok = p.by_parts.div(i), part = i - tok * (int)p.by_parts.d;
  t.b = p.by_S.div(tok);
  t.s = tok - t.b * p.S;
  t.g0 = part * p.share;
  t.g1 = min(p.groups, t.g0 + p.share);
  return t;
}
// Where the lane's vectors of a token lie in one tensor of queries and one of keys.
template <typename T>
struct Places {
  T *q, *k;
  __device__ Places(T* of_q, T* of_k, const NormRopeHeads& qs, const NormRopeHeads& ks, const Item& t, int mine, int v)
      : q(of_q + t.b * qs.b + t.s * qs.s + mine * qs.h + v * 8), k(of_k + t.b * ks.b + t.s * ks.s + mine * ks.h + v * 8) {}
  template <int G>
  __device__ T* at(bool is_q, int g, const NormRopeHeads& qs, const NormRopeHeads& ks) const { return is_q ? q + g * (G * qs.h) : k + g * (G * ks.h); }
};

constexpr int THREADS = 256, WARPS = THREADS / 32, ROUND = 2;

template <int P2>
__global__ void __launch_bounds__(THREADS) qk_norm_rope_kernel(const __grid_constant__ NormRopeParams p) {
  grid_go();
  grid_wait();
  const Lanes<P2> l(p.d);
  constexpr int G = Lanes<P2>::G;
  const int item = (int)blockIdx.x * WARPS + (int)(threadIdx.x >> 5);
  if (item >= p.items) return;
  const Item t = item_of(p, item);
  // groups where the lane has a head
  const int nq = l.works ? (p.hq - l.mine + G - 1) / G : 0, nk = l.works ? (p.hkv - l.mine + G - 1) / G : 0;
  const Places<const bf16> in(p.q, p.k, p.qs, p.ks, t, l.mine, l.v);
  const Places<bf16> out(p.oq, p.ok, p.oqs, p.oks, t, l.mine, l.v);
  auto load = [&](uint4* x, int g0) {
#pragma unroll
    for (int i = 0; i < ROUND; i++) {
      const bool is_q = g0 + i < p.of_q;
      const int g = is_q ? g0 + i : g0 + i - p.of_q;
      x[i] = make_uint4(0, 0, 0, 0);
      if (g0 + i < t.g1 && g < (is_q ? nq : nk)) x[i] = __ldcs(reinterpret_cast<const uint4*>(in.at<G>(is_q, g, p.qs, p.ks)));
    }
  };
  uint4 x[ROUND], next[ROUND];
  load(x, t.g0);
  const int col = l.works ? l.v * 8 : 0;
  const uint4 wq = *reinterpret_cast<const uint4*>(p.wq + col), wk = *reinterpret_cast<const uint4*>(p.wk + col);
  const Angles turn = angles(p, t.b, t.s, l.v, l.works);
  const float inv_d = 1.f / (float)p.d;
  for (int g0 = t.g0; g0 < t.g1; g0 += ROUND) {
    if (g0 + ROUND < t.g1) load(next, g0 + ROUND);
#pragma unroll
    for (int i = 0; i < ROUND; i++) {
      if (g0 + i >= t.g1) break;
      const bool is_q = g0 + i < p.of_q;
      const int g = is_q ? g0 + i : g0 + i - p.of_q;
      const Pairs f = pairs_of(x[i]);
      const float rstd = rsqrtf(head_sum<P2>(dot(f, f)) * inv_d + p.eps);
      const Pairs y = turned(times(times(f, rstd), pairs_of(is_q ? wq : wk)), turn, false);
      if (g < (is_q ? nq : nk)) *reinterpret_cast<uint4*>(out.at<G>(is_q, g, p.oqs, p.oks)) = packed(y);
    }
#pragma unroll
    for (int i = 0; i < ROUND; i++) x[i] = next[i];
  }
}

// A warp walks over tokens; every thread keeps its share of dw.
template <int P2>
__global__ void __launch_bounds__(THREADS, 2) qk_norm_rope_bwd_kernel(const __grid_constant__ NormRopeParams p) {
  grid_go();
  grid_wait();
  const Lanes<P2> l(p.d);
  constexpr int G = Lanes<P2>::G;
  const int step = (int)gridDim.x * WARPS;
  const float inv_d = 1.f / (float)p.d;
  const int col = l.works ? l.v * 8 : 0;
  const uint4 wq = *reinterpret_cast<const uint4*>(p.wq + col), wk = *reinterpret_cast<const uint4*>(p.wk + col);
  const int nq = l.works ? (p.hq - l.mine + G - 1) / G : 0, nk = l.works ? (p.hkv - l.mine + G - 1) / G : 0;
  Pairs aq, ak;
#pragma unroll
  for (int i = 0; i < 2; i++) aq.a[i] = aq.b[i] = ak.a[i] = ak.b[i] = 0;
  auto load = [&](uint4* x, uint4* y, const Item& t, int g0) {
    const Places<const bf16> in(p.q, p.k, p.qs, p.ks, t, l.mine, l.v), dy(p.dq, p.dk, p.dqs, p.dks, t, l.mine, l.v);
#pragma unroll
    for (int i = 0; i < ROUND; i++) {
      const bool is_q = g0 + i < p.of_q;
      const int g = is_q ? g0 + i : g0 + i - p.of_q;
      x[i] = y[i] = make_uint4(0, 0, 0, 0);
      if (g0 + i < t.g1 && g < (is_q ? nq : nk)) {
        x[i] = __ldcs(reinterpret_cast<const uint4*>(in.at<G>(is_q, g, p.qs, p.ks)));
        y[i] = __ldcs(reinterpret_cast<const uint4*>(dy.at<G>(is_q, g, p.dqs, p.dks)));
      }
    }
  };
  // (32 bits of an item: the step goes past the end at most once)
  unsigned item = blockIdx.x * WARPS + (threadIdx.x >> 5);
  uint4 x[ROUND], y[ROUND];
  Angles turn;
  Item t;
  if (item < (unsigned)p.items) {
    t = item_of(p, (int)item);
    load(x, y, t, t.g0);
    turn = angles(p, t.b, t.s, l.v, l.works);
  }
  while (item < (unsigned)p.items) {
    const bool more = item + step < (unsigned)p.items;
    const Item then = more ? item_of(p, (int)(item + step)) : t;
    const Places<bf16> out(p.oq, p.ok, p.oqs, p.oks, t, l.mine, l.v);
    for (int g0 = t.g0; g0 < t.g1; g0 += ROUND) {
      uint4 nx[ROUND], ny[ROUND];
      if (g0 + ROUND < t.g1) load(nx, ny, t, g0 + ROUND);
      else if (more) load(nx, ny, then, then.g0);
#pragma unroll
      for (int i = 0; i < ROUND; i++) {
        if (g0 + i >= t.g1) break;
        const bool is_q = g0 + i < p.of_q;
        const int g = is_q ? g0 + i : g0 + i - p.of_q;
        const bool in = g < (is_q ? nq : nk);
        Pairs f = pairs_of(x[i]);
        const float ss = head_sum<P2>(dot(f, f));
        // (0 where the lane has no head, of which there would be NaN with an eps of zero)
        const float rstd = in ? rsqrtf(ss * inv_d + p.eps) : 0.f;
        f = times(f, rstd);                                                    // xhat
        Pairs gx = turned(pairs_of(y[i]), turn, true);
        if (is_q) aq = plus(gx, f, aq); else ak = plus(gx, f, ak);
        gx = times(gx, pairs_of(is_q ? wq : wk));
        const float mean = head_sum<P2>(dot(gx, f)) * inv_d;
        const f32x2 off = pack2(-mean, -mean);
        gx = times(Pairs{{fma2(f.a[0], off, gx.a[0]), fma2(f.a[1], off, gx.a[1])}, {fma2(f.b[0], off, gx.b[0]), fma2(f.b[1], off, gx.b[1])}}, rstd);
        if (in) *reinterpret_cast<uint4*>(out.at<G>(is_q, g, p.oqs, p.oks)) = packed(gx);
      }
#pragma unroll
      for (int i = 0; i < ROUND; i++) { x[i] = nx[i]; y[i] = ny[i]; }
    }
    if (more) turn = angles(p, then.b, then.s, l.v, l.works);
    t = then;
    item += step;
  }
  if (!p.partial) return;
  // over the heads of a warp, then over the warps of the CTA
  __shared__ float sums[2][WARPS][P2 * 8];
#pragma unroll
  for (int of = 0; of < 2; of++) {
    const Pairs& from = of ? ak : aq;
    float c[8];
#pragma unroll
    for (int i = 0; i < 2; i++) {
      unpack2(from.a[i], c[4 * i], c[4 * i + 2]);
      unpack2(from.b[i], c[4 * i + 1], c[4 * i + 3]);
    }
#pragma unroll
    for (int j = 0; j < 8; j++) {
#pragma unroll
      for (int o = P2; o < 32; o <<= 1) c[j] += __shfl_xor_sync(0xffffffffu, c[j], o);
      if (l.mine == 0) sums[of][threadIdx.x >> 5][l.v * 8 + j] = c[j];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * p.d; i += THREADS) {
    const int of = i / p.d, c = i - of * p.d;
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; w++) t += sums[of][w][c];
    p.partial[(long long)blockIdx.x * 2 * p.d + i] = t;
  }
}

// dw = the sum of the CTAs' parts: 32 columns x 32 row lanes a block
__global__ void __launch_bounds__(1024) qk_norm_rope_dw_kernel(const float* __restrict__ partial, bf16* __restrict__ dwq, bf16* __restrict__ dwk, int ctas, int d) {
  grid_go();
  grid_wait();
  __shared__ float s[32][33];
  const int i = blockIdx.x * 32 + threadIdx.x;
  float v = 0.f;
  if (i < 2 * d)
    for (int c = threadIdx.y; c < ctas; c += 32) v += partial[(long long)c * 2 * d + i];
  s[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  v = warp_sum(s[threadIdx.x][threadIdx.y]);        // (a column is a warp's)
  const int c = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && c < 2 * d) (c < d ? dwq[c] : dwk[c - d]) = __float2bfloat16(v);
}

int padded(int d) {
  int p2 = 1;
  while (p2 * 8 < d) p2 *= 2;
  return p2;
}
// Groups of a token, and of a warp: all of a token's, or fewer where there are few tokens: one round of loads each at least, eight warps per SM.
int groups_of(int hq, int hkv, int d) {
  const int G = 32 / padded(d);
  return (hq + G - 1) / G + (hkv + G - 1) / G;
}
int share_of(long long tokens, int groups) {
  const int most = (groups + ROUND - 1) / ROUND;
  const long long want = (8LL * lb_num_sms() + tokens - 1) / tokens;
  const int parts = (int)(want < most ? want : most);
  return (groups + parts - 1) / parts;
}
long long items_of(long long tokens, int groups, int share) { return tokens * ((groups + share - 1) / share); }
int set_items(NormRopeParams& p) {
  const long long tokens = (long long)p.B * p.S;
  const int G = 32 / padded(p.d);
  p.of_q = (p.hq + G - 1) / G;
  p.groups = groups_of(p.hq, p.hkv, p.d);
  p.share = share_of(tokens, p.groups);
  if (items_of(tokens, p.groups, p.share) > 0x7fffffffLL) return LB_ERR_SHAPE;
  p.items = (int)items_of(tokens, p.groups, p.share);
  p.by_parts.set((unsigned)((p.groups + p.share - 1) / p.share));
  p.by_S.set((unsigned)p.S);
  return LB_OK;
}

bool bad(const NormRopeHeads& s) { return (s.b | s.s | s.h) % 8 != 0; }
NormRopeHeads heads_at(const long long* s) { return NormRopeHeads{s[0], s[1], s[2]}; }

int fill(NormRopeParams& p, const void* q, const void* k, const void* wq, const void* wk, const void* cosT, const void* sinT, const void* positions, const unsigned char* axes, int n_axes, int B,
         int S, int hq, int hkv, int d, int rows, long long pos_a, long long pos_b, float eps) {
  if (B <= 0 || S <= 0 || hq <= 0 || hkv <= 0 || rows <= 0 || d <= 0 || d % 8 || d > 2 * MAX_PAIRS || n_axes <= 0 || n_axes > MAX_AXES || (long long)hq + hkv > 0x3fffffff) return LB_ERR_SHAPE;
  if (!q || !k || !wq || !wk || !cosT || !sinT || !axes || !(eps >= 0.f && eps < INFINITY) || ((uintptr_t)q | (uintptr_t)k | (uintptr_t)wq | (uintptr_t)wk) & 15) return LB_ERR_ARG;
  p.q = (const bf16*)q; p.k = (const bf16*)k; p.wq = (const bf16*)wq; p.wk = (const bf16*)wk;
  p.cosT = (const float*)cosT; p.sinT = (const float*)sinT; p.positions = (const int*)positions;
  p.pos_a = pos_a; p.pos_b = pos_b;
  p.B = B; p.S = S; p.hq = hq; p.hkv = hkv; p.d = d; p.rows = rows; p.eps = eps;
  for (int i = 0; i < d / 2; i++) {
    if (axes[i] >= n_axes) return LB_ERR_ARG;
    p.axis[i] = axes[i];
  }
  p.plain = (((uintptr_t)cosT | (uintptr_t)sinT) & 15) == 0;
  for (int i = 0; i < d / 2; i++) p.plain &= axes[i] == 0;
  return LB_OK;
}

#define LB_BY_LANES(d, CALL)                                                       \
  switch (padded(d)) {                                                             \
    case 1: CALL(1); break;                                                        \
    case 2: CALL(2); break;                                                        \
    case 4: CALL(4); break;                                                        \
    case 8: CALL(8); break;                                                        \
    case 16: CALL(16); break;                                                      \
    default: CALL(32); break;                                                      \
  }

}  // namespace

// yq, yk = q [B, S, hq, d], k [B, S, hkv, d] normed and turned.  strides: 4 x {batch, token, head} of q, k, yq, yk in elements, multiples of 8, innermost contiguous; wq, wk [d] bf16, 16-byte aligned;
// cos, sin fp32 [rows, d / 2]; positions null or int32, axis a of token (b, s) at a * pos_a + b * pos_b + s; axes: host bytes, the axis of each of the d / 2 pairs.
extern "C" int lb_qk_norm_rope(const void* q, const void* k, void* yq, void* yk, const void* wq, const void* wk, const void* cosT, const void* sinT, const void* positions,
                               const unsigned char* axes, int n_axes, int B, int S, int hq, int hkv, int d, int rows, const long long* strides, long long pos_a, long long pos_b, float eps,
                               void* stream) {
  NormRopeParams p{};
  if (const int rc = fill(p, q, k, wq, wk, cosT, sinT, positions, axes, n_axes, B, S, hq, hkv, d, rows, pos_a, pos_b, eps)) return rc;
  if (!yq || !yk || !strides || ((uintptr_t)yq | (uintptr_t)yk) & 15) return LB_ERR_ARG;
  p.oq = (bf16*)yq; p.ok = (bf16*)yk;
  p.qs = heads_at(strides); p.ks = heads_at(strides + 3); p.oqs = heads_at(strides + 6); p.oks = heads_at(strides + 9);
  if (bad(p.qs) || bad(p.ks) || bad(p.oqs) || bad(p.oks)) return LB_ERR_SHAPE;
  if (const int rc = set_items(p)) return rc;
#define LB_CALL(P) LB_LAUNCH(qk_norm_rope_kernel<P>, (p.items + WARPS - 1) / WARPS, THREADS, 0, (cudaStream_t)stream, p)
  LB_BY_LANES(d, LB_CALL)
#undef LB_CALL
  return LB_OK;
}

// CTAs of the backward: its `partial` has 2 * d floats for each.
extern "C" int lb_qk_norm_rope_bwd_ctas(int B, int S, int hq, int hkv, int d) {
  if (B <= 0 || S <= 0 || hq <= 0 || hkv <= 0 || d <= 0 || d % 8 || d > 2 * MAX_PAIRS || (long long)hq + hkv > 0x3fffffff) return 0;
  const long long tokens = (long long)B * S;
  const int groups = groups_of(hq, hkv, d);
  const long long want = (items_of(tokens, groups, share_of(tokens, groups)) + WARPS - 1) / WARPS, most = 2LL * lb_num_sms();
  return (int)(want < most ? want : most);
}

// dxq, dxk from dyq, dyk; with dwq and dwk [d] bf16 and `partial` (lb_qk_norm_rope_bwd_ctas() * 2 * d floats, not initialised), or without (all null).  strides: 6 x of q, k, dyq, dyk, dxq, dxk; a dx
// may be its dy.  The rest as in the forward.
extern "C" int lb_qk_norm_rope_bwd(const void* q, const void* k, const void* dyq, const void* dyk, void* dxq, void* dxk, const void* wq, const void* wk, const void* cosT, const void* sinT,
                                   const void* positions, const unsigned char* axes, int n_axes, void* partial, int ctas, void* dwq, void* dwk, int B, int S, int hq, int hkv, int d, int rows,
                                   const long long* strides, long long pos_a, long long pos_b, float eps, void* stream) {
  NormRopeParams p{};
  if (const int rc = fill(p, q, k, wq, wk, cosT, sinT, positions, axes, n_axes, B, S, hq, hkv, d, rows, pos_a, pos_b, eps)) return rc;
  if (!dyq || !dyk || !dxq || !dxk || !strides || ((uintptr_t)dyq | (uintptr_t)dyk | (uintptr_t)dxq | (uintptr_t)dxk) & 15 || (!partial) != (!dwq) || (!partial) != (!dwk)) return LB_ERR_ARG;
  if (ctas != lb_qk_norm_rope_bwd_ctas(B, S, hq, hkv, d)) return LB_ERR_ARG;
  p.dq = (const bf16*)dyq; p.dk = (const bf16*)dyk; p.oq = (bf16*)dxq; p.ok = (bf16*)dxk; p.partial = (float*)partial;
  p.qs = heads_at(strides); p.ks = heads_at(strides + 3); p.dqs = heads_at(strides + 6); p.dks = heads_at(strides + 9); p.oqs = heads_at(strides + 12); p.oks = heads_at(strides + 15);
  if (bad(p.qs) || bad(p.ks) || bad(p.dqs) || bad(p.dks) || bad(p.oqs) || bad(p.oks)) return LB_ERR_SHAPE;
  if (const int rc = set_items(p)) return rc;
#define LB_CALL(P) LB_LAUNCH(qk_norm_rope_bwd_kernel<P>, ctas, THREADS, 0, (cudaStream_t)stream, p)
  LB_BY_LANES(d, LB_CALL)
#undef LB_CALL
  if (partial) LB_LAUNCH(qk_norm_rope_dw_kernel, (2 * d + 31) / 32, dim3(32, 32), 0, (cudaStream_t)stream, (const float*)partial, (bf16*)dwq, (bf16*)dwk, ctas, d);
  return LB_OK;
}
