// Norms of queries and keys for each head, with the position rotation in the same pass:
//     xhat = x / sqrt(mean(x^2) + eps)     y = R(position) (w * xhat)
// over the d columns of every head of q (weight wq) and of k (weight wk).  Backward, with g = R(-position) dy:
//     dw = sum over tokens and heads of g * xhat       dx = rstd (g w - xhat mean(g w xhat))
// x is read in the backward anyway and rstd is made anew from it, so that nothing but x is kept.  Memory bound: x in, y out; x and dy in, dx out.
// Sums of a head are over the lanes that have it, in 32 bits; dw is added up in 32 bits by every thread over its tokens, then over the CTA's threads and over the CTAs, in
// their order: the same bits in every run.  y, dx and dw are rounded once.
// 16384 tokens, 36 heads of 64, forward 27 to 29 us (5.2 to 5.7 of the 6.5 TB/s that a copy reaches), backward 42 to 45 (5.0 to 5.4), dw 5; 8192 tokens, 40 heads of 128 29 and 47.  Memory bounds them, with 55 % of the
// issue slots; 16 columns a lane instead of 8 take fewer instructions, but too many registers for enough loads on their way (41 and 60 us).
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

// A head is P2 lanes', 8 columns each (d / 8 of them, up to the next power of two, work); a warp takes 32 / P2 heads of q or of k at a time, a group, first those of q, then those of k: what differs
// between the two is decided outside of the loops.  AHEAD groups are on their way, and pointers are counted up: what bounds simpler forms is instructions, not memory (16384 tokens, 36 heads of
// 64: heads of q and k in one loop, strides multiplied out and numbers one at a time, 156 a group forward and 305 backward, 32 and 61 us).
// The first columns of a lane's four pairs are two pairs of numbers, the second ones two more: all but sums over lanes is done two numbers at a time.
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
__device__ __forceinline__ float dot(const Pairs& x, const Pairs& y) {
  float a, b;
  unpack2(add2(fma2(x.a[0], y.a[0], mul2(x.b[0], y.b[0])), fma2(x.a[1], y.a[1], mul2(x.b[1], y.b[1]))), a, b);
  return a + b;
}
// Angles of the lane's four pairs of a token; a position outside of the tables gives NaN, no access.
struct Angles { f32x2 c[2], s[2]; };
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
  return Angles{{pack2(c.x, c.y), pack2(c.z, c.w)}, {pack2(n.x, n.y), pack2(n.z, n.w)}};
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
// The lane's columns of the first group of a walk.
template <typename T>
__device__ __forceinline__ T* place(T* base, const NormRopeHeads& st, const Item& t, int head, int v) { return base + (t.b * st.b + t.s * st.s + head * st.h + v * 8); }

constexpr int THREADS = 256, WARPS = THREADS / 32;

template <int P2>
__global__ void __launch_bounds__(THREADS) qk_norm_rope_kernel(const __grid_constant__ NormRopeParams p) {
  grid_go();
  grid_wait();
  constexpr int G = Lanes<P2>::G, AHEAD = 4;
  const Lanes<P2> l(p.d);
  const int item = (int)blockIdx.x * WARPS + (int)(threadIdx.x >> 5);
  if (item >= p.items) return;
  const Item t = item_of(p, item);
  const float inv_d = 1.f / (float)p.d;
  Angles turn;
  // groups [lo, hi) of one tensor of `heads` heads
  auto walk = [&](const bf16* in, const NormRopeHeads& is, bf16* out, const NormRopeHeads& os, const bf16* weight, int heads, int lo, int hi, bool first) {
    if (lo >= hi) return;
    const bf16* from = place(in, is, t, lo * G + l.mine, l.v);
    bf16* to = place(out, os, t, lo * G + l.mine, l.v);
    const long long from_step = G * is.h, to_step = G * os.h;
    const int mine = l.works ? min(hi, (heads - l.mine + G - 1) / G) : 0;       // groups up to here have a head of the lane's
    uint4 x[AHEAD];
    auto load = [&](uint4& x, int g) {
      x = make_uint4(0, 0, 0, 0);
      if (g < mine) x = __ldcs(reinterpret_cast<const uint4*>(from));
      from += from_step;
    };
#pragma unroll
    for (int u = 0; u < AHEAD; u++) load(x[u], lo + u);
    const Pairs w = pairs_of(*reinterpret_cast<const uint4*>(weight + (l.works ? l.v * 8 : 0)));
    if (first) turn = angles(p, t.b, t.s, l.v, l.works);
    // a weight and an angle are one number: y = (w a) c - (w b) s, (w b) c + (w a) s
    f32x2 ac[2], as[2], bc[2], bs[2];
#pragma unroll
    for (int k = 0; k < 2; k++) {
      ac[k] = mul2(w.a[k], turn.c[k]);
      as[k] = mul2(w.a[k], turn.s[k]);
      bc[k] = mul2(w.b[k], turn.c[k]);
      bs[k] = mul2(w.b[k], turn.s[k]);
    }
    for (int g0 = lo; g0 < hi; g0 += AHEAD) {
#pragma unroll
      for (int u = 0; u < AHEAD; u++) {
        const int g = g0 + u;
        if (g >= hi) break;
        const Pairs f = pairs_of(x[u]);
        if (g0 + AHEAD < hi) load(x[u], g + AHEAD);
        const float rstd = rsqrtf(head_sum<P2>(dot(f, f)) * inv_d + p.eps);
        const f32x2 by = pack2(rstd, rstd);
        Pairs y;
#pragma unroll
        for (int k = 0; k < 2; k++) {
          y.a[k] = mul2(sub2(mul2(f.a[k], ac[k]), mul2(f.b[k], bs[k])), by);
          y.b[k] = mul2(fma2(f.b[k], bc[k], mul2(f.a[k], as[k])), by);
        }
        if (g < mine) *reinterpret_cast<uint4*>(to) = packed(y);
        to += to_step;
      }
    }
  };
  walk(p.q, p.qs, p.oq, p.oqs, p.wq, p.hq, t.g0, min(t.g1, p.of_q), true);
  walk(p.k, p.ks, p.ok, p.oks, p.wk, p.hkv, max(t.g0 - p.of_q, 0), t.g1 - p.of_q, t.g0 >= p.of_q);
}

// A warp walks over tokens.  A thread adds up its share of dw in registers over the heads of q or of k of a token, and over tokens in shared memory.
template <int P2>
__global__ void __launch_bounds__(THREADS, 3) qk_norm_rope_bwd_kernel(const __grid_constant__ NormRopeParams p) {
  grid_go();
  grid_wait();
  constexpr int G = Lanes<P2>::G, AHEAD = 2;
  __shared__ float2 kept[2][4][THREADS];
  const Lanes<P2> l(p.d);
  const float inv_d = 1.f / (float)p.d;
#pragma unroll
  for (int i = 0; i < 4; i++) kept[0][i][threadIdx.x] = kept[1][i][threadIdx.x] = make_float2(0.f, 0.f);
  // (the step goes past the end once, within 32 bits)
  for (unsigned item = blockIdx.x * WARPS + (threadIdx.x >> 5); item < (unsigned)p.items; item += gridDim.x * WARPS) {
    const Item t = item_of(p, (int)item);
    Angles turn;
    auto walk = [&](const bf16* in, const NormRopeHeads& is, const bf16* dy, const NormRopeHeads& ds, bf16* out, const NormRopeHeads& os, const bf16* weight, int heads, int lo, int hi, bool first,
                    float2 (*sums)[THREADS]) {
      if (lo >= hi) return;
      const bf16 *from = place(in, is, t, lo * G + l.mine, l.v), *from_dy = place(dy, ds, t, lo * G + l.mine, l.v);
      bf16* to = place(out, os, t, lo * G + l.mine, l.v);
      const int mine = l.works ? min(hi, (heads - l.mine + G - 1) / G) : 0;
      uint4 x[AHEAD], y[AHEAD];
      auto load = [&](uint4& x, uint4& y, int g) {
        x = y = make_uint4(0, 0, 0, 0);
        if (g < mine) {
          x = __ldcs(reinterpret_cast<const uint4*>(from));
          y = __ldcs(reinterpret_cast<const uint4*>(from_dy));
        }
        from += G * is.h;
        from_dy += G * ds.h;
      };
#pragma unroll
      for (int u = 0; u < AHEAD; u++) load(x[u], y[u], lo + u);
      const Pairs w = pairs_of(*reinterpret_cast<const uint4*>(weight + (l.works ? l.v * 8 : 0)));
      if (first) turn = angles(p, t.b, t.s, l.v, l.works);
      Pairs sum;
#pragma unroll
      for (int k = 0; k < 2; k++) sum.a[k] = sum.b[k] = 0;
      for (int g0 = lo; g0 < hi; g0 += AHEAD) {
#pragma unroll
        for (int u = 0; u < AHEAD; u++) {
          const int g = g0 + u;
          if (g >= hi) break;
          Pairs f = pairs_of(x[u]), gx;
          const Pairs r = pairs_of(y[u]);
          if (g0 + AHEAD < hi) load(x[u], y[u], g + AHEAD);
          const float ss = head_sum<P2>(dot(f, f));
          // (0 where the lane has no head, of which there would be NaN with an eps of zero)
          const float rstd = g < mine ? rsqrtf(ss * inv_d + p.eps) : 0.f;
          const f32x2 by = pack2(rstd, rstd);
#pragma unroll
          for (int k = 0; k < 2; k++) {
            f.a[k] = mul2(f.a[k], by);             // xhat
            f.b[k] = mul2(f.b[k], by);
            gx.a[k] = fma2(r.a[k], turn.c[k], mul2(r.b[k], turn.s[k]));        // dy turned back
            gx.b[k] = sub2(mul2(r.b[k], turn.c[k]), mul2(r.a[k], turn.s[k]));
            sum.a[k] = fma2(gx.a[k], f.a[k], sum.a[k]);
            sum.b[k] = fma2(gx.b[k], f.b[k], sum.b[k]);
            gx.a[k] = mul2(gx.a[k], w.a[k]);
            gx.b[k] = mul2(gx.b[k], w.b[k]);
          }
          const float mean = head_sum<P2>(dot(gx, f)) * inv_d;
          const f32x2 off = pack2(-mean, -mean);
#pragma unroll
          for (int k = 0; k < 2; k++) {
            gx.a[k] = mul2(fma2(f.a[k], off, gx.a[k]), by);
            gx.b[k] = mul2(fma2(f.b[k], off, gx.b[k]), by);
          }
          if (g < mine) *reinterpret_cast<uint4*>(to) = packed(gx);
          to += G * os.h;
        }
      }
      if (!p.partial) return;
#pragma unroll
      for (int k = 0; k < 4; k++) {
        float a, b;
        unpack2(k < 2 ? sum.a[k] : sum.b[k - 2], a, b);
        const float2 old = sums[k][threadIdx.x];
        sums[k][threadIdx.x] = make_float2(old.x + a, old.y + b);
      }
    };
    walk(p.q, p.qs, p.dq, p.dqs, p.oq, p.oqs, p.wq, p.hq, t.g0, min(t.g1, p.of_q), true, kept[0]);
    walk(p.k, p.ks, p.dk, p.dks, p.ok, p.oks, p.wk, p.hkv, max(t.g0 - p.of_q, 0), t.g1 - p.of_q, t.g0 >= p.of_q, kept[1]);
  }
  if (!p.partial) return;
  // over the heads of a group and the warps: a column is that of the same lane and place in all of them
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * p.d; i += THREADS) {
    const int of = i / p.d, c = i - of * p.d, pair = (c & 7) >> 1, k = (c & 1) * 2 + (pair >> 1);
    float total = 0.f;
    for (int j = c / 8; j < THREADS; j += P2) {
      const float2 s = kept[of][k][j];
      total += pair & 1 ? s.y : s.x;
    }
    p.partial[(long long)blockIdx.x * 2 * p.d + i] = total;
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
// Groups of a token, and of a warp: all of a token's, or fewer where there are few tokens: two at least, eight warps per SM.
int groups_of(int hq, int hkv, int d) {
  const int G = 32 / padded(d);
  return (hq + G - 1) / G + (hkv + G - 1) / G;
}
int share_of(long long tokens, int groups) {
  const int most = (groups + 1) / 2;
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
  const long long want = (items_of(tokens, groups, share_of(tokens, groups)) + WARPS - 1) / WARPS, most = 3LL * lb_num_sms();      // as many as are resident
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
