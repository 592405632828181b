// Norms of queries and keys for each head, with the position rotation in the same pass:
//     xhat = x / sqrt(mean(x^2) + eps)     y = R(position) (w * xhat)
// over the d columns of every head of q (weight wq) and of k (weight wk).  Backward, with g = R(-position) dy:
//     dw = sum over tokens and heads of g * xhat       dx = rstd (g w - xhat mean(g w xhat))
// x is read in the backward anyway and rstd is made anew from it, so that nothing but x is kept.  Memory bound: x in, y out; x and dy in, dx out.
// Sums of a head are over the lanes that have it, in 32 bits; dw is added up in 32 bits by every thread over its tokens, then over the CTA's threads and over the CTAs, in
// their order: the same bits in every run.  y, dx and dw are rounded once.
#include "common.cuh"

namespace {

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
  int B, S, hq, hkv, d, rows, share;
  float eps;
  unsigned char axis[MAX_PAIRS];
};

// A head is P2 lanes', 8 columns each (d / 8 of them, up to the next power of two, work); a warp takes 32 / P2 heads of a token at a time, ROUND loads of each lane in flight.
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

// Cosines and sines of the lane's four pairs of a token; a position outside of the tables gives NaN, no access.
__device__ __forceinline__ void angles(const NormRopeParams& p, int b, int s, int v, bool works, float* cs) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int pair = works ? v * 4 + i : 0;
    const int pos = p.positions ? p.positions[p.axis[pair] * p.pos_a + b * p.pos_b + s] : s;
    const bool there = (unsigned)pos < (unsigned)p.rows;
    const long long at = (long long)pos * (p.d >> 1) + pair;
    cs[i] = there ? p.cosT[at] : __int_as_float(0x7fffffff);
    cs[4 + i] = there ? p.sinT[at] : __int_as_float(0x7fffffff);
  }
}

constexpr int ROUND = 4;

template <int P2>
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(const __grid_constant__ NormRopeParams p) {
  grid_go();
  grid_wait();
  const Lanes<P2> l(p.d);
  constexpr int G = Lanes<P2>::G;
  const long long tok = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (tok >= (long long)p.B * p.S) return;
  const int b = (int)(tok / p.S), s = (int)(tok - (long long)b * p.S), heads = p.hq + p.hkv;
  const int h0 = (int)blockIdx.y * p.share, h1 = min(heads, h0 + p.share);
  const bf16 *q = p.q + b * p.qs.b + s * p.qs.s + l.v * 8, *k = p.k + b * p.ks.b + s * p.ks.s + l.v * 8;
  uint4 a[ROUND];
  auto load = [&](int h) {
#pragma unroll
    for (int i = 0; i < ROUND; i++) {
      const int at = h + i * G;
      a[i] = make_uint4(0, 0, 0, 0);
      if (at < h1 && l.works) a[i] = __ldcs(reinterpret_cast<const uint4*>(at < p.hq ? q + at * p.qs.h : k + (at - p.hq) * p.ks.h));
    }
  };
  load(h0 + l.mine);
  float cs[8], wq[8], wk[8];
  const int col = l.works ? l.v * 8 : 0;
  unpack8(*reinterpret_cast<const uint4*>(p.wq + col), wq);
  unpack8(*reinterpret_cast<const uint4*>(p.wk + col), wk);
  angles(p, b, s, l.v, l.works, cs);
  const float inv_d = 1.f / (float)p.d;
  bf16 *oq = p.oq + b * p.oqs.b + s * p.oqs.s + l.v * 8, *ok = p.ok + b * p.oks.b + s * p.oks.s + l.v * 8;
  for (int h = h0; h < h1; h += ROUND * G) {        // (the same for all lanes: they meet in the sums)
    if (h != h0) load(h + l.mine);
#pragma unroll
    for (int i = 0; i < ROUND; i++) {
      if (h + i * G >= h1) break;
      const int at = h + i * G + l.mine;
      float f[8], ss = 0.f;
      unpack8(a[i], f);
#pragma unroll
      for (int j = 0; j < 8; j++) ss += f[j] * f[j];
      const float rstd = rsqrtf(head_sum<P2>(ss) * inv_d + p.eps);
      const bool is_q = at < p.hq;
#pragma unroll
      for (int j = 0; j < 8; j++) f[j] = f[j] * rstd * (is_q ? wq[j] : wk[j]);
      rope_rotate8(cs, f);
      if (at < h1 && l.works) *reinterpret_cast<uint4*>(is_q ? oq + at * p.oqs.h : ok + (at - p.hq) * p.oks.h) = pack8(f);
    }
  }
}

// A warp walks over tokens; every thread keeps its share of dw.
constexpr int BWD_ROUND = 2, BWD_THREADS = 256;
template <int P2>
__global__ void __launch_bounds__(BWD_THREADS, 2) qk_norm_rope_bwd_kernel(const __grid_constant__ NormRopeParams p) {
  grid_go();
  grid_wait();
  const Lanes<P2> l(p.d);
  constexpr int G = Lanes<P2>::G, WARPS = BWD_THREADS / 32;
  const int heads = p.hq + p.hkv, parts = (heads + p.share - 1) / p.share;
  const long long items = (long long)p.B * p.S * parts;
  const float inv_d = 1.f / (float)p.d;
  float wq[8], wk[8], aq[8], ak[8];
  const int col = l.works ? l.v * 8 : 0;
  unpack8(*reinterpret_cast<const uint4*>(p.wq + col), wq);
  unpack8(*reinterpret_cast<const uint4*>(p.wk + col), wk);
#pragma unroll
  for (int j = 0; j < 8; j++) aq[j] = ak[j] = 0.f;
  for (long long item = (long long)blockIdx.x * WARPS + (threadIdx.x >> 5); item < items; item += (long long)gridDim.x * WARPS) {
    const long long tok = item / parts;
    const int part = (int)(item - tok * parts), b = (int)(tok / p.S), s = (int)(tok - (long long)b * p.S);
    const int h0 = part * p.share, h1 = min(heads, h0 + p.share);
    const bf16 *q = p.q + b * p.qs.b + s * p.qs.s + l.v * 8, *k = p.k + b * p.ks.b + s * p.ks.s + l.v * 8;
    const bf16 *dq = p.dq + b * p.dqs.b + s * p.dqs.s + l.v * 8, *dk = p.dk + b * p.dks.b + s * p.dks.s + l.v * 8;
    bf16 *oq = p.oq + b * p.oqs.b + s * p.oqs.s + l.v * 8, *ok = p.ok + b * p.oks.b + s * p.oks.s + l.v * 8;
    uint4 x[BWD_ROUND], y[BWD_ROUND];
    auto load = [&](int h) {
#pragma unroll
      for (int i = 0; i < BWD_ROUND; i++) {
        const int at = h + i * G;
        x[i] = y[i] = make_uint4(0, 0, 0, 0);
        if (at < h1 && l.works) {
          x[i] = __ldcs(reinterpret_cast<const uint4*>(at < p.hq ? q + at * p.qs.h : k + (at - p.hq) * p.ks.h));
          y[i] = __ldcs(reinterpret_cast<const uint4*>(at < p.hq ? dq + at * p.dqs.h : dk + (at - p.hq) * p.dks.h));
        }
      }
    };
    load(h0 + l.mine);
    float cs[8];
    angles(p, b, s, l.v, l.works, cs);
    for (int h = h0; h < h1; h += BWD_ROUND * G) {
      if (h != h0) load(h + l.mine);
#pragma unroll
      for (int i = 0; i < BWD_ROUND; i++) {
        if (h + i * G >= h1) break;
        const int at = h + i * G + l.mine;
        const bool is_q = at < p.hq, in = at < h1 && l.works;
        float f[8], g[8], ss = 0.f, dot = 0.f;
        unpack8(x[i], f);
        unpack8(y[i], g);
        if (in) rope_rotate8(cs, g, true);          // (elsewhere zeros, which a NaN of the tables leaves alone)
#pragma unroll
        for (int j = 0; j < 8; j++) ss += f[j] * f[j];
        ss = head_sum<P2>(ss);                      // (all lanes meet here)
        const float rstd = in ? rsqrtf(ss * inv_d + p.eps) : 0.f;
#pragma unroll
        for (int j = 0; j < 8; j++) {
          f[j] *= rstd;
          const float gx = g[j] * f[j];
          if (in) (is_q ? aq[j] : ak[j]) += gx;
          const float w = is_q ? wq[j] : wk[j];
          dot += gx * w;
          g[j] *= w;
        }
        dot = head_sum<P2>(dot) * inv_d;
#pragma unroll
        for (int j = 0; j < 8; j++) g[j] = rstd * (g[j] - f[j] * dot);
        if (in) *reinterpret_cast<uint4*>(is_q ? oq + at * p.oqs.h : ok + (at - p.hq) * p.oks.h) = pack8(g);
      }
    }
  }
  if (!p.partial) return;
  // over the heads of a warp, then over the warps of the CTA
  __shared__ float sums[2][WARPS][P2 * 8];
#pragma unroll
  for (int j = 0; j < 8; j++) {
#pragma unroll
    for (int o = P2; o < 32; o <<= 1) {
      aq[j] += __shfl_xor_sync(0xffffffffu, aq[j], o);
      ak[j] += __shfl_xor_sync(0xffffffffu, ak[j], o);
    }
  }
  if (l.mine == 0) {
#pragma unroll
    for (int j = 0; j < 8; j++) {
      sums[0][threadIdx.x >> 5][l.v * 8 + j] = aq[j];
      sums[1][threadIdx.x >> 5][l.v * 8 + j] = ak[j];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * p.d; i += BWD_THREADS) {
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
// Heads of a warp: all of a token's, or fewer where there are few tokens: one round of loads each at least, eight warps per SM.
int share_of(long long tokens, int heads, int d, int round) {
  const int per = 32 / padded(d) * round, most = (heads + per - 1) / per;
  const long long want = (8LL * lb_num_sms() + tokens - 1) / tokens;
  const int parts = (int)(want < most ? want : most);
  return (heads + parts - 1) / parts;
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
  const long long tokens = (long long)B * S, blocks = (tokens + 7) / 8;
  if (blocks > 2147483647LL) return LB_ERR_SHAPE;
  p.share = share_of(tokens, hq + hkv, d, ROUND);
  const int parts = (hq + hkv + p.share - 1) / p.share;
  if (parts > 65535) return LB_ERR_SHAPE;
#define LB_CALL(P) LB_LAUNCH(qk_norm_rope_kernel<P>, dim3((unsigned)blocks, (unsigned)parts), 256, 0, (cudaStream_t)stream, p)
  LB_BY_LANES(d, LB_CALL)
#undef LB_CALL
  return LB_OK;
}

// CTAs of the backward: its `partial` has 2 * d floats for each.
extern "C" int lb_qk_norm_rope_bwd_ctas(int B, int S, int hq, int hkv, int d) {
  if (B <= 0 || S <= 0 || hq <= 0 || hkv <= 0 || d <= 0 || d % 8 || d > 2 * MAX_PAIRS || (long long)hq + hkv > 0x3fffffff) return 0;
  const long long tokens = (long long)B * S;
  const int share = share_of(tokens, hq + hkv, d, BWD_ROUND), parts = (hq + hkv + share - 1) / share;
  const long long want = (tokens * parts + 7) / 8, most = 2LL * lb_num_sms();
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
  p.share = share_of((long long)B * S, hq + hkv, d, BWD_ROUND);
#define LB_CALL(P) LB_LAUNCH(qk_norm_rope_bwd_kernel<P>, ctas, BWD_THREADS, 0, (cudaStream_t)stream, p)
  LB_BY_LANES(d, LB_CALL)
#undef LB_CALL
  if (partial) LB_LAUNCH(qk_norm_rope_dw_kernel, (2 * d + 31) / 32, dim3(32, 32), 0, (cudaStream_t)stream, (const float*)partial, (bf16*)dwq, (bf16*)dwk, ctas, d);
  return LB_OK;
}
