// Attention under interval masks, with capped scores and a bias that falls with distance: what its kernels share.
//
// Query i sits at key position i + off, off = Sk - Sq.  With x = scale * q_i . k_j
//     s_ij = softcap * tanh(x / softcap) - slope_h * |i + off - j|        (x itself without a cap)
// and the softmax of row i runs over the keys lo <= j < hi of its interval.  Documents, prefixes and causality all make such intervals, whose ends
// never fall from one row to the next; the rows that see a key are then an interval too.  So a tile's keys follow from its first and last row,
// a mask costs two comparisons in the tiles where an interval ends, and nothing anywhere else.
#pragma once
#include "common.cuh"

struct MaStrides { long long b, s, h; };      // elements; the innermost dimension is contiguous

struct MaParams {
  const bf16 *q, *k, *v;
  MaStrides qs, ks, vs;
  bf16 *o, *o_lo;                // [B, Sq, hq, d]; o_lo: null, or what rounding o to bf16 left
  float* lse;                    // [B, hq, Sq], with o_lo; -inf: a row that sees nothing
  int B, Sq, Sk, hq, hkv, d;
  float scale;
  int causal;
  float softcap;                 // 0: none
  const float* slopes;           // null, or [hq]
  const int2 *qb, *kb;           // null, or [B, Sk]: keys that a position sees, positions that see a key
};

struct MaBwdParams {
  MaParams f;
  const bf16* dout;
  MaStrides dos;
  bf16 *dq, *dk, *dv;
  MaStrides dqs, dks, dvs;
  float* stats;
};

// A kernel's attributes count on the device where they were set: the flag of the current one (null: none, or not among the first 64).
struct MaOnce {
  bool done[64] = {false};
  bool* here() {
    int dev = 0;
    return cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64 ? done + dev : nullptr;
  }
};

int ma_launch_fwd(const MaParams& p, void* ws, long long ws_bytes, cudaStream_t s);
long long ma_fwd_ws_bytes(const MaParams& p);
int ma_launch_bwd(const MaBwdParams& w, cudaStream_t s);
long long ma_bwd_ws_bytes(const MaParams& p);

// What the kernels need of the scores' form, in units of log2: x * scale without a cap; with one, tanh(u) * times, u = x * by, as x * (c[0] + c[1] x^2 + c[2] x^4 + c[3] x^6) while
// |x| <= limit: relative error 2.2e-6 up to u = 0.6 (coefficients of tanh(u) / u in u^2, found by least squares over Chebyshev points with weights that were raised
// where the error was largest).  The limit is u = 0.6 or less:
//   * 33 / cap, that is scores of 33, where the error is 7e-5 of a score; the definition's, some 1.3e-7 caps wherever the score lies, is reached at u = 0.06, which is the least;
//   * coefficients that fp32 holds as zero (small scales, large caps: powers of by) have to be small against the error where they are missing: 0.041 u^6, 0.13 u^4, u^2 / 3;
//   * where one overflows (caps below some 1e-7 times the scale) the definition is taken for every score: infinity times the square of a score that is exactly zero would be NaN.
// Pairs hold a value twice.
struct MaTerms {
  unsigned long long scale, cap, c[4];
  float scale1, cap1, by2, limit;       // by2: 2 * log2(e) * by, for tanh by its definition
  void set(const MaParams& p, bool times_cap, unsigned long long (*twice)(float)) {
    const double log2e = 1.4426950408889634, k[4] = {0.9999978542327881, -0.33314040303230286, 0.13057856261730194, -0.04092942178249359};
    scale1 = (float)(p.scale * log2e);
    cap1 = (float)(p.softcap * log2e);
    scale = twice(scale1);
    cap = twice(cap1);
    by2 = limit = 0.f;
    const double by = p.softcap > 0.f ? (double)p.scale / p.softcap : 0.0;
    double pw = by * (times_cap ? p.softcap * log2e : 1.0);
    constexpr double missing[4] = {0.0, 0.0025, 0.06, 0.1};      // u up to which c[i] may be left out: 2.1e-6, 1.7e-6, 4.1e-8
    double most = p.softcap > 55.f ? fmax(33.0 / p.softcap, 0.06) : 0.6;
    for (int i = 0; i < 4; i++, pw *= by * by) {
      c[i] = twice((float)(k[i] * pw));
      if (!(pw < 3e38)) most = -1.0;
      if (fabs(k[i] * pw) < 1.2e-38) most = fmin(most, missing[i]);
    }
    if (p.softcap > 0.f) {
      by2 = (float)(2.0 * log2e * by < 3e38 ? 2.0 * log2e * by : 3e38);
      limit = most < 0.0 ? -1.f : (float)(most / by);
    } else {
      c[0] = scale;
    }
  }
};

// Bits [lo, hi) of 32 columns, of which column 0 is at `at`.
__device__ __forceinline__ uint32_t ma_bits(int lo, int hi, int at) {
  const int a = min(max(lo - at, 0), 32), e = min(max(hi - at, 0), 32);
  const uint32_t below_e = e == 32 ? 0xffffffffu : (1u << e) - 1u, below_a = a == 32 ? 0xffffffffu : (1u << a) - 1u;
  return below_e & ~below_a;
}

// Keys [x, y) that query i of sequence b sees.
__device__ __forceinline__ int2 ma_keys(const MaParams& p, int b, int i) {
  const int at = i + p.Sk - p.Sq;
  if (p.qb) return p.qb[(long long)b * p.Sk + at];
  return make_int2(0, p.causal ? at + 1 : p.Sk);
}
// Queries [x, y) that see key j.
__device__ __forceinline__ int2 ma_queries(const MaParams& p, int b, int j) {
  const int off = p.Sk - p.Sq;
  if (p.kb) {
    const int2 r = p.kb[(long long)b * p.Sk + j];
    return make_int2(max(r.x - off, 0), max(r.y - off, 0));
  }
  return make_int2(p.causal ? max(j - off, 0) : 0, p.Sq);
}
