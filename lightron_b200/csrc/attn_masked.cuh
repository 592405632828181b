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
  float* lse;                    // [B, hq, Sq]; -inf: a row that sees nothing
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

int ma_launch_fwd(const MaParams& p, cudaStream_t s);

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
