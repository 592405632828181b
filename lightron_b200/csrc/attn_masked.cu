// Attention under interval masks (attn_masked.cuh): the intervals of a batch, forward and backward.
#include "attn_masked.cuh"

namespace {

constexpr int PLAN_THREADS = 1024;

// Value of the nearest thread before (or, REVERSE, behind) this one that has one (>= 0); -1: none has.
template <bool REVERSE>
__device__ __forceinline__ int carry_in(int own, int* sh) {
  const int t = REVERSE ? PLAN_THREADS - 1 - (int)threadIdx.x : (int)threadIdx.x;
  const int lane = threadIdx.x & 31, w = t >> 5, l = REVERSE ? 31 - lane : lane;
  int v = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = REVERSE ? __shfl_down_sync(0xffffffffu, v, o) : __shfl_up_sync(0xffffffffu, v, o);
    if (l >= o && v < 0) v = x;
  }
  __syncthreads();
  if (l == 31) sh[w] = v;
  __syncthreads();
  int before = REVERSE ? __shfl_down_sync(0xffffffffu, v, 1) : __shfl_up_sync(0xffffffffu, v, 1);
  if (l == 0) before = -1;
  for (int i = w - 1; i >= 0 && before < 0; i--) before = sh[i];
  return before;
}

// Intervals of one sequence by one CTA, a run of positions per thread.  A document is a run of equal ids; ids below zero are padding, which sees nothing and
// is seen by nothing (an empty interval at its own place keeps the ends in order).  The prefix of a document is the marked run at its start.
template <typename Id>
__global__ void __launch_bounds__(PLAN_THREADS) attn_mask_kernel(const Id* __restrict__ ids, const unsigned char* __restrict__ marks, const int* __restrict__ lens,
                                                                 int S, int causal, int2* __restrict__ qb, int2* __restrict__ kb) {
  __shared__ int sh[32];
  grid_go();
  grid_wait();
  const long long base = (long long)blockIdx.x * S;
  if (ids) ids += base;
  if (marks) marks += base;
  qb += base;
  kb += base;
  const int len = lens ? lens[blockIdx.x] : 0;
  const int per = (S + PLAN_THREADS - 1) / PLAN_THREADS;
  const int a = min(S, (int)threadIdx.x * per), e = min(S, a + per);
  auto starts = [&](int i) { return i == 0 || (ids && ids[i] != ids[i - 1]); };
  auto plain = [&](int i) { return marks ? marks[i] == 0 : i >= len; };          // outside the prefix part
  int first_start = -1, last_start = -1, first_plain = -1;
  for (int i = a; i < e; i++) {
    if (starts(i)) { last_start = i; if (first_start < 0) first_start = i; }
    if (first_plain < 0 && plain(i)) first_plain = i;
  }
  int end = carry_in<true>(first_start, sh), np = carry_in<true>(first_plain, sh), start = carry_in<false>(last_start, sh);
  if (end < 0) end = S;
  if (np < 0) np = S;
  // backwards: end of the document, and the first position from here on that is not marked
  for (int i = e - 1; i >= a; i--) {
    if (plain(i)) np = i;
    kb[i].y = end;
    qb[i].y = np;
    if (starts(i)) end = i;
  }
  __syncthreads();
  int prefix = start >= 0 && a < e ? qb[start].y : 0;      // (unused where this thread's first position starts a document)
  __syncthreads();
  for (int i = a; i < e; i++) {
    if (starts(i)) { start = i; prefix = qb[i].y; }
    const int stop = kb[i].y, pe = min(prefix, stop);
    if (ids && ids[i] < 0) {
      qb[i] = kb[i] = make_int2(i, i);
    } else {
      qb[i] = make_int2(start, causal ? max(i + 1, pe) : stop);
      kb[i] = make_int2(causal && i >= pe ? i : start, stop);
    }
  }
}

bool bad_strides(const MaStrides& s) { return (s.b | s.s | s.h) % 8 != 0; }
bool misaligned(const void* p) { return ((uintptr_t)p & 15) != 0; }
MaStrides strides_at(const long long* s) { return MaStrides{s[0], s[1], s[2]}; }

int check_sizes(int B, int Sq, int Sk, int hq, int hkv, int d) {
  return B <= 0 || Sq <= 0 || Sk < Sq || hq <= 0 || hkv <= 0 || hq % hkv || d <= 0 || d % 8 || d > 128 ? LB_ERR_SHAPE : LB_OK;
}

int fill(MaParams& p, const void* q, const void* k, const void* v, void* o, void* o_lo, void* lse, int B, int Sq, int Sk, int hq, int hkv, int d, const long long* st,
         float scale, int causal, float softcap, const void* slopes, const void* q_bounds, const void* k_bounds) {
  if (check_sizes(B, Sq, Sk, hq, hkv, d)) return LB_ERR_SHAPE;
  if (!q || !k || !v || !o || !lse || !st || !(softcap >= 0.f && softcap < INFINITY) || !(scale > 0.f && scale < INFINITY) || (!q_bounds) != (!k_bounds)) return LB_ERR_ARG;
  if (misaligned(q) || misaligned(k) || misaligned(v) || misaligned(o) || misaligned(o_lo)) return LB_ERR_ARG;
  p = MaParams{(const bf16*)q, (const bf16*)k, (const bf16*)v, strides_at(st), strides_at(st + 3), strides_at(st + 6), (bf16*)o, (bf16*)o_lo, (float*)lse, B, Sq, Sk, hq, hkv, d,
               scale, causal, softcap, (const float*)slopes, (const int2*)q_bounds, (const int2*)k_bounds};
  return bad_strides(p.qs) || bad_strides(p.ks) || bad_strides(p.vs) ? LB_ERR_SHAPE : LB_OK;
}

}  // namespace

// Intervals of B sequences of S positions: q_bounds [B, S, 2] the keys that a position sees, k_bounds [B, S, 2] the positions that see a key.
// ids: null or [B, S] of id_bytes (4 or 8) each; marks: null or [B, S] bytes, or lens: null or [B], the prefix part by its marks or its length.
extern "C" int lb_attn_mask(const void* ids, int id_bytes, const void* marks, const void* lens, int B, int S, int causal, void* q_bounds, void* k_bounds, void* stream) {
  if (B <= 0 || S <= 0) return LB_ERR_SHAPE;
  if (!q_bounds || !k_bounds || (ids && id_bytes != 4 && id_bytes != 8) || (marks && lens)) return LB_ERR_ARG;
  cudaStream_t s = (cudaStream_t)stream;
  if (id_bytes == 8)
    LB_LAUNCH(attn_mask_kernel<long long>, B, PLAN_THREADS, 0, s, (const long long*)ids, (const unsigned char*)marks, (const int*)lens, S, causal, (int2*)q_bounds, (int2*)k_bounds);
  else
    LB_LAUNCH(attn_mask_kernel<int>, B, PLAN_THREADS, 0, s, (const int*)ids, (const unsigned char*)marks, (const int*)lens, S, causal, (int2*)q_bounds, (int2*)k_bounds);
  return LB_OK;
}

// Forward.  strides: 3 x {batch, token, head} of q, k, v in elements, multiples of 8; o, o_lo (or null) [B, Sq, hq, d] and lse [B, hq, Sq] contiguous.
// head_dim a multiple of 8 up to 128, Sk >= Sq; slopes null or fp32 [hq]; q_bounds / k_bounds of lb_attn_mask() over Sk positions, or null: causal or all keys.
extern "C" int lb_masked_attn_fwd(const void* q, const void* k, const void* v, void* o, void* o_lo, void* lse, int B, int Sq, int Sk, int hq, int hkv, int d,
                                  const long long* strides, float scale, int causal, float softcap, const void* slopes, const void* q_bounds, const void* k_bounds,
                                  void* stream) {
  MaParams p;
  if (const int rc = fill(p, q, k, v, o, o_lo, lse, B, Sq, Sk, hq, hkv, d, strides, scale, causal, softcap, slopes, q_bounds, k_bounds)) return rc;
  return ma_launch_fwd(p, (cudaStream_t)stream);
}

// Bytes of the backward's workspace; 0 for sizes that it does not take.
extern "C" long long lb_masked_attn_bwd_ws_bytes(int B, int Sq, int Sk, int hq, int hkv, int d, int causal) {
  MaParams p{};
  if (check_sizes(B, Sq, Sk, hq, hkv, d)) return 0;
  p.B = B; p.Sq = Sq; p.Sk = Sk; p.hq = hq; p.hkv = hkv; p.d = d; p.causal = causal;
  return ma_bwd_ws_bytes(p);
}

// Backward.  strides: 7 x {batch, token, head} of q, k, v, dout, dq, dk, dv; o, o_lo, lse as the forward left them; ws: lb_masked_attn_bwd_ws_bytes(), 16-byte aligned.
extern "C" int lb_masked_attn_bwd(const void* q, const void* k, const void* v, const void* o, const void* o_lo, const void* dout, const void* lse, void* ws, long long ws_bytes,
                                  void* dq, void* dk, void* dv, int B, int Sq, int Sk, int hq, int hkv, int d, const long long* strides, float scale, int causal, float softcap,
                                  const void* slopes, const void* q_bounds, const void* k_bounds, void* stream) {
  MaBwdParams w;
  if (const int rc = fill(w.f, q, k, v, const_cast<void*>(o), const_cast<void*>(o_lo), const_cast<void*>(lse), B, Sq, Sk, hq, hkv, d, strides, scale, causal, softcap, slopes, q_bounds, k_bounds)) return rc;
  if (!o_lo || !dout || !ws || !dq || !dk || !dv || misaligned(dout) || misaligned(ws) || misaligned(dq) || misaligned(dk) || misaligned(dv)) return LB_ERR_ARG;
  if (ws_bytes < ma_bwd_ws_bytes(w.f)) return LB_ERR_CAPACITY;
  w.dout = (const bf16*)dout; w.dq = (bf16*)dq; w.dk = (bf16*)dk; w.dv = (bf16*)dv; w.stats = (float*)ws;
  w.dos = strides_at(strides + 9); w.dqs = strides_at(strides + 12); w.dks = strides_at(strides + 15); w.dvs = strides_at(strides + 18);
  if (bad_strides(w.dos) || bad_strides(w.dqs) || bad_strides(w.dks) || bad_strides(w.dvs)) return LB_ERR_SHAPE;
  return ma_launch_bwd(w, (cudaStream_t)stream);
}
