// Attention under interval masks (attn_masked.cuh): the intervals of a batch, forward and backward.
#include "attn_masked.cuh"

namespace {

constexpr int PLAN_THREADS = 512;

// Within a warp: value of the nearest lane before (or, REVERSE, behind) this one that has one (>= 0), in `before`; of the nearest up to and with it, returned.  -1: none has.
template <bool REVERSE>
__device__ __forceinline__ int nearest_in_warp(int v, int& before) {
  const int l = REVERSE ? 31 - ((int)threadIdx.x & 31) : (int)threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = REVERSE ? __shfl_down_sync(0xffffffffu, v, o) : __shfl_up_sync(0xffffffffu, v, o);
    if (l >= o && v < 0) v = x;
  }
  before = REVERSE ? __shfl_down_sync(0xffffffffu, v, 1) : __shfl_up_sync(0xffffffffu, v, 1);
  if (l == 0) before = -1;
  return v;
}
// The same over the warps, of which `of_warps` has a value each, where the warp itself has none.
template <bool REVERSE>
__device__ __forceinline__ int nearest_of(const int* of_warps, int before) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, x = lane < (int)(blockDim.x >> 5) ? of_warps[lane] : -1;
  const unsigned has = __ballot_sync(0xffffffffu, x >= 0 && (REVERSE ? lane > w : lane < w));
  const int y = __shfl_sync(0xffffffffu, x, !has ? 0 : REVERSE ? __ffs(has) - 1 : 31 - __clz(has));
  return before >= 0 ? before : has ? y : -1;
}

// Intervals of one sequence.  A document is a run of equal ids; ids below zero are padding, which sees nothing and is seen by nothing (an empty interval at its own
// place keeps the ends in order).  The prefix of a document is the marked run at its start.
// Every CTA of a sequence reads all of its ids, 32 positions a warp and load, into two words: where documents start, and what is outside of prefixes.  The words' nearest
// starts on either side and nearest outside position come from scans over the words; a position's own from its word.  A CTA then writes its share of the positions.
template <typename Id>
__global__ void __launch_bounds__(PLAN_THREADS) attn_mask_kernel(const Id* __restrict__ ids, const unsigned char* __restrict__ marks, const int* __restrict__ lens,
                                                                 int S, int causal, int2* __restrict__ qb, int2* __restrict__ kb) {
  extern __shared__ uint32_t words[];             // [5][n]: starts, outside, start before the word, start behind it, outside behind it
  __shared__ int of_warps[3][32];
  grid_go();
  grid_wait();
  const long long base = (long long)blockIdx.y * S;
  if (ids) ids += base;
  if (marks) marks += base;
  qb += base;
  kb += base;
  const int len = lens ? lens[blockIdx.y] : 0;
  const int n = (S + 31) / 32, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t *starts = words, *outside = words + n;
  int *before = reinterpret_cast<int*>(words + 2 * n), *behind = before + n, *outside_behind = behind + n;
  constexpr int U = 4;                            // words of a warp on their way
  for (int w0 = warp; w0 < n; w0 += U * (PLAN_THREADS / 32)) {
    Id id[U], prev[U];
    unsigned char m[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int i = (w0 + u * (PLAN_THREADS / 32)) * 32 + lane;
      const bool in = i < S;
      id[u] = in && ids ? ids[i] : Id(0);
      prev[u] = in && ids && i > 0 ? ids[i - 1] : Id(0);
      m[u] = in && marks ? marks[i] : 0;
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int w = w0 + u * (PLAN_THREADS / 32), i = w * 32 + lane;
      const uint32_t s = __ballot_sync(0xffffffffu, i < S && (i == 0 || id[u] != prev[u])), o = __ballot_sync(0xffffffffu, i < S && (marks ? m[u] == 0 : i >= len));
      if (lane == 0 && w < n) { starts[w] = s; outside[w] = o; }
    }
  }
  __syncthreads();
  const int per = (n + PLAN_THREADS - 1) / PLAN_THREADS, a = min(n, (int)threadIdx.x * per), e = min(n, a + per);
  int first_start = -1, last_start = -1, first_out = -1;
  for (int w = a; w < e; w++) {
    const uint32_t s = starts[w], o = outside[w];
    if (s) { last_start = w * 32 + 31 - __clz(s); if (first_start < 0) first_start = w * 32 + __ffs(s) - 1; }
    if (o && first_out < 0) first_out = w * 32 + __ffs(o) - 1;
  }
  int run, next, out;
  const int w_last = nearest_in_warp<false>(last_start, run), w_first = nearest_in_warp<true>(first_start, next), w_out = nearest_in_warp<true>(first_out, out);
  if (lane == 31) of_warps[0][warp] = w_last;
  if (lane == 0) { of_warps[1][warp] = w_first; of_warps[2][warp] = w_out; }
  __syncthreads();
  run = nearest_of<false>(of_warps[0], run);
  next = nearest_of<true>(of_warps[1], next);
  out = nearest_of<true>(of_warps[2], out);
  for (int w = a; w < e; w++) {
    before[w] = run;
    if (starts[w]) run = w * 32 + 31 - __clz(starts[w]);
  }
  for (int w = e - 1; w >= a; w--) {
    behind[w] = next < 0 ? S : next;
    outside_behind[w] = out < 0 ? S : out;
    if (starts[w]) next = w * 32 + __ffs(starts[w]) - 1;
    if (outside[w]) out = w * 32 + __ffs(outside[w]) - 1;
  }
  __syncthreads();
  for (int i = (int)blockIdx.x * PLAN_THREADS + (int)threadIdx.x; i < S; i += (int)gridDim.x * PLAN_THREADS) {
    const int w = i >> 5, b = i & 31;
    const uint32_t upto = starts[w] & (0xffffffffu >> (31 - b)), after = b == 31 ? 0u : starts[w] >> (b + 1);
    const int start = upto ? w * 32 + 31 - __clz(upto) : before[w], stop = after ? i + __ffs(after) : behind[w];
    const uint32_t o = outside[start >> 5] >> (start & 31);
    const int pe = min(o ? start + __ffs(o) - 1 : outside_behind[start >> 5], stop);
    if (ids && ids[i] < 0) {
      qb[i] = kb[i] = make_int2(i, i);
    } else {
      qb[i] = make_int2(start, causal ? max(i + 1, pe) : stop);
      kb[i] = make_int2(causal && i >= pe ? i : start, stop);
    }
  }
}

constexpr int MAX_MASK_LENGTH = 200 * 1024 / 20 * 32;      // five words for 32 positions in 200 KB of shared memory

bool bad_strides(const MaStrides& s) { return (s.b | s.s | s.h) % 8 != 0; }
bool misaligned(const void* p) { return ((uintptr_t)p & 15) != 0; }
MaStrides strides_at(const long long* s) { return MaStrides{s[0], s[1], s[2]}; }

int check_sizes(int B, int Sq, int Sk, int hq, int hkv, int d) {
  return B <= 0 || Sq <= 0 || Sk < Sq || hq <= 0 || hkv <= 0 || hq % hkv || d <= 0 || d % 8 || d > 128 ? LB_ERR_SHAPE : LB_OK;
}

int fill(MaParams& p, const void* q, const void* k, const void* v, void* o, void* o_lo, void* lse, int B, int Sq, int Sk, int hq, int hkv, int d, const long long* st,
         float scale, int causal, float softcap, const void* slopes, const void* q_bounds, const void* k_bounds) {
  if (check_sizes(B, Sq, Sk, hq, hkv, d)) return LB_ERR_SHAPE;
  if (!q || !k || !v || !o || (!o_lo) != (!lse) || !st || !(softcap >= 0.f && softcap < INFINITY) || !(scale > 0.f && scale < INFINITY) || (!q_bounds) != (!k_bounds)) return LB_ERR_ARG;
  if (misaligned(q) || misaligned(k) || misaligned(v) || misaligned(o) || misaligned(o_lo)) return LB_ERR_ARG;
  p = MaParams{(const bf16*)q, (const bf16*)k, (const bf16*)v, strides_at(st), strides_at(st + 3), strides_at(st + 6), (bf16*)o, (bf16*)o_lo, (float*)lse, B, Sq, Sk, hq, hkv, d,
               scale, causal, softcap, (const float*)slopes, (const int2*)q_bounds, (const int2*)k_bounds, 0, 0};
  return bad_strides(p.qs) || bad_strides(p.ks) || bad_strides(p.vs) ? LB_ERR_SHAPE : LB_OK;
}

// Whether the forward takes a window over all keys as one of their number, which has the heads of a group as a tile's rows, instead of as none: where heads fill the SMs by themselves, or the cache is
// long.  One key short of all / as none, us, hq / hkv, d 128, one query: 8 sequences of 32 / 8 heads, 256 keys 14 / 16, 4096 43 / 88, 65536 352 / 1182; one sequence, 1024 keys 25 / 25, 4096 27 / 39; 32 of
// 16 / 1, 4096 keys 33 / 166; 64 queries, 8 sequences of 32 / 8, 4096 keys 70 / 90; left as none: one sequence of 16 / 1, 512 keys 20 / 18; 64 queries over 16384 70 / 53; 100 queries, 8 sequences of 32 / 8,
// 4096 keys 92 / 90.
bool rows_of_heads(const MaParams& p) {
  const int shift = ma_group_shift(p);
  return shift > 0 && p.Sq <= 64 && ((long long)p.hq * p.B >= lb_num_sms() || (p.Sq << shift <= 128 && p.Sk >= 2048));
}
// A window over all keys is none, but for that.  (Sums of a place and the window have to stay in 32 bits.)
int set_window(MaParams& p, int window, int sinks, bool forward) {
  if (window <= 0 || sinks < 0) return LB_ERR_ARG;
  if (p.Sk > (1 << 29)) return LB_ERR_SHAPE;
  p.window = window < p.Sk ? window : forward && rows_of_heads(p) ? p.Sk : 0;
  p.sinks = !p.window || p.window == p.Sk ? 0 : sinks < p.Sk ? sinks : p.Sk;
  return LB_OK;
}

}  // namespace

// Intervals of B sequences of S positions: q_bounds [B, S, 2] the keys that a position sees, k_bounds [B, S, 2] the positions that see a key.
// ids: null or [B, S] of id_bytes (4 or 8) each; marks: null or [B, S] bytes, or lens: null or [B], the prefix part by its marks or its length.
extern "C" int lb_attn_mask(const void* ids, int id_bytes, const void* marks, const void* lens, int B, int S, int causal, void* q_bounds, void* k_bounds, void* stream) {
  if (B <= 0 || B > 65535 || S <= 0) return LB_ERR_SHAPE;
  if (!q_bounds || !k_bounds || (ids && id_bytes != 4 && id_bytes != 8) || (marks && lens)) return LB_ERR_ARG;
  cudaStream_t s = (cudaStream_t)stream;
  if (S > MAX_MASK_LENGTH) return LB_ERR_SHAPE;
  const int smem = (S + 31) / 32 * 20;
  static MaOnce once;
  bool* const set = once.here();
  if (!set) return LB_ERR_LAUNCH;
  if (!*set) {
    cudaFuncSetAttribute(attn_mask_kernel<int>, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_MASK_LENGTH / 32 * 20);
    cudaFuncSetAttribute(attn_mask_kernel<long long>, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_MASK_LENGTH / 32 * 20);
    *set = true;
  }
  // four positions a thread, where the sequences leave room for as many CTAs
  const int most = (S + 4 * PLAN_THREADS - 1) / (4 * PLAN_THREADS), room = lb_num_sms() / B;
  const dim3 grid((unsigned)(room < 1 ? 1 : room < most ? room : most), (unsigned)B);
  if (id_bytes == 8)
    LB_LAUNCH(attn_mask_kernel<long long>, grid, PLAN_THREADS, smem, s, (const long long*)ids, (const unsigned char*)marks, (const int*)lens, S, causal, (int2*)q_bounds, (int2*)k_bounds);
  else
    LB_LAUNCH(attn_mask_kernel<int>, grid, PLAN_THREADS, smem, s, (const int*)ids, (const unsigned char*)marks, (const int*)lens, S, causal, (int2*)q_bounds, (int2*)k_bounds);
  return LB_OK;
}

// Bytes of the forward's workspace: 0 where it uses none, as for sizes that it does not take.
extern "C" long long lb_masked_attn_fwd_ws_bytes(int B, int Sq, int Sk, int hq, int hkv, int d) {
  MaParams p{};
  if (check_sizes(B, Sq, Sk, hq, hkv, d)) return 0;
  p.B = B; p.Sq = Sq; p.Sk = Sk; p.hq = hq; p.hkv = hkv; p.d = d;
  return ma_fwd_ws_bytes(p);
}

// Forward.  strides: 3 x {batch, token, head} of q, k, v in elements, multiples of 8; o [B, Sq, hq, d] contiguous, as are, for the backward, o_lo [B, Sq, hq, d] and lse
// [B, hq, Sq] (both, or both null).
// head_dim a multiple of 8 up to 128, Sk >= Sq; slopes null or fp32 [hq]; q_bounds / k_bounds of lb_attn_mask() over Sk positions, or null: causal or all keys.
// ws: lb_masked_attn_fwd_ws_bytes(), 16-byte aligned, not initialised (with less, or null, few tiles are not split over their keys).
extern "C" int lb_masked_attn_fwd(const void* q, const void* k, const void* v, void* o, void* o_lo, void* lse, void* ws, long long ws_bytes, int B, int Sq, int Sk, int hq, int hkv,
                                  int d, const long long* strides, float scale, int causal, float softcap, const void* slopes, const void* q_bounds, const void* k_bounds, void* stream) {
  MaParams p;
  if (const int rc = fill(p, q, k, v, o, o_lo, lse, B, Sq, Sk, hq, hkv, d, strides, scale, causal, softcap, slopes, q_bounds, k_bounds)) return rc;
  if (misaligned(ws)) return LB_ERR_ARG;
  return ma_launch_fwd(p, ws, ws ? ws_bytes : 0, (cudaStream_t)stream);
}

// The forward under a window: of the keys of its interval a query sees those less than `window` (1 or more) positions away, and the first `sinks` of the interval.  The rest as in
// lb_masked_attn_fwd(), with a workspace of lb_window_attn_fwd_ws_bytes().
extern "C" long long lb_window_attn_fwd_ws_bytes(int B, int Sq, int Sk, int hq, int hkv, int d, int causal, int window, int sinks) {
  MaParams p{};
  if (check_sizes(B, Sq, Sk, hq, hkv, d)) return 0;
  p.B = B; p.Sq = Sq; p.Sk = Sk; p.hq = hq; p.hkv = hkv; p.d = d; p.causal = causal;
  return set_window(p, window, sinks, true) ? 0 : ma_fwd_ws_bytes(p);
}
extern "C" int lb_window_attn_fwd(const void* q, const void* k, const void* v, void* o, void* o_lo, void* lse, void* ws, long long ws_bytes, int B, int Sq, int Sk, int hq, int hkv,
                                  int d, const long long* strides, float scale, int causal, float softcap, const void* slopes, const void* q_bounds, const void* k_bounds, int window, int sinks,
                                  void* stream) {
  MaParams p;
  if (const int rc = fill(p, q, k, v, o, o_lo, lse, B, Sq, Sk, hq, hkv, d, strides, scale, causal, softcap, slopes, q_bounds, k_bounds)) return rc;
  if (const int rc = set_window(p, window, sinks, true)) return rc;
  if (misaligned(ws)) return LB_ERR_ARG;
  return (p.window ? ma_launch_window_fwd : ma_launch_fwd)(p, ws, ws ? ws_bytes : 0, (cudaStream_t)stream);
}

// Bytes of the backward's workspace; 0 for sizes that it does not take.
extern "C" long long lb_masked_attn_bwd_ws_bytes(int B, int Sq, int Sk, int hq, int hkv, int d, int causal) {
  MaParams p{};
  if (check_sizes(B, Sq, Sk, hq, hkv, d)) return 0;
  p.B = B; p.Sq = Sq; p.Sk = Sk; p.hq = hq; p.hkv = hkv; p.d = d; p.causal = causal;
  return ma_bwd_ws_bytes(p, false);
}

namespace {
int backward(const void* q, const void* k, const void* v, const void* o, const void* o_lo, const void* dout, const void* lse, void* ws, long long ws_bytes, void* dq, void* dk, void* dv, int B, int Sq,
             int Sk, int hq, int hkv, int d, const long long* strides, float scale, int causal, float softcap, const void* slopes, const void* q_bounds, const void* k_bounds, bool windowed, int window,
             int sinks, void* stream) {
  MaBwdParams w;
  if (const int rc = fill(w.f, q, k, v, const_cast<void*>(o), const_cast<void*>(o_lo), const_cast<void*>(lse), B, Sq, Sk, hq, hkv, d, strides, scale, causal, softcap, slopes, q_bounds, k_bounds)) return rc;
  if (windowed)
    if (const int rc = set_window(w.f, window, sinks, false)) return rc;
  if (!o_lo || !dout || !ws || !dq || !dk || !dv || misaligned(dout) || misaligned(ws) || misaligned(dq) || misaligned(dk) || misaligned(dv)) return LB_ERR_ARG;
  if (ws_bytes < ma_bwd_ws_bytes(w.f, w.f.qb != nullptr)) return LB_ERR_CAPACITY;
  w.dout = (const bf16*)dout; w.dq = (bf16*)dq; w.dk = (bf16*)dk; w.dv = (bf16*)dv; w.stats = (float*)ws;
  w.dos = strides_at(strides + 9); w.dqs = strides_at(strides + 12); w.dks = strides_at(strides + 15); w.dvs = strides_at(strides + 18);
  if (bad_strides(w.dos) || bad_strides(w.dqs) || bad_strides(w.dks) || bad_strides(w.dvs)) return LB_ERR_SHAPE;
  return ma_launch_bwd(w, (cudaStream_t)stream);
}
}  // namespace

// Backward.  strides: 7 x {batch, token, head} of q, k, v, dout, dq, dk, dv; o, o_lo, lse as the forward left them; ws: lb_masked_attn_bwd_ws_bytes(), 16-byte aligned.
extern "C" int lb_masked_attn_bwd(const void* q, const void* k, const void* v, const void* o, const void* o_lo, const void* dout, const void* lse, void* ws, long long ws_bytes,
                                  void* dq, void* dk, void* dv, int B, int Sq, int Sk, int hq, int hkv, int d, const long long* strides, float scale, int causal, float softcap,
                                  const void* slopes, const void* q_bounds, const void* k_bounds, void* stream) {
  return backward(q, k, v, o, o_lo, dout, lse, ws, ws_bytes, dq, dk, dv, B, Sq, Sk, hq, hkv, d, strides, scale, causal, softcap, slopes, q_bounds, k_bounds, false, 0, 0, stream);
}

// Under a window, as lb_window_attn_fwd(); ws: lb_window_attn_bwd_ws_bytes(), of calls with bounds (masked 1) or without (0).
extern "C" long long lb_window_attn_bwd_ws_bytes(int B, int Sq, int Sk, int hq, int hkv, int d, int causal, int window, int sinks, int masked) {
  MaParams p{};
  if (check_sizes(B, Sq, Sk, hq, hkv, d)) return 0;
  p.B = B; p.Sq = Sq; p.Sk = Sk; p.hq = hq; p.hkv = hkv; p.d = d; p.causal = causal;
  return set_window(p, window, sinks, false) ? 0 : ma_bwd_ws_bytes(p, masked != 0);
}
extern "C" int lb_window_attn_bwd(const void* q, const void* k, const void* v, const void* o, const void* o_lo, const void* dout, const void* lse, void* ws, long long ws_bytes,
                                  void* dq, void* dk, void* dv, int B, int Sq, int Sk, int hq, int hkv, int d, const long long* strides, float scale, int causal, float softcap,
                                  const void* slopes, const void* q_bounds, const void* k_bounds, int window, int sinks, void* stream) {
  return backward(q, k, v, o, o_lo, dout, lse, ws, ws_bytes, dq, dk, dv, B, Sq, Sk, hq, hkv, d, strides, scale, causal, softcap, slopes, q_bounds, k_bounds, true, window, sinks, stream);
}
