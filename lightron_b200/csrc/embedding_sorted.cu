// Scaled embedding, and its gradient by sorted tokens:
//     y_t = scale * w[id_t]         dw[v] = scale * sum over the t with id_t = v, in their order, of dy_t
// The weight holds vocab ids [v0, v1); ids outside give zero rows and no gradient (vocab-parallel partial result).
//
// Forward: memory bound, rows of w in, rows of y out.
// Backward: the tokens are ordered by id, equal ids by their places (few by comparison, many by a radix sort of one cluster); then CTAs take chunks of that order and sum rows in 32
// bits, scale, round once and write, while others clear the rows that have no token.  What chunks have of a row that is longer than two of them goes to places of their own in 32 bits, which a
// last kernel adds up, always in the same order.  No atomics on values: the same bits in every run.  Bound by memory: every dy once, every row of dw once.
// 16384 tokens of 2048 columns into 32000 rows: forward 15 us, order 13 to 15 (latency: two passes, six barriers each), sums and clearing 33 (198 MB at 6.0 TB/s), join 7; 8192 x 4096 into 128256 rows 17, 13,
// 156 (7.1 TB/s: part of it stays in L2) and 8.  Rows of odd length go by single columns: 15001 x 1021, two thirds of them one row, 13, 13, 36 and 11.
#include "common.cuh"

namespace {

template <int VEC> struct Vec;      // VEC bf16 of a row
template <> struct Vec<8> { typedef uint4 type; };
template <> struct Vec<2> { typedef uint32_t type; };
template <> struct Vec<1> { typedef unsigned short type; };

template <int VEC>
__device__ __forceinline__ void unpack(const typename Vec<VEC>::type& u, float* f) {
  if constexpr (VEC == 8) {
    unpack8(u, f);
  } else {
    const bf16* p = reinterpret_cast<const bf16*>(&u);
#pragma unroll
    for (int i = 0; i < VEC; i++) f[i] = __bfloat162float(p[i]);
  }
}
template <int VEC>
__device__ __forceinline__ typename Vec<VEC>::type packed(const float* f) {
  if constexpr (VEC == 8) {
    return pack8(f);
  } else {
    typename Vec<VEC>::type u;
    bf16* p = reinterpret_cast<bf16*>(&u);
#pragma unroll
    for (int i = 0; i < VEC; i++) p[i] = __float2bfloat16(f[i]);
    return u;
  }
}

__device__ __forceinline__ long long id_at(const void* tok, int wide, long long t) {
  return wide ? reinterpret_cast<const long long*>(tok)[t] : (long long)reinterpret_cast<const int*>(tok)[t];
}

// A warp per token and slab of columns
template <int VEC>
__global__ void __launch_bounds__(256) embed_scaled_kernel(const void* __restrict__ tok, int wide, const bf16* __restrict__ w, bf16* __restrict__ out, int T, int H, long long v0, long long v1,
                                                           float scale) {
  grid_go();
  grid_wait();
  typedef typename Vec<VEC>::type V;
  constexpr int U = VEC == 8 ? 4 : 8;
  const int lane = threadIdx.x & 31, nvec = H / VEC;
  for (long long t = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); t < T; t += (long long)gridDim.x * 8) {
    const long long id = id_at(tok, wide, t);
    const bool in = id >= v0 && id < v1;
    const V* src = reinterpret_cast<const V*>(w + (in ? id - v0 : 0) * H);
    V* o = reinterpret_cast<V*>(out + t * H);
    for (int c = lane; c < nvec; c += 32 * U) {
      V a[U];
#pragma unroll
      for (int u = 0; u < U; u++)
        if (c + 32 * u < nvec && in) a[u] = src[c + 32 * u];
#pragma unroll
      for (int u = 0; u < U; u++)
        if (c + 32 * u < nvec) {
          float f[VEC];
#pragma unroll
          for (int i = 0; i < VEC; i++) f[i] = 0.f;
          if (in) {
            unpack<VEC>(a[u], f);
#pragma unroll
            for (int i = 0; i < VEC; i++) f[i] *= scale;
          }
          o[c + 32 * u] = packed<VEC>(f);
        }
    }
  }
}

// ---- order --------------------------------------------------------------------------------------
struct OrderParams {
  const void* tok;
  int wide, T, V;
  long long v0;
  int *ids, *place;              // [T] each: the tokens' rows in order, and their places
  int2 *a, *b;                   // [T] each: between the passes
  int passes, bits;              // of the radix sort
};
constexpr int ORDER_THREADS = 1024, ORDER_WARPS = ORDER_THREADS / 32;
// Row of token t; those outside, V, come behind all others.
__device__ __forceinline__ int row_of(const OrderParams& p, int t) {
  const long long id = id_at(p.tok, p.wide, t) - p.v0;
  return id >= 0 && id < p.V ? (int)id : p.V;
}

// Few tokens: each one's rank by comparison with all others, RANK_PARTS threads a token.
constexpr int RANK_MOST = 4096, RANK_PARTS = 16, RANK_TOKENS = ORDER_THREADS / RANK_PARTS;
__global__ void __launch_bounds__(ORDER_THREADS) embed_rank_kernel(const __grid_constant__ OrderParams p) {
  grid_go();
  grid_wait();
  __shared__ int s[RANK_MOST];
  for (int i = threadIdx.x; i < p.T; i += ORDER_THREADS) s[i] = row_of(p, i);
  __syncthreads();
  const int t = (int)blockIdx.x * RANK_TOKENS + (int)threadIdx.x / RANK_PARTS, part = threadIdx.x % RANK_PARTS;
  const int mine = t < p.T ? s[t] : 0;
  int rank = 0;
#pragma unroll 8
  for (int i = part; i < p.T; i += RANK_PARTS) rank += s[i] < mine || (s[i] == mine && i < t);
#pragma unroll
  for (int o = RANK_PARTS / 2; o > 0; o >>= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
  if (t < p.T && part == 0) {
    p.ids[rank] = mine;
    p.place[rank] = t;
  }
}

// Many: a radix sort by one cluster, which keeps the order of equals.  A warp has a share of the elements in their order; it counts their digits 32 at a time, the lowest lane of equal digits for all of
// them; counts of the warps ahead, then of the CTAs ahead and of the lower digits (through the cluster's shared memory), give every element its place.
constexpr int CLUSTER = 8, DIGITS = 1024;
struct RadixShared {
  uint32_t count[ORDER_WARPS][DIGITS];
  uint32_t total[DIGITS], base[DIGITS], of_warps[32];
};
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() { asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t peer_word(const uint32_t* at, uint32_t cta) {
  uint32_t a = (uint32_t)__cvta_generic_to_shared(at), v;
  asm volatile("mapa.shared::cluster.u32 %0, %0, %1;" : "+r"(a) : "r"(cta));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
// KEEP: at most so many elements of a lane, which stay in its registers; 0: any number, read twice a pass.
template <int KEEP>
__global__ void __launch_bounds__(ORDER_THREADS, 1) embed_radix_kernel(const __grid_constant__ OrderParams p) {
  extern __shared__ __align__(16) char radix_smem[];
  RadixShared& s = *reinterpret_cast<RadixShared*>(radix_smem);
  grid_go();
  grid_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, digits = 1 << p.bits;
  const uint32_t me = cluster_rank(), below = (1u << lane) - 1u;
  const long long per = (p.T + 32LL * CLUSTER * ORDER_WARPS - 1) / (32LL * CLUSTER * ORDER_WARPS) * 32;
  const long long first = ((long long)me * ORDER_WARPS + warp) * per, end = min((long long)p.T, first + per);
  for (int pass = 0; pass < p.passes; pass++) {
    const int shift = pass * p.bits;
    const int2* from = pass & 1 ? p.a : p.b;       // (pass 0 writes a)
    int2* to = pass & 1 ? p.b : p.a;
    auto load = [&](long long i) {
      if (i >= end) return make_int2(-1, 0);
      return pass == 0 ? make_int2(row_of(p, (int)i), (int)i) : __ldcg(from + i);
    };
    auto digit = [&](int2 x, long long i) { return i < end ? (x.x >> shift) & (digits - 1) : digits; };
    // rank of the lane's element among the warp's equal digits so far
    auto count = [&](int d) {
      const uint32_t same = __match_any_sync(0xffffffffu, d);
      uint32_t rank = 0;
      if (d < digits) rank = s.count[warp][d] + __popc(same & below);
      __syncwarp();
      if (d < digits && (same & below) == 0) s.count[warp][d] += __popc(same);
      __syncwarp();
      return rank;
    };
    auto put = [&](int2 x, uint32_t at) {
      if (pass + 1 < p.passes) {
        __stcg(to + at, x);
      } else {
        p.ids[at] = x.x;
        p.place[at] = x.y;
      }
    };
    [[maybe_unused]] int2 x[KEEP > 0 ? KEEP : 1];
    [[maybe_unused]] uint32_t rank[KEEP > 0 ? KEEP : 1];
    if constexpr (KEEP > 0) {
#pragma unroll
      for (int u = 0; u < KEEP; u++) x[u] = load(first + 32 * u + lane);
    }
    for (int i = threadIdx.x; i < ORDER_WARPS * digits; i += ORDER_THREADS) s.count[i >> p.bits][i & (digits - 1)] = 0;
    __syncthreads();
    if constexpr (KEEP > 0) {
#pragma unroll
      for (int u = 0; u < KEEP; u++)
        if (first + 32 * u < end) rank[u] = count(digit(x[u], first + 32 * u + lane));
    } else {
      for (long long i = first + lane; i - lane < end; i += 32) count(digit(load(i), i));
    }
    __syncthreads();
    const int d = threadIdx.x;
    if (d < digits) {
      uint32_t run = 0;
#pragma unroll 8
      for (int w = 0; w < ORDER_WARPS; w++) {
        const uint32_t c = s.count[w][d];
        s.count[w][d] = run;
        run += c;
      }
      s.total[d] = run;
    }
    cluster_sync();
    uint32_t ahead = 0, all = 0;
    if (d < digits) {
#pragma unroll
      for (uint32_t c = 0; c < CLUSTER; c++) {
        const uint32_t v = peer_word(&s.total[d], c);
        all += v;
        if (c < me) ahead += v;
      }
    }
    uint32_t sum = all;                            // of the lower digits
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += v;
    }
    if (lane == 31) s.of_warps[warp] = sum;
    __syncthreads();
    uint32_t w = s.of_warps[lane];
    w = lane < warp ? w : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
    if (d < digits) s.base[d] = sum - all + w + ahead;
    __syncthreads();
    if constexpr (KEEP > 0) {
#pragma unroll
      for (int u = 0; u < KEEP; u++) {
        const int dx = digit(x[u], first + 32 * u + lane);
        if (dx < digits) put(x[u], s.base[dx] + s.count[warp][dx] + rank[u]);
      }
    } else {
      for (long long i = first + lane; i - lane < end; i += 32) {
        const int2 e = load(i);
        const int dx = digit(e, i);
        const uint32_t at = count(dx);
        if (dx < digits) put(e, s.base[dx] + at);
      }
    }
    cluster_sync();                                // the elements are where the next pass reads them, and nobody reads totals any more
  }
}

// ---- sums ---------------------------------------------------------------------------------------
// The first CTAs take a chunk of the order and a slab of columns each.  A row is summed by the chunk that it begins in, where it ends in that or the next one; a longer one leaves what each chunk has of it,
// in 32 bits.  The other CTAs clear rows that have no token.
struct SumParams {
  const bf16* dy;
  bf16* dw;
  const int *ids, *place;        // [T] in order of id, then place
  float* parts;                  // [chunks][2][H]: of a longer row from the chunk before, and of one that begins here
  int T, H, V, chunk;
  float scale;
  unsigned sums, slabs;          // CTAs that sum, of a chunk
  int clear;                     // rows of a CTA that clears
};
constexpr int SUM_THREADS = 256, MAX_CHUNK = 64, MOST_CLEAR = 1024;

// First place in the order of row r or a later one: the warp looks in 32 places at a time.
__device__ __forceinline__ int first_of(const int* ids, int T, long long r) {
  const int lane = threadIdx.x & 31;
  int lo = 0, n = T;                               // it is in [lo, lo + n]
  while (n > 0) {
    const int step = (n + 31) / 32;
    const long long at = (long long)lo + (long long)(lane + 1) * step - 1;
    const bool less = at < (long long)lo + n && ids[at] < r;
    const int skip = __popc(__ballot_sync(0xffffffffu, less)) * step;
    lo += skip;
    n = min(step - 1, n - skip);
  }
  return lo;
}

template <int VEC>
__device__ __forceinline__ void clear_rows(const SumParams& p, int cta) {
  typedef typename Vec<VEC>::type V;
  __shared__ uint32_t marks[MOST_CLEAR / 32];      // rows that have tokens
  __shared__ int range[2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long begin = (long long)cta * p.clear, end = min((long long)p.V, begin + p.clear);
  if (threadIdx.x < MOST_CLEAR / 32) marks[threadIdx.x] = 0;
  if (warp < 2) {
    const int at = first_of(p.ids, p.T, warp ? end : begin);
    if (lane == 0) range[warp] = at;
  }
  __syncthreads();
  constexpr int U = 8;                             // (a row may come ten thousand times)
  for (int i = range[0] + (int)threadIdx.x; i < range[1]; i += U * SUM_THREADS) {
    int r[U], before[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int at = i + u * SUM_THREADS;
      r[u] = at < range[1] ? p.ids[at] : -1;
      before[u] = at < range[1] && at > range[0] ? p.ids[at - 1] : -1;
    }
#pragma unroll
    for (int u = 0; u < U; u++)
      if (r[u] != before[u]) atomicOr(&marks[(r[u] - (int)begin) >> 5], 1u << ((r[u] - (int)begin) & 31));
  }
  __syncthreads();
  for (int r = warp; r < (int)(end - begin); r += SUM_THREADS / 32) {
    if (marks[r >> 5] >> (r & 31) & 1u) continue;
    bf16* row = p.dw + (begin + r) * p.H;
    if constexpr (VEC == 1) {
      // (a row of any alignment: whole words between its ends)
      const int c = ((uintptr_t)row & 2) ? 1 : 0;
      if (c && lane == 0) row[0] = __float2bfloat16(0.f);
      for (int k = lane; k < (p.H - c) / 2; k += 32) *reinterpret_cast<uint32_t*>(row + c + 2 * k) = 0u;
      if ((p.H - c) % 2 && lane == 0) row[p.H - 1] = __float2bfloat16(0.f);
    } else {
      const float zeros[VEC] = {};
      for (int c = lane; c < p.H / VEC; c += 32) reinterpret_cast<V*>(row)[c] = packed<VEC>(zeros);
    }
  }
}

// A thread has K vectors of a row, a CTA's width apart; U places on their way.  (Rows of odd length are taken by single columns, 34 instructions each: 15001 x 1021 36 us.  By pairs from
// two words each, every second row being askew, loads no longer go out together: 46.)
template <int VEC, int K, int U>
__global__ void __launch_bounds__(SUM_THREADS, 3) embed_sum_kernel(const __grid_constant__ SumParams p) {
  grid_go();
  grid_wait();
  if (blockIdx.x >= p.sums) {
    clear_rows<VEC>(p, (int)(blockIdx.x - p.sums));
    return;
  }
  typedef typename Vec<VEC>::type V;
  __shared__ int ids[3 * MAX_CHUNK + 2], place[2 * MAX_CHUNK];      // of the chunk before (and one more), this and the next (and one more)
  const int slab = (int)(blockIdx.x % p.slabs), chunk = (int)(blockIdx.x / p.slabs);
  const long long first = (long long)chunk * p.chunk;
  const int C = p.chunk, n = (int)min((long long)C, p.T - first);
  for (int i = threadIdx.x; i < 3 * C + 2; i += SUM_THREADS) {
    const long long at = first + i - C - 1;
    ids[i] = at >= 0 && at < p.T ? p.ids[at] : -1;
    if (i < 2 * C && first + i < p.T) place[i] = p.place[first + i];
  }
  __syncthreads();
  const int* id_of = ids + C + 1;                  // of the chunk's places
  // The row that goes on from the chunk before: skipped, where that one sums it (it began there, and ends here).
  int begin = 0;
  bool from = chunk > 0 && id_of[-1] == id_of[0];
  if (from) {
    int end = 1;
    while (end < C + 1 && id_of[end] == id_of[0]) end++;
    if (end <= C && !(id_of[-C] == id_of[0] && id_of[-C - 1] == id_of[0])) {
      begin = end;
      from = false;
    }
  }
  // The row that goes on in the next chunk: all of it, where it began here and ends there.
  int stop = n;
  bool on = n == C && id_of[C] == id_of[C - 1] && begin < C;
  if (on && !(from && id_of[0] == id_of[C - 1])) {
    int end = C + 1;
    while (end < 2 * C + 1 && id_of[end] == id_of[C]) end++;
    if (end <= 2 * C) {
      stop = end;
      on = false;
    }
  }
  const int c0 = (slab * K * SUM_THREADS + (int)threadIdx.x) * VEC;
  constexpr int STEP = SUM_THREADS * VEC;
  float sum[K][VEC] = {};
  for (int i0 = begin; i0 < stop && id_of[i0] < p.V; i0 += U) {
    V a[U][K];
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int k = 0; k < K; k++)
        if (i0 + u < stop && c0 + k * STEP < p.H) a[u][k] = *reinterpret_cast<const V*>(p.dy + (long long)place[i0 + u] * p.H + c0 + k * STEP);
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int i = i0 + u;
      if (i >= stop) break;
      const int id = id_of[i];
#pragma unroll
      for (int k = 0; k < K; k++) {
        float f[VEC];
        unpack<VEC>(a[u][k], f);
#pragma unroll
        for (int v = 0; v < VEC; v++) sum[k][v] += f[v];
      }
      if (i + 1 < stop && id_of[i + 1] == id) continue;
      const bool whole = !from && !(i + 1 == stop && on);
#pragma unroll
      for (int k = 0; k < K; k++) {
        const int c = c0 + k * STEP;
        if (id < p.V && c < p.H) {
          if (whole) {
#pragma unroll
            for (int v = 0; v < VEC; v++) sum[k][v] *= p.scale;
            *reinterpret_cast<V*>(p.dw + (long long)id * p.H + c) = packed<VEC>(sum[k]);
          } else {
            float* to = p.parts + ((long long)chunk * 2 + (from ? 0 : 1)) * p.H + c;
#pragma unroll
            for (int v = 0; v < VEC; v++)
              to[v] = sum[k][v];
          }
        }
#pragma unroll
        for (int v = 0; v < VEC; v++) sum[k][v] = 0.f;
      }
      from = false;
    }
  }
}

// Rows of more than two chunks: every CTA looks for the chunks where one begins, and takes its share of (row, columns): JOIN_SLAB columns, JOIN_ROWS parts at a time.
constexpr int JOIN_COLS = 32, JOIN_ROWS = 16, JOIN_THREADS = JOIN_COLS * JOIN_ROWS, JOIN_K = 4, JOIN_SLAB = JOIN_COLS * JOIN_K;
__global__ void __launch_bounds__(JOIN_THREADS) embed_join_kernel(const __grid_constant__ SumParams p) {
  grid_go();
  grid_wait();
  __shared__ int2 list[JOIN_THREADS];              // chunk of the round where a row begins, and the row
  __shared__ long long ends[JOIN_THREADS];         // the last chunk that it goes on in
  __shared__ int found, heads[JOIN_THREADS];       // rows that the round's chunks begin with
  __shared__ float s[JOIN_ROWS][JOIN_SLAB];
  const int col = threadIdx.x % JOIN_COLS, r = threadIdx.x / JOIN_COLS, slabs = (p.H + JOIN_SLAB - 1) / JOIN_SLAB;
  const long long last = (p.T - 1LL) / p.chunk;    // chunk
  long long item = blockIdx.x;                     // of this CTA, counted over all rounds
  for (long long c0 = 0; c0 + 2 <= last; c0 += JOIN_THREADS) {
    const long long chunk = c0 + threadIdx.x;
    bool here = chunk + 2 <= last;
    heads[threadIdx.x] = chunk <= last ? p.ids[chunk * p.chunk] : -1;
    int id = 0;
    if (here) {
      const long long begin = chunk * p.chunk;
      id = p.ids[begin + p.chunk - 1];
      const int over = p.ids[begin + 2LL * p.chunk], head = p.ids[begin], before = begin > 0 ? p.ids[begin - 1] : -1;
      here = id < p.V && over == id && !(head == id && before == id);
    }
    // (in the order of the chunks: all CTAs have the same list)
    const uint32_t some = __ballot_sync(0xffffffffu, here);
    __shared__ int of_warps[JOIN_THREADS / 32];
    if ((threadIdx.x & 31) == 0) of_warps[threadIdx.x / 32] = __popc(some);
    __syncthreads();
    int at = __popc(some & ((1u << (threadIdx.x & 31)) - 1u));
    for (int w = 0; w < (int)threadIdx.x / 32; w++) at += of_warps[w];
    if (here) {
      long long lo = chunk + 2, hi = last;
      while (lo < hi) {                            // up to the last chunk that begins with the row
        const long long mid = (lo + hi + 1) / 2;
        if ((mid - c0 < JOIN_THREADS ? heads[mid - c0] : p.ids[mid * p.chunk]) == id) lo = mid; else hi = mid - 1;
      }
      list[at] = make_int2((int)threadIdx.x, id);
      ends[at] = lo;
    }
    if (threadIdx.x == JOIN_THREADS - 1) found = at + (here ? 1 : 0);
    __syncthreads();
    const long long items = (long long)found * slabs;
    for (; item < items; item += gridDim.x) {
      const int2 row = list[item / slabs];
      const long long first = c0 + row.x, end = ends[item / slabs];
      const int c = (int)(item % slabs) * JOIN_SLAB + col;
      float sum[JOIN_K] = {};
#pragma unroll
      for (int k = 0; k < JOIN_K; k++)
        if (r == 0 && c + k * JOIN_COLS < p.H) sum[k] = p.parts[(first * 2 + 1) * p.H + c + k * JOIN_COLS];
#pragma unroll 4
      for (long long part = first + 1 + r; part <= end; part += JOIN_ROWS)
#pragma unroll
        for (int k = 0; k < JOIN_K; k++)
          if (c + k * JOIN_COLS < p.H) sum[k] += p.parts[part * 2 * p.H + c + k * JOIN_COLS];
      __syncthreads();
#pragma unroll
      for (int k = 0; k < JOIN_K; k++) s[r][col + k * JOIN_COLS] = sum[k];
      __syncthreads();
      const int at = (int)(item % slabs) * JOIN_SLAB + (int)threadIdx.x;
      if (threadIdx.x < JOIN_SLAB && at < p.H) {
        float all = 0.f;
#pragma unroll
        for (int k = 0; k < JOIN_ROWS; k++) all += s[k][threadIdx.x];
        p.dw[(long long)row.y * p.H + at] = __float2bfloat16(all * p.scale);
      }
    }
    item -= items;
    __syncthreads();
  }
}

int vec_of(int H, uintptr_t at) { return H % 8 == 0 && at % 16 == 0 ? 8 : H % 2 == 0 && at % 4 == 0 ? 2 : 1; }
// Tokens of a chunk: three chunks per SM, as many as are resident, at least 8 tokens
int chunk_of(int T) {
  const int most = (T + 3 * lb_num_sms() - 1) / (3 * lb_num_sms());
  return most < 8 ? 8 : most > MAX_CHUNK ? MAX_CHUNK : most;
}
// Bits of a row or V, in passes of up to ten
int passes_of(int V, int& bits) {
  int all = 1;
  while ((long long)V >> all) all++;
  const int passes = (all + 9) / 10;
  bits = (all + passes - 1) / passes;
  return passes;
}
long long up(long long bytes) { return (bytes + 255) / 256 * 256; }
// (an attribute counts on the device where it was set)
int launch_order(void (*fn)(const OrderParams), bool* done, const OrderParams& o, cudaStream_t s) {
  constexpr int smem = (int)sizeof(RadixShared);
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return LB_ERR_LAUNCH;
  if (!done[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void*>(fn), cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) { cudaGetLastError(); g_lb_last_cuda_error = (int)e; return LB_ERR_LAUNCH; }
    done[dev] = true;
  }
  return lb_launch_cluster(true, CLUSTER, fn, CLUSTER, ORDER_THREADS, smem, s, o);
}
constexpr int KEPT = 4;                // elements of a lane in registers: up to 32768 tokens
constexpr long long CLEAR_BYTES = 65536;      // of a CTA that clears

// (columns are counted in 32 bits, in steps of up to 2048 past the last one)
constexpr int MOST_COLUMNS = 1 << 30;
int check_sizes(int T, int H, long long v0, long long v1) {
  return T <= 0 || T > (1 << 30) || H <= 0 || H > MOST_COLUMNS || v0 < 0 || v1 <= v0 || v1 - v0 > 0x7ffffffeLL ? LB_ERR_SHAPE : LB_OK;
}

}  // namespace

// y [T, H] = scale * w[tok - v0]; tok: id_bytes (4 or 8) each; w [v1 - v0, H].
extern "C" int lb_embed_scaled(const void* tok, int id_bytes, const void* w, void* y, int T, int H, long long v0, long long v1, float scale, void* stream) {
  if (check_sizes(T, H, v0, v1)) return LB_ERR_SHAPE;
  if (!tok || !w || !y || (id_bytes != 4 && id_bytes != 8)) return LB_ERR_ARG;
  const int most = lb_num_sms() * 16, blocks = (T + 7LL) / 8 < most ? (T + 7) / 8 : most;
#define LB_CALL(VEC) \
  LB_LAUNCH(embed_scaled_kernel<VEC>, blocks, 256, 0, (cudaStream_t)stream, tok, id_bytes == 8 ? 1 : 0, (const bf16*)w, (bf16*)y, T, H, v0, v1, scale)
  switch (vec_of(H, (uintptr_t)w | (uintptr_t)y)) {
    case 8: LB_CALL(8); break;
    case 2: LB_CALL(2); break;
    default: LB_CALL(1); break;
  }
#undef LB_CALL
  return LB_OK;
}

// Bytes of the backward's workspace; 0 for sizes that it does not take.
extern "C" long long lb_embed_sorted_ws_bytes(int T, int H) {
  if (check_sizes(T, H, 0, 1)) return 0;
  const int chunk = chunk_of(T);
  return 2 * up(4LL * T) + (T > RANK_MOST ? 2 * up(8LL * T) : 0) + up(((T + chunk - 1LL) / chunk) * 2 * H * 4);
}

// dw [v1 - v0, H] (all of it) from dy [T, H]; ws: lb_embed_sorted_ws_bytes(), 16-byte aligned, not initialised.
extern "C" int lb_embed_sorted_bwd(const void* tok, int id_bytes, const void* dy, void* dw, void* ws, long long ws_bytes, int T, int H, long long v0, long long v1, float scale, void* stream) {
  if (check_sizes(T, H, v0, v1)) return LB_ERR_SHAPE;
  if (!tok || !dy || !dw || !ws || (uintptr_t)ws & 15 || (id_bytes != 4 && id_bytes != 8)) return LB_ERR_ARG;
  if (ws_bytes < lb_embed_sorted_ws_bytes(T, H)) return LB_ERR_CAPACITY;
  cudaStream_t s = (cudaStream_t)stream;
  const int V = (int)(v1 - v0);
  if ((T / 8 + 1LL) * (H / SUM_THREADS + 1LL) + V / 8 + 1LL > 0x7fffffffLL) return LB_ERR_SHAPE;      // (more CTAs than a grid has)
  char* at = (char*)ws;
  OrderParams o{tok, id_bytes == 8 ? 1 : 0, T, V, v0, (int*)at, (int*)(at + up(4LL * T)), nullptr, nullptr, 0, 0};
  at += 2 * up(4LL * T);
  if (T <= RANK_MOST) {
    LB_LAUNCH(embed_rank_kernel, (T + RANK_TOKENS - 1) / RANK_TOKENS, ORDER_THREADS, 0, s, o);
  } else {
    o.a = (int2*)at;
    o.b = (int2*)(at + up(8LL * T));
    at += 2 * up(8LL * T);
    o.passes = passes_of(V, o.bits);
    static bool done[2][64] = {};
    const int rc = T <= KEPT * 32 * ORDER_WARPS * CLUSTER ? launch_order(embed_radix_kernel<KEPT>, done[0], o, s) : launch_order(embed_radix_kernel<0>, done[1], o, s);
    if (rc) return rc;
  }
  const int vec = vec_of(H, (uintptr_t)dy | (uintptr_t)dw);
  const int width = SUM_THREADS * (vec == 8 ? 8 : vec * 4);      // columns of a CTA
  SumParams p{(const bf16*)dy, (bf16*)dw, o.ids, o.place, (float*)at, T, H, V, chunk_of(T), scale, 0, 0, 0};
  const long long chunks = (T + p.chunk - 1LL) / p.chunk, rows = CLEAR_BYTES / (H * 2LL);
  p.slabs = (unsigned)((H + width - 1LL) / width);
  p.clear = (int)(rows < 8 ? 8 : rows > MOST_CLEAR ? MOST_CLEAR : rows);
  const long long sums = chunks * p.slabs, grid = sums + ((long long)V + p.clear - 1) / p.clear;
  p.sums = (unsigned)sums;
#define LB_CALL(VEC, K, U) LB_LAUNCH((embed_sum_kernel<VEC, K, U>), (unsigned)grid, SUM_THREADS, 0, s, p)
  switch (vec) {
    case 8: LB_CALL(8, 1, 8); break;
    case 2: LB_CALL(2, 4, 8); break;
    default: LB_CALL(1, 4, 8); break;
  }
#undef LB_CALL
  if (chunks > 2) LB_LAUNCH(embed_join_kernel, 2 * lb_num_sms(), JOIN_THREADS, 0, s, p);
  return LB_OK;
}
