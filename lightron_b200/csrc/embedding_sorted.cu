// Scaled embedding, and its gradient by sorted tokens:
//     y_t = scale * w[id_t]         dw[v] = scale * sum over the t with id_t = v, in their order, of dy_t
// The weight holds vocab ids [v0, v1); ids outside give zero rows and no gradient (vocab-parallel partial result).
//
// Forward: memory bound, rows of w in, rows of y out.
// Backward: the tokens are ordered by id, equal ids by their places (few by comparison, many by a radix sort of one cluster), while the other SMs clear the rows without tokens; then CTAs take runs of equal CHUNKs of that order: a row whose tokens lie inside one is summed in 32
// bits, scaled, rounded once and written; what a chunk has of a row that begins or ends in another goes to a place of its own in 32 bits, and a last kernel adds those up in the order of
// the chunks.  No atomics on values: the same bits in every run.  Bound by memory: every dy once, every row of dw once.
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
  constexpr int U = 4;
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
// One launch orders the tokens and meanwhile clears the rows of dw that have none: the first CTAs order, the others each have a share of the rows, find in all tokens which of them have
// one, and write zeros to the rest.
struct OrderParams {
  const void* tok;
  int wide, T, V, H;
  long long v0;
  int *ids, *place;              // [T] each: the tokens' rows in order, and their places
  int2 *a, *b;                   // [T] each: between the passes
  int passes, bits;              // of the radix sort
  bf16* dw;
  int order_ctas;
};
constexpr int ORDER_THREADS = 1024, ORDER_WARPS = ORDER_THREADS / 32;
// Row of token t; those outside, V, come behind all others.
__device__ __forceinline__ int row_of(const OrderParams& p, int t) {
  const long long id = id_at(p.tok, p.wide, t) - p.v0;
  return id >= 0 && id < p.V ? (int)id : p.V;
}

constexpr int FILL_WORDS = 4096;      // rows of a round: 32 of each word
__device__ __forceinline__ void clear_rows(const OrderParams& p, uint32_t* marks, int cta, int ctas) {
  const int per = (int)((p.V + (long long)ctas - 1) / ctas);
  const long long begin = (long long)cta * per, end = min((long long)p.V, begin + per);
  const int lane = threadIdx.x & 31;
  const bool wide = p.H % 8 == 0 && ((uintptr_t)p.dw & 15) == 0;
  for (long long r0 = begin; r0 < end; r0 += FILL_WORDS * 32) {
    const int n = (int)min((long long)FILL_WORDS * 32, end - r0);
    for (int i = threadIdx.x; i < (n + 31) / 32; i += ORDER_THREADS) marks[i] = 0;
    __syncthreads();
    constexpr int U = 8;
    for (long long t = threadIdx.x; t < p.T; t += U * ORDER_THREADS) {
      int r[U];
#pragma unroll
      for (int u = 0; u < U; u++) r[u] = t + u * ORDER_THREADS < p.T ? row_of(p, (int)(t + u * ORDER_THREADS)) : p.V;
#pragma unroll
      for (int u = 0; u < U; u++) {
        const long long at = r[u] - r0;
        // (looked at first: an id that comes ten thousand times is marked once)
        if (at >= 0 && at < n && !(reinterpret_cast<volatile uint32_t*>(marks)[at >> 5] >> (at & 31) & 1u)) atomicOr(&marks[at >> 5], 1u << (at & 31));
      }
    }
    __syncthreads();
    for (int r = threadIdx.x >> 5; r < n; r += ORDER_WARPS) {
      if (marks[r >> 5] >> (r & 31) & 1u) continue;
      bf16* row = p.dw + (r0 + r) * p.H;
      if (wide) {
        for (int c = lane; c < p.H / 8; c += 32) reinterpret_cast<uint4*>(row)[c] = make_uint4(0, 0, 0, 0);
      } else {
        // (a row of any alignment: whole words between its ends)
        int c = ((uintptr_t)row & 2) ? 1 : 0;
        if (c && lane == 0) row[0] = __float2bfloat16(0.f);
        for (int k = lane; k < (p.H - c) / 2; k += 32) *reinterpret_cast<uint32_t*>(row + c + 2 * k) = 0u;
        if ((p.H - c) % 2 && lane == 0) row[p.H - 1] = __float2bfloat16(0.f);
      }
    }
    __syncthreads();
  }
}

// Few tokens: each one's rank by comparison with all others, RANK_PARTS threads a token.
constexpr int RANK_MOST = 4096, RANK_PARTS = 16, RANK_TOKENS = ORDER_THREADS / RANK_PARTS;
__global__ void __launch_bounds__(ORDER_THREADS) embed_rank_kernel(const __grid_constant__ OrderParams p) {
  grid_go();
  grid_wait();
  __shared__ int s[RANK_MOST];                     // (of the rows that are cleared: which have tokens)
  if ((int)blockIdx.x >= p.order_ctas) {
    clear_rows(p, reinterpret_cast<uint32_t*>(s), (int)blockIdx.x - p.order_ctas, (int)gridDim.x - p.order_ctas);
    return;
  }
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
static_assert(FILL_WORDS <= RANK_MOST, "the marks take the place of the rows");

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
__global__ void __launch_bounds__(ORDER_THREADS, 1) embed_radix_kernel(const __grid_constant__ OrderParams p) {
  extern __shared__ __align__(16) char radix_smem[];
  RadixShared& s = *reinterpret_cast<RadixShared*>(radix_smem);
  grid_go();
  grid_wait();
  if ((int)blockIdx.x >= CLUSTER) {
    clear_rows(p, reinterpret_cast<uint32_t*>(radix_smem), (int)blockIdx.x - CLUSTER, (int)gridDim.x - CLUSTER);
    return;
  }
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
    for (int i = threadIdx.x; i < ORDER_WARPS * digits; i += ORDER_THREADS) s.count[i / digits][i % digits] = 0;
    __syncthreads();
    for (long long i0 = first; i0 < end; i0 += 32) {
      const long long i = i0 + lane;
      const int d = digit(load(i), i);
      const uint32_t same = __match_any_sync(0xffffffffu, d);
      if (d < digits && (same & below) == 0) s.count[warp][d] += __popc(same);
      __syncwarp();
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
      const uint32_t x = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += x;
    }
    if (lane == 31) s.of_warps[warp] = sum;
    __syncthreads();
    uint32_t w = s.of_warps[lane];
    w = lane < warp ? w : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
    if (d < digits) s.base[d] = sum - all + w + ahead;
    __syncthreads();
    for (long long i0 = first; i0 < end; i0 += 32) {
      const long long i = i0 + lane;
      const int2 x = load(i);
      const int dx = digit(x, i);
      const uint32_t same = __match_any_sync(0xffffffffu, dx);
      uint32_t at = 0;
      if (dx < digits) at = s.base[dx] + s.count[warp][dx] + __popc(same & below);
      __syncwarp();
      if (dx < digits) {
        if ((same & below) == 0) s.count[warp][dx] += __popc(same);
        if (pass + 1 < p.passes) {
          __stcg(to + at, x);
        } else {
          p.ids[at] = x.x;
          p.place[at] = x.y;
        }
      }
      __syncwarp();
    }
    cluster_sync();                                // the elements are where the next pass reads them, and nobody reads totals any more
  }
}

// ---- sums ---------------------------------------------------------------------------------------
struct SumParams {
  const bf16* dy;
  bf16* dw;
  const int *ids, *place;        // [T] in order of id, then place
  float* parts;                  // [chunks][2][H]: of the row that a chunk has from the one before it, and of the one that goes on in the next
  int T, H, V, chunk;
  float scale;
};
constexpr int SUM_THREADS = 256, MAX_CHUNK = 64;

template <int VEC>
__global__ void __launch_bounds__(SUM_THREADS) embed_sum_kernel(const SumParams p) {
  grid_go();
  grid_wait();
  typedef typename Vec<VEC>::type V;
  __shared__ int ids[MAX_CHUNK + 2], place[MAX_CHUNK];
  const long long first = (long long)blockIdx.x * p.chunk;
  const int n = (int)min((long long)p.chunk, p.T - first);
  for (int i = threadIdx.x; i < n + 2; i += SUM_THREADS) {
    const long long at = first + i - 1;
    ids[i] = at >= 0 && at < p.T ? p.ids[at] : -1;
    if (i < n) place[i] = p.place[first + i];
  }
  __syncthreads();
  const int c = (blockIdx.y * SUM_THREADS + threadIdx.x) * VEC;
  if (c >= p.H) return;
  constexpr int U = 8;
  float sum[VEC];
#pragma unroll
  for (int k = 0; k < VEC; k++) sum[k] = 0.f;
  int begin = 0;                                   // of the run
  for (int i0 = 0; i0 < n && ids[i0 + 1] < p.V; i0 += U) {
    V a[U];
#pragma unroll
    for (int u = 0; u < U; u++)
      if (i0 + u < n) a[u] = *reinterpret_cast<const V*>(p.dy + (long long)place[i0 + u] * p.H + c);
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int i = i0 + u;
      if (i >= n) break;
      const int id = ids[i + 1];
      float f[VEC];
      unpack<VEC>(a[u], f);
#pragma unroll
      for (int k = 0; k < VEC; k++) sum[k] += f[k];
      if (i + 1 < n && ids[i + 2] == id) continue;
      if (id < p.V) {
        const bool from = begin == 0 && ids[0] == id, on = ids[i + 2] == id;      // (on: at the chunk's end alone)
        if (!from && !on) {
#pragma unroll
          for (int k = 0; k < VEC; k++) sum[k] *= p.scale;
          *reinterpret_cast<V*>(p.dw + (long long)id * p.H + c) = packed<VEC>(sum);
        } else {
          float* to = p.parts + ((long long)blockIdx.x * 2 + (from ? 0 : 1)) * p.H + c;
#pragma unroll
          for (int k = 0; k < VEC; k++) to[k] = sum[k];
        }
      }
#pragma unroll
      for (int k = 0; k < VEC; k++) sum[k] = 0.f;
      begin = i + 1;
    }
  }
}

// Rows of several chunks: the CTA of the chunk where one begins adds up its parts.  32 columns, 8 parts at a time.
constexpr int JOIN_COLS = 32, JOIN_ROWS = 8;
__global__ void __launch_bounds__(JOIN_COLS* JOIN_ROWS) embed_join_kernel(const SumParams p) {
  grid_go();
  grid_wait();
  const long long next = ((long long)blockIdx.x + 1) * p.chunk;
  if (next >= p.T) return;
  const int id = p.ids[next - 1];
  if (id >= p.V || p.ids[next] != id) return;
  if (p.ids[next - p.chunk] == id && next > p.chunk && p.ids[next - p.chunk - 1] == id) return;      // (began in an earlier chunk)
  // chunks that the row goes on in: up to the last that begins with it
  long long lo = blockIdx.x + 1, hi = (p.T - 1LL) / p.chunk;
  while (lo < hi) {
    const long long mid = (lo + hi + 1) / 2;
    if (p.ids[mid * p.chunk] == id) lo = mid; else hi = mid - 1;
  }
  __shared__ float s[JOIN_ROWS][JOIN_COLS];
  const int c = blockIdx.y * JOIN_COLS + threadIdx.x;
  float sum = 0.f;
  if (c < p.H) {
    if (threadIdx.y == 0) sum = p.parts[((long long)blockIdx.x * 2 + 1) * p.H + c];
#pragma unroll 4
    for (long long k = blockIdx.x + 1 + threadIdx.y; k <= lo; k += JOIN_ROWS) sum += p.parts[k * 2 * p.H + c];
  }
  s[threadIdx.y][threadIdx.x] = sum;
  __syncthreads();
  if (threadIdx.y || c >= p.H) return;
  for (int r = 1; r < JOIN_ROWS; r++) sum += s[r][threadIdx.x];
  p.dw[(long long)id * p.H + c] = __float2bfloat16(sum * p.scale);
}

int vec_of(int H, uintptr_t at) { return H % 8 == 0 && at % 16 == 0 ? 8 : H % 2 == 0 && at % 4 == 0 ? 2 : 1; }
// Tokens of a chunk: four chunks per SM, at least 8 tokens
int chunk_of(int T) {
  const int most = (T + 4 * lb_num_sms() - 1) / (4 * lb_num_sms());
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
int check_sizes(int T, int H, long long v0, long long v1) { return T <= 0 || T > (1 << 30) || H <= 0 || v0 < 0 || v1 <= v0 || v1 - v0 > 0x7ffffffeLL ? LB_ERR_SHAPE : LB_OK; }

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
  char* at = (char*)ws;
  OrderParams o{tok, id_bytes == 8 ? 1 : 0, T, V, H, v0, (int*)at, (int*)(at + up(4LL * T)), nullptr, nullptr, 0, 0, (bf16*)dw, 0};
  at += 2 * up(4LL * T);
  // CTAs that clear: 64 KB of rows each at least
  const long long want = ((long long)V * H * 2 + 65535) / 65536, sms = lb_num_sms();
  if (T <= RANK_MOST) {
    o.order_ctas = (T + RANK_TOKENS - 1) / RANK_TOKENS;
    LB_LAUNCH(embed_rank_kernel, (unsigned)(o.order_ctas + (want < 2 * sms ? want : 2 * sms)), ORDER_THREADS, 0, s, o);
  } else {
    o.a = (int2*)at;
    o.b = (int2*)(at + up(8LL * T));
    at += 2 * up(8LL * T);
    o.passes = passes_of(V, o.bits);
    static bool done[64] = {false};      // (of a device: an attribute counts where it was set)
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return LB_ERR_LAUNCH;
    if (!done[dev]) {
      const cudaError_t e = cudaFuncSetAttribute(embed_radix_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(RadixShared));
      if (e != cudaSuccess) { cudaGetLastError(); g_lb_last_cuda_error = (int)e; return LB_ERR_LAUNCH; }
      done[dev] = true;
    }
    const long long fill = (want < sms ? want : sms) / CLUSTER, clusters = 1 + (fill < 1 ? 1 : fill);
    const int rc = lb_launch_cluster(true, CLUSTER, embed_radix_kernel, (unsigned)(clusters * CLUSTER), ORDER_THREADS, sizeof(RadixShared), s, o);
    if (rc) return rc;
  }
  SumParams p{(const bf16*)dy, (bf16*)dw, o.ids, o.place, (float*)at, T, H, V, chunk_of(T), scale};
  const unsigned chunks = (unsigned)((T + p.chunk - 1LL) / p.chunk);
  const int vec = vec_of(H, (uintptr_t)dy | (uintptr_t)dw);
  const unsigned slabs = (unsigned)((H + SUM_THREADS * vec - 1) / (SUM_THREADS * vec));
  if (slabs > 65535 || (H + JOIN_COLS - 1) / JOIN_COLS > 65535) return LB_ERR_SHAPE;
#define LB_CALL(VEC) LB_LAUNCH(embed_sum_kernel<VEC>, dim3(chunks, slabs), SUM_THREADS, 0, s, p)
  switch (vec) {
    case 8: LB_CALL(8); break;
    case 2: LB_CALL(2); break;
    default: LB_CALL(1); break;
  }
#undef LB_CALL
  if (chunks > 1) LB_LAUNCH(embed_join_kernel, dim3(chunks - 1, (unsigned)((H + JOIN_COLS - 1) / JOIN_COLS)), dim3(JOIN_COLS, JOIN_ROWS), 0, s, p);
  return LB_OK;
}
