// Scaled embedding, and its gradient by sorted tokens:
//     y_t = scale * w[id_t]         dw[v] = scale * sum over the t with id_t = v, in their order, of dy_t
// The weight holds vocab ids [v0, v1); ids outside give zero rows and no gradient (vocab-parallel partial result).
//
// Forward: memory bound, rows of w in, rows of y out.
// Backward: the tokens are ordered by id (and by place among equal ids), then CTAs take runs of equal CHUNKs of that order: a row whose tokens lie inside one is summed in 32
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
// Rank of every token by comparison with all others.
constexpr int RANK_THREADS = 256, RANK_TILE = 2048;
__global__ void __launch_bounds__(RANK_THREADS) embed_rank_kernel(const void* __restrict__ tok, int wide, int T, long long v0, int V, int* __restrict__ ids, int* __restrict__ place) {
  grid_go();
  grid_wait();
  __shared__ int s[RANK_TILE];
  const int t = blockIdx.x * RANK_THREADS + threadIdx.x;
  auto key = [&](int i) {
    const long long id = id_at(tok, wide, i) - v0;
    return id >= 0 && id < V ? (int)id : V;          // (those outside: behind all rows)
  };
  const int mine = t < T ? key(t) : 0;
  int rank = 0;
  for (int at = 0; at < T; at += RANK_TILE) {
    __syncthreads();
    const int n = min(RANK_TILE, T - at);
    for (int i = threadIdx.x; i < n; i += RANK_THREADS) s[i] = key(at + i);
    __syncthreads();
#pragma unroll 8
    for (int i = 0; i < n; i++) rank += s[i] < mine || (s[i] == mine && at + i < t);
  }
  if (t < T) {
    ids[rank] = mine;
    place[rank] = t;
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
  return 2 * up(4LL * T) + ((T + chunk - 1LL) / chunk) * 2 * H * 4;
}

// dw [v1 - v0, H] (all of it) from dy [T, H]; ws: lb_embed_sorted_ws_bytes(), 16-byte aligned, not initialised.
extern "C" int lb_embed_sorted_bwd(const void* tok, int id_bytes, const void* dy, void* dw, void* ws, long long ws_bytes, int T, int H, long long v0, long long v1, float scale, void* stream) {
  if (check_sizes(T, H, v0, v1)) return LB_ERR_SHAPE;
  if (!tok || !dy || !dw || !ws || (uintptr_t)ws & 15 || (id_bytes != 4 && id_bytes != 8)) return LB_ERR_ARG;
  if (ws_bytes < lb_embed_sorted_ws_bytes(T, H)) return LB_ERR_CAPACITY;
  cudaStream_t s = (cudaStream_t)stream;
  const int V = (int)(v1 - v0);
  cudaError_t e = cudaMemsetAsync(dw, 0, (size_t)V * H * 2, s);
  if (e != cudaSuccess) { g_lb_last_cuda_error = (int)e; return LB_ERR_LAUNCH; }
  char* at = (char*)ws;
  int* ids = (int*)at;
  int* place = (int*)(at + up(4LL * T));
  SumParams p{(const bf16*)dy, (bf16*)dw, ids, place, (float*)(at + 2 * up(4LL * T)), T, H, V, chunk_of(T), scale};
  LB_LAUNCH(embed_rank_kernel, (T + RANK_THREADS - 1) / RANK_THREADS, RANK_THREADS, 0, s, tok, id_bytes == 8 ? 1 : 0, T, v0, V, ids, place);
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
