// Global norm of many tensors, and their scaling by it.
//
//     norm = sqrt(sum over all tensors of sum g^2)        g * min(1, max_norm / (norm + eps))
//
// Both are memory bound: the sum reads every element once, the scaling reads it again and writes it.  The tensors' addresses travel as
// kernel parameters, so that a call uploads nothing and can be captured.  Every tensor is cut into chunks of CHUNK elements, chunk c belongs to CTA
// c % grid, and a CTA leaves the fp32 sum of its squares in a place of its own; whoever needs the total adds those up in 64 bits, in their order: the
// norm is the same bits in every run.  The scaling goes through the chunks backwards: what the sum has read last is still in L2.
// 1.1 B bf16 elements, 201 tensors, clipped into another buffer: 1140 us (6.6 GB in all three passes, 5.8 TB/s of 6.5 that a copy reaches), the norm alone 366; 134 M in 111 tensors 145 us.
#include <cuda_fp16.h>
#include "common.cuh"

namespace {

// (Lists of few tensors in fewer parameters: clipping 38 of them, alone on the GPU, 38 -> 35 us.)
constexpr int THREADS = 256, MAX_TENSORS = 768, FEW_TENSORS = 96, CHUNK = 16384;
enum : int { BF16 = 0, FP16 = 1, FP32 = 2 };

template <int N>
struct Tensors {
  int n, chunks;
  const void* src[N];
  void* dst[N];
  long long count[N];
  int first[N];                                // chunks ahead of a tensor's, with its type in the upper two bits
};
static_assert(sizeof(Tensors<MAX_TENSORS>) <= 32000 && sizeof(Tensors<FEW_TENSORS>) <= 4000, "kernel parameters: 32 KB, or 4 KB");

__device__ __forceinline__ float to_f(bf16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(float x) { return x; }
template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ bf16 from_f<bf16>(float x) { return __float2bfloat16(x); }
template <> __device__ __forceinline__ __half from_f<__half>(float x) { return __float2half(x); }
template <> __device__ __forceinline__ float from_f<float>(float x) { return x; }

// Sum over the CTA, in the same order in every run; to thread 0.
__device__ __forceinline__ float block_sum(float s) {
  __shared__ float sh[THREADS / 32];
  s = warp_sum(s);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = s;
  __syncthreads();
  float t = 0.f;
  if (threadIdx.x == 0)
    for (int i = 0; i < THREADS / 32; i++) t += sh[i];
  return t;
}

// The chunk's tensor: the last whose first chunk is not behind it (empty tensors have none and are never the last).
template <int N>
__device__ __forceinline__ int tensor_of(const Tensors<N>& t, int chunk) {
  int lo = 0, hi = t.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if ((t.first[mid] & 0x3fffffff) <= chunk) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// Elements of a 16-byte vector.
template <typename T>
__device__ __forceinline__ void spread(const uint4& u, float* f) {
  const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
  for (int i = 0; i < 16 / (int)sizeof(T); i++) f[i] = to_f(e[i]);
}

// Elements ahead of the first one at a 16-byte boundary.
template <typename T>
__device__ __forceinline__ int ahead_of_16(const T* x, int n) { return min(n, (int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(T)); }

template <typename T>
__device__ __forceinline__ float chunk_squares(const T* x, int n) {
  constexpr int E = 16 / (int)sizeof(T), U = 8;      // U vectors of a thread on their way
  const int lead = ahead_of_16(x, n), vecs = (n - lead) / E;
  const uint4* v = reinterpret_cast<const uint4*>(x + lead);
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  for (int i0 = 0; i0 < vecs; i0 += U * THREADS) {
    uint4 a[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int i = i0 + u * THREADS + (int)threadIdx.x;
      a[u] = i < vecs ? v[i] : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      float f[E];
      spread<T>(a[u], f);
#pragma unroll
      for (int k = 0; k < E; k++) s[k & 3] += f[k] * f[k];
    }
  }
  // (up to 7 elements ahead of the vectors and 7 behind them)
  const int rest = lead + vecs * E, i = (int)threadIdx.x < lead ? (int)threadIdx.x : rest + (int)threadIdx.x - lead;
  if (i < n && (i < lead || i >= rest)) { const float f = to_f(x[i]); s[0] += f * f; }
  return (s[0] + s[1]) + (s[2] + s[3]);
}

template <int N>
__global__ void __launch_bounds__(THREADS) grad_squares_kernel(const __grid_constant__ Tensors<N> t, float* __restrict__ partial) {
  grid_go();
  grid_wait();
  float s = 0.f;
  for (int c = blockIdx.x; c < t.chunks; c += gridDim.x) {
    const int k = tensor_of(t, c), type = (unsigned)t.first[k] >> 30;
    const long long at = (long long)(c - (t.first[k] & 0x3fffffff)) * CHUNK;
    const int n = (int)min((long long)CHUNK, t.count[k] - at);
    s += type == FP32 ? chunk_squares((const float*)t.src[k] + at, n) : type == BF16 ? chunk_squares((const bf16*)t.src[k] + at, n) : chunk_squares((const __half*)t.src[k] + at, n);
  }
  s = block_sum(s);
  if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

// Sum of the parts in 64 bits, in an order of its own; to all threads.
__device__ __forceinline__ double total_of(const float* partial, int n) {
  __shared__ double sh[THREADS / 32];
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += THREADS) s += (double)partial[i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = s;
  __syncthreads();
  s = 0.0;
#pragma unroll
  for (int i = 0; i < THREADS / 32; i++) s += sh[i];
  return s;
}

__global__ void __launch_bounds__(THREADS) grad_total_kernel(const float* __restrict__ partial, int n, float* __restrict__ sumsq, float* __restrict__ norm) {
  grid_go();
  grid_wait();
  const double s = total_of(partial, n);
  if (threadIdx.x == 0) {
    if (sumsq) *sumsq = (float)s;
    if (norm) *norm = (float)sqrt(s);
  }
}

template <typename T>
__device__ __forceinline__ uint4 scaled(const uint4& a, float by) {
  uint4 r;
  const T* e = reinterpret_cast<const T*>(&a);
  T* o = reinterpret_cast<T*>(&r);
#pragma unroll
  for (int i = 0; i < 16 / (int)sizeof(T); i++) o[i] = from_f<T>(to_f(e[i]) * by);
  return r;
}

// 16 bytes that start `words` words and `bits` bits into two neighbouring vectors.
template <int WORDS>
__device__ __forceinline__ uint4 cut(const uint4& a, const uint4& b, int bits) {
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  return make_uint4(__funnelshift_r(w[WORDS], w[WORDS + 1], bits), __funnelshift_r(w[WORDS + 1], w[WORDS + 2], bits), __funnelshift_r(w[WORDS + 2], w[WORDS + 3], bits),
                    __funnelshift_r(w[WORDS + 3], w[(WORDS + 4) & 7], bits));
}

// Stores are whole vectors of y.  Where x has another offset from a 16-byte boundary, a vector is cut out of the two of x that hold it: each of them has an element of
// the chunk, so neither is outside the memory that holds it.  (Norm and clipping of 4 x 2048 x 2048 bf16: 17.3 us aligned,
// 18.4 to 18.7 at other offsets.)
template <typename T>
__device__ __forceinline__ void chunk_scale(const T* x, T* y, int n, float by) {
  constexpr int E = 16 / (int)sizeof(T), U = 4;
  const int lead = ahead_of_16(y, n), vecs = (n - lead) / E, skew = (int)((uintptr_t)(x + lead) & 15);
  const uint4* v = reinterpret_cast<const uint4*>((uintptr_t)(x + lead) - skew);
  uint4* o = reinterpret_cast<uint4*>(y + lead);
  for (int i0 = 0; i0 < vecs; i0 += U * THREADS) {
    uint4 a[U], b[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int i = i0 + u * THREADS + (int)threadIdx.x;
      if (i < vecs) {
        a[u] = v[i];
        if (skew) b[u] = v[i + 1];
      }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int i = i0 + u * THREADS + (int)threadIdx.x;
      if (i >= vecs) continue;
      if (skew) {
        const int bits = (skew & 3) * 8;
        switch (skew >> 2) {
          case 0: a[u] = cut<0>(a[u], b[u], bits); break;
          case 1: a[u] = cut<1>(a[u], b[u], bits); break;
          case 2: a[u] = cut<2>(a[u], b[u], bits); break;
          default: a[u] = cut<3>(a[u], b[u], bits); break;
        }
      }
      __stcs(o + i, scaled<T>(a[u], by));
    }
  }
  const int rest = lead + vecs * E, i = (int)threadIdx.x < lead ? (int)threadIdx.x : rest + (int)threadIdx.x - lead;
  if (i < n && (i < lead || i >= rest)) y[i] = from_f<T>(to_f(x[i]) * by);
}

template <int N>
__global__ void __launch_bounds__(THREADS) grad_scale_kernel(const __grid_constant__ Tensors<N> t, const float* __restrict__ partial, int n_partial, float max_norm, float eps,
                                                             float* __restrict__ norm_out) {
  grid_go();
  grid_wait();
  const float norm = (float)sqrt(total_of(partial, n_partial));
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = norm;
  const float r = max_norm / (norm + eps), by = r > 1.f ? 1.f : r;       // (a NaN stays one)
  // (from the last chunk back: what the sum has read last is still in L2)
  for (int c = t.chunks - 1 - (int)blockIdx.x; c >= 0; c -= gridDim.x) {
    const int k = tensor_of(t, c), type = (unsigned)t.first[k] >> 30;
    if (by == 1.f && t.src[k] == t.dst[k]) continue;
    const long long at = (long long)(c - (t.first[k] & 0x3fffffff)) * CHUNK;
    const int n = (int)min((long long)CHUNK, t.count[k] - at);
    if (type == FP32) chunk_scale((const float*)t.src[k] + at, (float*)t.dst[k] + at, n, by);
    else if (type == BF16) chunk_scale((const bf16*)t.src[k] + at, (bf16*)t.dst[k] + at, n, by);
    else chunk_scale((const __half*)t.src[k] + at, (__half*)t.dst[k] + at, n, by);
  }
}

int grid_of(int chunks) { const int most = lb_num_sms() * 8; return chunks < most ? chunks : most; }

// The next tensors of a list, up to what one launch takes; `at` moves on.
template <int N>
int next_tensors(Tensors<N>& t, int n, int& at, const void* const* src, void* const* dst, const long long* counts, const int* types) {
  t.n = t.chunks = 0;
  for (; at < n && t.n < N; at++) {
    if (counts[at] < 0 || (counts[at] && (!src[at] || (dst && !dst[at]))) || types[at] < BF16 || types[at] > FP32) return LB_ERR_ARG;
    const long long chunks = (counts[at] + CHUNK - 1) / CHUNK;
    if (!chunks) continue;
    if (t.chunks + chunks >= (1LL << 30)) {
      if (!t.n) return LB_ERR_SHAPE;
      break;
    }
    t.src[t.n] = src[at];
    t.dst[t.n] = dst ? dst[at] : nullptr;
    t.count[t.n] = counts[at];
    t.first[t.n++] = (int)((unsigned)t.chunks | (unsigned)types[at] << 30);
    t.chunks += (int)chunks;
  }
  return LB_OK;
}

template <int N>
int squares(int n, const void* const* src, const long long* counts, const int* types, float* partial, int partials, int* filled, cudaStream_t s) {
  static thread_local Tensors<N> t;
  for (int at = 0; at < n;) {
    if (const int rc = next_tensors(t, n, at, src, nullptr, counts, types)) return rc;
    if (!t.n) break;
    const int grid = grid_of(t.chunks);
    if (*filled + grid > partials) return LB_ERR_CAPACITY;
    LB_LAUNCH(grad_squares_kernel<N>, grid, THREADS, 0, s, t, partial + *filled);
    *filled += grid;
  }
  return LB_OK;
}

template <int N>
int scale(int n, const void* const* src, void* const* dst, const long long* counts, const int* types, const float* partial, int n_partial, float max_norm, float eps, float*& norm_out,
          cudaStream_t s) {
  static thread_local Tensors<N> t;
  for (int at = 0; at < n;) {
    if (const int rc = next_tensors(t, n, at, src, dst, counts, types)) return rc;
    if (!t.n) break;
    LB_LAUNCH(grad_scale_kernel<N>, grid_of(t.chunks), THREADS, 0, s, t, partial, n_partial, max_norm, eps, norm_out);
    norm_out = nullptr;
  }
  return LB_OK;
}

}  // namespace

// Floats of `partial` that lb_grad_squares() of n tensors may fill.
extern "C" int lb_grad_norm_parts(int n) { return n < 0 ? LB_ERR_ARG : (n / MAX_TENSORS + 1) * lb_num_sms() * 8; }

// partial[0 .. *filled): sums of squares of parts of the n tensors (host arrays of device addresses, element counts and types: 0 bf16, 1 fp16, 2 fp32).
extern "C" int lb_grad_squares(int n, const void* const* src, const long long* counts, const int* types, void* partial, int partials, int* filled, void* stream) {
  if (n < 0 || !partial || !filled || (n && (!src || !counts || !types))) return LB_ERR_ARG;
  *filled = 0;
  cudaStream_t s = (cudaStream_t)stream;
  return n <= FEW_TENSORS ? squares<FEW_TENSORS>(n, src, counts, types, (float*)partial, partials, filled, s)
                          : squares<MAX_TENSORS>(n, src, counts, types, (float*)partial, partials, filled, s);
}

// Total of n parts: its fp32 value and its root (either may be null).
extern "C" int lb_grad_total(const void* partial, int n, void* sumsq, void* norm, void* stream) {
  if (n < 0 || !partial) return LB_ERR_ARG;
  LB_LAUNCH(grad_total_kernel, 1, THREADS, 0, (cudaStream_t)stream, (const float*)partial, n, (float*)sumsq, (float*)norm);
  return LB_OK;
}

// dst = src * min(1, max_norm / (norm + eps)), norm the root of the total of the parts, also written to norm_out (null: not).  dst may be src, whose elements are
// then left alone where the factor is 1.
extern "C" int lb_grad_scale(int n, const void* const* src, void* const* dst, const long long* counts, const int* types, const void* partial, int n_partial, float max_norm,
                             float eps, void* norm_out, void* stream) {
  if (n < 0 || n_partial < 0 || !partial || (n && (!src || !dst || !counts || !types))) return LB_ERR_ARG;
  float* norm = (float*)norm_out;
  cudaStream_t s = (cudaStream_t)stream;
  if (const int rc = n <= FEW_TENSORS ? scale<FEW_TENSORS>(n, src, dst, counts, types, (const float*)partial, n_partial, max_norm, eps, norm, s)
                                      : scale<MAX_TENSORS>(n, src, dst, counts, types, (const float*)partial, n_partial, max_norm, eps, norm, s))
    return rc;
  if (norm) return lb_grad_total(partial, n_partial, nullptr, norm, stream);      // (nothing to scale)
  return LB_OK;
}
