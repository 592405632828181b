// Rotary positions with several axes (time, height, width): pair i of every head of a token turns by the angle that belongs to the token's position on
// axis(i).  Reads x and writes y once; the tables of cosines and sines stay in L2.
#include "common.cuh"

namespace {

constexpr int MAX_AXES = 8, MAX_PAIRS = 128;
struct RopeAxesParams {
  const bf16* x;
  bf16* y;
  const float *cosT, *sinT;
  const int* positions;          // [axes, B, S], or [axes, S] with pos_b = 0
  long long xb, xs, xh, pos_a, pos_b;
  int B, S, h, d, rows, inverse;
  unsigned char axis[MAX_PAIRS];
};

__global__ void rope_axes_kernel(const __grid_constant__ RopeAxesParams p) {
  grid_go();
  grid_wait();
  const int vecs = p.d >> 3;
  const long long total = (long long)p.B * p.S * p.h * vecs;
  for (long long idx = (long long)blockIdx.x * blockDim.x + threadIdx.x; idx < total; idx += (long long)gridDim.x * blockDim.x) {
    const int v = (int)(idx % vecs);
    const long long th = idx / vecs;
    const int h = (int)(th % p.h), s = (int)(th / p.h % p.S), b = (int)(th / p.h / p.S);
    float f[8], cs[8];
    unpack8(*reinterpret_cast<const uint4*>(p.x + b * p.xb + s * p.xs + h * p.xh + v * 8), f);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int pos = p.positions[p.axis[v * 4 + i] * p.pos_a + b * p.pos_b + s];
      const bool there = (unsigned)pos < (unsigned)p.rows;      // (a position outside the table gives NaN, no access)
      const long long at = (long long)pos * (p.d >> 1) + v * 4 + i;
      cs[i] = there ? p.cosT[at] : __int_as_float(0x7fffffff);
      cs[4 + i] = there ? p.sinT[at] : __int_as_float(0x7fffffff);
    }
    rope_rotate8(cs, f, p.inverse != 0);
    *reinterpret_cast<uint4*>(p.y + idx * 8) = pack8(f);
  }
}

}  // namespace

// y [B, S, h, d] = x turned (back, with inverse).  x: strides {batch, token, head} in elements, multiples of 8, innermost contiguous; cos, sin fp32 [rows, d / 2];
// positions int32, axis a of token (b, s) at a * pos_a + b * pos_b + s; axes: host bytes, the axis (0 to n_axes - 1) of each of the d / 2 pairs.
extern "C" int lb_rope_axes(const void* x, void* y, const void* cosT, const void* sinT, const void* positions, const unsigned char* axes, int n_axes, int B, int S, int h, int d,
                            int rows, const long long* strides, long long pos_a, long long pos_b, int inverse, void* stream) {
  if (B <= 0 || S <= 0 || h <= 0 || rows <= 0 || d <= 0 || d % 8 || d > 2 * MAX_PAIRS || n_axes <= 0 || n_axes > MAX_AXES) return LB_ERR_SHAPE;
  if (!x || !y || !cosT || !sinT || !positions || !axes || !strides || ((uintptr_t)x | (uintptr_t)y | (uintptr_t)cosT | (uintptr_t)sinT) & 15) return LB_ERR_ARG;
  if ((strides[0] | strides[1] | strides[2]) % 8) return LB_ERR_SHAPE;
  RopeAxesParams p{(const bf16*)x, (bf16*)y, (const float*)cosT, (const float*)sinT, (const int*)positions, strides[0], strides[1], strides[2], pos_a, pos_b, B, S, h, d, rows, inverse, {}};
  for (int i = 0; i < d / 2; i++) {
    if (axes[i] >= n_axes) return LB_ERR_ARG;
    p.axis[i] = axes[i];
  }
  const long long total = (long long)B * S * h * (d / 8), blocks = (total + 255) / 256, cap = lb_num_sms() * 16;
  LB_LAUNCH(rope_axes_kernel, (unsigned)(blocks < cap ? blocks : cap), 256, 0, (cudaStream_t)stream, p);
  return LB_OK;
}
