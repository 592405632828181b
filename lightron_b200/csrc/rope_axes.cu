// Rotary positions with several axes (time, height, width): pair i of every head of a token turns by the angle that belongs to the token's position on
// axis(i).  Reads x and writes y once; the tables of cosines and sines stay in L2.  Memory bound: 16384 tokens, 36 heads of 64 5.8 TB/s of 6.5 that a copy reaches; a thread per
// vector that looked up its own angles took 54 us.
#include "common.cuh"

namespace {

constexpr int MAX_AXES = 8, MAX_PAIRS = 128;
struct RopeAxesParams {
  const bf16* x;
  bf16* y;
  const float *cosT, *sinT;
  const int* positions;          // [axes, B, S], or [axes, S] with pos_b = 0
  long long xb, xs, xh, yb, ys, yh, pos_a, pos_b;
  int B, S, h, d, rows, inverse;
  int share;                     // heads of a warp
  unsigned char axis[MAX_PAIRS];
};

// A warp takes one token's heads [h0, h0 + share), a lane the same 8 columns of every G-th of them: the angles of its four pairs are looked up once, and
// AHEAD vectors of x are on their way before the first position has come (4 / 8 / 12 of them: 16384 tokens, 36 heads of 64 26.1 / 30.8 / 26.9 us, 8192 tokens, 40 heads of 128
// 30.6 / 32.0 / 30.6: fewer registers and more warps do as well as more loads each).
constexpr int AHEAD = 4;
__global__ void __launch_bounds__(256) rope_axes_kernel(const __grid_constant__ RopeAxesParams p) {
  grid_go();
  grid_wait();
  const int vecs = p.d >> 3, G = 32 / vecs, lane = threadIdx.x & 31, mine = lane / vecs, v = lane - mine * vecs;
  const long long tok = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (tok >= (long long)p.B * p.S || mine >= G) return;
  const int b = (int)(tok / p.S), s = (int)(tok - (long long)b * p.S);
  const int h0 = (int)blockIdx.y * p.share, h1 = min(p.h, h0 + p.share);
  const bf16* x = p.x + b * p.xb + s * p.xs + v * 8;
  bf16* y = p.y + b * p.yb + s * p.ys + v * 8;
  uint4 a[AHEAD];
  auto load = [&](int h) {
#pragma unroll
    for (int i = 0; i < AHEAD; i++)
      if (h + i * G < h1) a[i] = __ldcs(reinterpret_cast<const uint4*>(x + (h + i * G) * p.xh));
  };
  load(h0 + mine);
  float cs[8];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int pos = p.positions[p.axis[v * 4 + i] * p.pos_a + b * p.pos_b + s];
    const bool there = (unsigned)pos < (unsigned)p.rows;      // (a position outside the table gives NaN, no access)
    const long long at = (long long)pos * (p.d >> 1) + v * 4 + i;
    cs[i] = there ? p.cosT[at] : __int_as_float(0x7fffffff);
    cs[4 + i] = there ? p.sinT[at] : __int_as_float(0x7fffffff);
  }
  for (int h = h0 + mine; h < h1; h += AHEAD * G) {
    if (h != h0 + mine) load(h);
#pragma unroll
    for (int i = 0; i < AHEAD; i++)
      if (h + i * G < h1) {
        float f[8];
        unpack8(a[i], f);
        rope_rotate8(cs, f, p.inverse != 0);
        *reinterpret_cast<uint4*>(y + (h + i * G) * p.yh) = pack8(f);
      }
  }
}

}  // namespace

// y = x [B, S, h, d] turned (back, with inverse).  strides: {batch, token, head} of x, then of y, in elements, multiples of 8, innermost contiguous; y may be x; cos, sin fp32 [rows, d / 2];
// positions int32, axis a of token (b, s) at a * pos_a + b * pos_b + s; axes: host bytes, the axis (0 to n_axes - 1) of each of the d / 2 pairs.
extern "C" int lb_rope_axes(const void* x, void* y, const void* cosT, const void* sinT, const void* positions, const unsigned char* axes, int n_axes, int B, int S, int h, int d,
                            int rows, const long long* strides, long long pos_a, long long pos_b, int inverse, void* stream) {
  if (B <= 0 || S <= 0 || h <= 0 || rows <= 0 || d <= 0 || d % 8 || d > 2 * MAX_PAIRS || n_axes <= 0 || n_axes > MAX_AXES) return LB_ERR_SHAPE;
  if (!x || !y || !cosT || !sinT || !positions || !axes || !strides || ((uintptr_t)x | (uintptr_t)y) & 15) return LB_ERR_ARG;
  for (int i = 0; i < 6; i++)
    if (strides[i] % 8) return LB_ERR_SHAPE;
  RopeAxesParams p{(const bf16*)x, (bf16*)y, (const float*)cosT, (const float*)sinT, (const int*)positions, strides[0], strides[1], strides[2], strides[3], strides[4], strides[5], pos_a, pos_b, B, S, h, d, rows, inverse, h, {}};
  for (int i = 0; i < d / 2; i++) {
    if (axes[i] >= n_axes) return LB_ERR_ARG;
    p.axis[i] = axes[i];
  }
  // all heads of a token by one warp, or by several where there are few tokens: at least one round of loads each, eight warps per SM (1 and 20 tokens, 40 heads of 128, as a graph, one warp /
  // several, us: 6.2 / 4.1; 300 and 1000 tokens 6.2 in both)
  const long long tokens = (long long)B * S, blocks = (tokens + 7) / 8;
  if (blocks > 2147483647LL) return LB_ERR_SHAPE;
  const int round = 32 / (d / 8) * AHEAD, most = (h + round - 1) / round;
  const long long want = (8LL * lb_num_sms() + tokens - 1) / tokens;
  const int parts = (int)(want < most ? want : most);
  p.share = (h + parts - 1) / parts;
  LB_LAUNCH(rope_axes_kernel, dim3((unsigned)blocks, (unsigned)((h + p.share - 1) / p.share)), 256, 0, (cudaStream_t)stream, p);
  return LB_OK;
}
