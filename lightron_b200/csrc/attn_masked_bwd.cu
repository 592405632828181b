// Backward of attention under interval masks (attn_masked.cuh) on the 5th-generation tensor cores, head_dim up to 128 (a multiple of 8, in tiles
// of 64 or 128 columns).
//
//     P_ij = exp(s_ij - lse_i)     D_i = do_i . o_i     dS_ij = scale * P_ij (dP_ij - D_i) (1 - tanh^2)     dP = dO V^T
//     dV = P^T dO                  dK = dS^T Q          dQ = dS K
//
// A CTA owns a block of 128 keys of one (batch, kv head) and walks over the 128-query blocks, of every query head of the group, that see any of
// them: from the first query of its first key to the last of its last.  Scores are computed transposed, keys in the lanes, so that P^T and dS^T go back to tensor memory
// as the A operands of dV and dK and only dS also goes to shared memory, for dQ; dQ tiles are drained by warps of their own and added in fp32 by bulk
// reductions.  That is the pipeline of the causal backward (flash_bwd_tcgen05.cu has what each part of it is worth).  What is different here: the
// query range of a key block and the rows that a key's lane keeps come from the intervals; cap and bias are made as in the forward, two queries at a time, and
// the cap's derivative is folded into P once P^T has left; D is made of o and what its rounding left.
// Where key blocks are few, the walk of each is cut into `parts` equal shares, a CTA each, which leave dK and dV in fp32 in places of their own; the kernel
// that converts dQ adds them in their order.  dK and dV are the same bits in every run; dQ is up to 128 keys, where one CTA makes all of it and
// writes it.
// What bounds it.  d 64: a block takes 2890 cycles, most of them the math warps' (tensor pipe 44 %, exponentials 36 % of the active cycles), and a CTA's fixed part is some 6 blocks, a fifth
// of a walk of documents of 300 tokens.  d 128: 4300 cycles, the chain dS - dK, dQ - drain - dP; with a cap the math warps again (5100; tensor pipe 50 %).  All kernels, us: 8 x 2048, 32 / 4 heads, d 64
// causal 505, bias 525, cap 660, documents of 300 288; 1 x 8192, 32 / 8 heads, d 128 causal 1400 to 1450, bias 1340 to 1390, cap 1605 to 1630.
// Under a window a key block's walk is short, but a block of sinks is seen by all queries behind it: 256 query blocks instead of 38 at 1 x 8192, window 1024, 32 / 8 heads.  Where they would
// leave the others waiting, walks are then cut into pieces of a length that is chosen here and listed on the device, longest first, where the lengths are known (documents cut them); pieces of one block
// leave dK and dV in fp32 in places of their own, as parts do.  Main kernel, whole / cut: that case, 4 sinks, d 128 647 / 385 to 400 us; 3 x 1531, window 333, 130 sinks, cap 30, 16 / 4 heads, d 96
// 128 / 74 to 82.  What bounds it is what bounds the others, the block's chain and a CTA's fixed part.
// Warp roles (512 threads): warp 0 TMA producer, warp 1 MMA issuer + TMEM owner, warps 4-11 math, 12-15 dQ drain.
// P^T and dS^T are rounded to bf16, the type of Q, K and dO, as operands of the tensor cores: 1.7e-3 of a gradient in the 2-norm beside the 1.7e-3 of its own rounding; all sums are fp32.
// All waits are bounded; on expiry a status word is set and the CTA drains and frees its TMEM.
#include <algorithm>
#include <climits>
#include <type_traits>
#include "attn_masked.cuh"
#include "tcgen05.cuh"

static __device__ unsigned int g_mab_status[4] = {0, 0, 0, 0};

namespace {
using namespace bw;

constexpr float LOG2E = 1.4426950408889634f;

struct BwdParams {
  MaBwdParams w;
  float *dq_acc, *dk_acc, *dv_acc;
  int* order;                    // null, or the key blocks (sequence * blocks + block) in the order of their CTAs
  int parts;                     // CTAs of a key block
  // LIST: pieces of the key blocks' walks {key block, first, length, place of its sums or -1}, longest first; of every key block {place of the first, pieces that leave sums}
  int4* items;
  int2* joined;
  int *n_items, *cut_blocks;     // {how many pieces, how many key blocks in several, how many pieces come first}, and those
  int chunk, extra, sums;        // longest piece wanted, pieces beyond one per key block that there is room for, and pieces that leave sums
  int ordinary, lead;            // LIST: pieces longer than this come first, of all heads, then the others head by head; of `order`: how many key blocks come so
  int acc_d;                     // columns of dq_acc: head_dim in whole pieces of 32
  MaTerms f;
  f32x2 scale2;                  // the scale, twice
};

// Entry and head of a CTA: the first `lead` entries of a list for all heads, longest first, then the others head by head.
__device__ __forceinline__ int2 entry_and_head(int cta, int grid, int heads, int lead) {
  if (cta < lead * heads) return make_int2(cta / heads, cta % heads);
  const int rest = cta - lead * heads, each = grid / heads - lead;
  return make_int2(lead + rest % each, rest / each);
}

// (batch, kv head) pairs whose key blocks are ordered together: enough to keep the chip busy to the end, few enough that several key blocks of a pair run
// at a time and share its Q / dO / dQ traffic in L2.
constexpr int GROUP = 32;

template <int D>
struct Cfg {
  static constexpr int BM = 128, BN = 128;
  // Q stays until dK of its block, one block longer than S needs it; dO is released by dV, before dP of the next block needs the next one.
  static constexpr int QS = (D == 64) ? 3 : 2;
  static constexpr int DS = (D == 64) ? 3 : 1;
  static constexpr bool DQ_ALIAS = (D == 128);          // dQ takes the dP columns
  static constexpr int ATOMS = D / 64;
  static constexpr int ATOM_BYTES = 128 * 128;
  static constexpr int TILE_BYTES = ATOMS * ATOM_BYTES;
  static constexpr int OFF_K = 0;
  static constexpr int OFF_V = OFF_K + TILE_BYTES;
  static constexpr int OFF_Q = OFF_V + TILE_BYTES;              // [QS]
  static constexpr int OFF_DO = OFF_Q + QS * TILE_BYTES;        // [DS]
  static constexpr int OFF_DS = OFF_DO + DS * TILE_BYTES;
  static constexpr int STG_BYTES = 32 * 32 * 4;                 // one 32 x 32 chunk of dQ; two per drain warp
  static constexpr int OFF_STG = OFF_DS + 2 * ATOM_BYTES;
  static constexpr int OFF_ST = OFF_STG + 8 * STG_BYTES;        // [QS] row statistics of a query block
  static constexpr int OFF_BAR = OFF_ST + QS * 1024;
  static constexpr int SMEM = OFF_BAR + 256;
  static constexpr int NBAR = 1 + 2 * QS + 2 * DS + 6;
  static constexpr int NTHREADS = 512;
  // Registers per thread: loads and MMAs / math / drain, which holds a whole row of dQ so that its columns are free at once.
  static constexpr int REGS_ISSUE = 96, REGS_MATH = (D == 64) ? 160 : 128, REGS_DRAIN = (D == 64) ? 96 : 160;
  static_assert(REGS_ISSUE + 2 * REGS_MATH + REGS_DRAIN <= 4 * 128, "a CTA has 512 x 128 registers");
  // TMEM columns
  static constexpr int COL_S = 0, COL_DP = 128, COL_DV = 256, COL_DK = 256 + D;
  static constexpr int COL_DQ = DQ_ALIAS ? COL_DP : 384;
};
static_assert(Cfg<128>::SMEM <= 232448, "shared memory of a CTA");

// What a CTA leaves: WHOLE dK and dV of a key block, and its share of dQ, added to the fp32 sums; PARTS that, and its share of dK and dV; ALONE all three; LIST, under a window, dK and dV or its share
// of them: sinks are seen by all queries of their document, many times those of other keys, and such walks are cut.
enum : int { WHOLE, PARTS, ALONE, LIST };

// Query blocks of one head that see a key block: [x, y).
__device__ __forceinline__ int2 query_blocks(const MaParams& p, int b, int n0, bool alone) {
  if (alone) return make_int2(0, (p.Sq + 127) / 128);      // (all are written)
  const int lo = ma_queries(p, b, n0).x, last = min(n0 + 128, p.Sk) - 1;
  // (the first key's queries begin first, the last one's end last; but where the last one's document has sinks in the block, all of the document sees those)
  const bool sinks = p.window && ma_start(p, b, last) + p.sinks > n0;
  const int hi = min((sinks ? ma_queries_all(p, b, last) : ma_queries(p, b, last)).y, p.Sq);
  return hi > lo ? make_int2(lo / 128, (hi + 127) / 128) : make_int2(0, 0);
}

// Row statistics, one 1 KB record per (b, h, 128-query block): 128 x -lse * log2(e), then 128 x -scale * D.  Rows without a sum, and rows past Sq, get (-inf, 0), which
// makes their P and dS zero.  Also clears dQ's accumulator.  D/8 threads per (token, head).
// With `order`, the first CTA instead sorts the key blocks by the query blocks that see them, most first, for the longest walks to begin first whatever the documents are
// (walks of more than MOST blocks count as equal).  Against the order of a causal mask, main kernel: 8 x 2048, documents of 300, 32 / 4 heads, d 64 199 -> 188 us; 3 x 1531 of
// 500, 32 / 8 heads, d 128 95 -> 86.
constexpr int MOST = 1023;

// Entries ahead of each size: count[i + 1] holds how many have size i.
__device__ __forceinline__ void count_ahead(int* count) {
  if (threadIdx.x < 32) {
    int run = 0;
    for (int k = 0; k < MOST + 2; k += 32) {
      const int i = k + (int)threadIdx.x;
      int v = i < MOST + 2 ? count[i] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, v, o);
        if ((int)threadIdx.x >= o) v += x;
      }
      if (i < MOST + 2) count[i] = run + v;
      run += __shfl_sync(0xffffffffu, v, 31);
    }
  }
}

// One CTA lists the pieces of all walks.  Which of equal pieces comes first is left open; what they are is not.
__device__ void list_pieces(const BwdParams& pp, int* count) {
  const MaParams& p = pp.w.f;
  constexpr int KEPT = 2048;                                   // walks that are looked up once
  __shared__ int of_warps[32], kept[KEPT], n_cut;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, rep = p.hq / p.hkv;
  const int n_nblk = (p.Sk + 127) / 128, n = p.B * n_nblk;
  auto walk_of = [&](int e) {
    const int2 mb = query_blocks(p, e / n_nblk, (e % n_nblk) * 128, false);
    return (mb.y - mb.x) * rep;
  };
  for (int e = threadIdx.x; e < min(n, KEPT); e += blockDim.x) kept[e] = walk_of(e);
  if (threadIdx.x == 0) n_cut = 0;
  __syncthreads();
  auto walk = [&](int e) { return e < KEPT ? kept[e] : walk_of(e); };
  // of all threads; in `before`: of those before this one
  auto sum_of = [&](int v, int& before) {
    int run = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += x;
    }
    __syncthreads();
    if (lane == 31) of_warps[warp] = run;
    __syncthreads();
    int all = 0, ahead = 0;
    for (int w = 0; w < warps; w++) {
      if (w == warp) ahead = all;
      all += of_warps[w];
    }
    before = ahead + run - v;
    return all;
  };
  const int per = (n + (int)blockDim.x - 1) / (int)blockDim.x, a = min(n, (int)threadIdx.x * per), end = min(n, a + per);
  // pieces twice as long until there is room for all, and for the sums that they leave
  int length = pp.chunk, beyond = 0, before = 0;               // before: place of this thread's first sums
  for (;; length *= 2) {
    int more = 0, sums = 0;
    for (int e = a; e < end; e++) {
      const int of_walk = max((walk(e) + length - 1) / length - 1, 0);
      more += of_walk;
      if (of_walk) sums += of_walk + 1;
    }
    beyond = sum_of(more, before);
    if (beyond <= pp.extra && sum_of(sums, before) <= pp.sums) break;
  }
  auto cut = [&](int e, int& its, int& pieces, int& share) {
    its = walk(e);
    pieces = max((its + length - 1) / length, 1);
    share = (its + pieces - 1) / pieces;
  };
  auto bucket = [&](int size) { return MOST - min(size, MOST); };
  for (int i = threadIdx.x; i < MOST + 2; i += blockDim.x) count[i] = 0;
  __syncthreads();
  int its, pieces, share;
  for (int e = a; e < end; e++) {
    cut(e, its, pieces, share);
    if (pieces > 1) atomicAdd(&count[bucket(share) + 1], pieces - 1);
    atomicAdd(&count[bucket(its - (pieces - 1) * share) + 1], 1);
  }
  __syncthreads();
  count_ahead(count);
  __syncthreads();
  const int lead = count[bucket(pp.ordinary)];                 // (pieces longer than that are in the buckets ahead)
  __syncthreads();
  for (int e = a; e < end; e++) {
    cut(e, its, pieces, share);
    if (pieces > 1) {
      const int at = atomicAdd(&count[bucket(share)], pieces - 1);
      for (int k = 0; k + 1 < pieces; k++) pp.items[at + k] = make_int4(e, k * share, share, before + k);
    }
    pp.items[atomicAdd(&count[bucket(its - (pieces - 1) * share)], 1)] = make_int4(e, (pieces - 1) * share, its - (pieces - 1) * share, pieces > 1 ? before + pieces - 1 : -1);
    pp.joined[e] = make_int2(before, pieces > 1 ? pieces : 0);
    if (pieces > 1) {
      before += pieces;
      pp.cut_blocks[atomicAdd(&n_cut, 1)] = e;
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    pp.n_items[0] = n + beyond;
    pp.n_items[1] = n_cut;
    pp.n_items[2] = lead;
  }
}

// LISTED: the first CTA lists the pieces (its registers spill: with as many as it would like, 60 for 32, the others, which are memory's, took 66 us instead of 52 at 1 x 8192, 32 heads, d 128).
template <int D, bool LISTED>
__global__ void __launch_bounds__(256, LISTED ? 8 : 1) ma_bwd_prep_kernel(const __grid_constant__ BwdParams pp, const int clear) {
  grid_go();
  grid_wait();
  const MaParams& p = pp.w.f;
  const int planners = LISTED || pp.order ? 1 : 0, workers = (int)gridDim.x - planners;
  if ((int)blockIdx.x < planners) {                            // (the first: what it does is a chain)
    __shared__ int count[MOST + 2];
    if constexpr (LISTED) {
      list_pieces(pp, count);
      return;
    }
    const int n_nblk = (p.Sk + 127) / 128, n = p.B * n_nblk;
    auto size = [&](int e) {
      const int2 mb = query_blocks(p, e / n_nblk, (e % n_nblk) * 128, false);
      return MOST - min(mb.y - mb.x, MOST);                    // ascending: most first
    };
    for (int i = threadIdx.x; i < MOST + 2; i += blockDim.x) count[i] = 0;
    __syncthreads();
    for (int e = threadIdx.x; e < n; e += blockDim.x) atomicAdd(&count[size(e) + 1], 1);
    __syncthreads();
    count_ahead(count);
    __syncthreads();
    for (int e = threadIdx.x; e < n; e += blockDim.x) pp.order[atomicAdd(&count[size(e)], 1)] = e;
    return;
  }
  constexpr int TPR = D / 8;                                   // threads per row: 8 or 16
  const int n_mblocks = (p.Sq + 127) / 128, Sp = n_mblocks * 128;
  const long long total = (long long)p.B * Sp * p.hq;
  const int rpb = blockDim.x / TPR;                            // rows per block and iteration
  const int sub = threadIdx.x % TPR;
  // every thread of the block runs the same number of iterations, so the shuffles see whole warps
  for (long long base = (long long)((int)blockIdx.x - planners) * rpb; base < total; base += (long long)workers * rpb) {
    const long long idx = base + threadIdx.x / TPR;
    const bool live = idx < total;
    float s = 0.f;
    int h = 0, b = 0, i = 0;
    if (live) {
      h = (int)(idx % p.hq);
      const long long bi = idx / p.hq;
      b = (int)(bi / Sp);
      i = (int)(bi % Sp);
      if (clear && sub * 8 < pp.acc_d) {
        float4* z = reinterpret_cast<float4*>(pp.dq_acc + idx * pp.acc_d + sub * 8);
        z[0] = make_float4(0.f, 0.f, 0.f, 0.f);
        z[1] = make_float4(0.f, 0.f, 0.f, 0.f);
      }
      if (i < p.Sq && sub * 8 < p.d) {
        const long long at = (((long long)b * p.Sq + i) * p.hq + h) * p.d + sub * 8;
        float a[8], r[8], e[8];
        unpack8(*reinterpret_cast<const uint4*>(p.o + at), a);
        unpack8(*reinterpret_cast<const uint4*>(p.o_lo + at), r);
        unpack8(*reinterpret_cast<const uint4*>(pp.w.dout + b * pp.w.dos.b + i * pp.w.dos.s + h * pp.w.dos.h + sub * 8), e);
#pragma unroll
        for (int k = 0; k < 8; k++) s += (a[k] + r[k]) * e[k];
      }
    }
#pragma unroll
    for (int o = TPR / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);   // whole warps stay converged
    if (live && sub == 0) {
      float* rec = pp.w.stats + (((long long)b * p.hq + h) * n_mblocks + (i >> 7)) * 256 + (i & 127);
      const float lse = i < p.Sq ? p.lse[((long long)b * p.hq + h) * p.Sq + i] : -INFINITY;
      rec[0] = lse == -INFINITY ? -INFINITY : -lse * LOG2E;
      rec[128] = lse == -INFINITY ? 0.f : -s * p.scale;
    }
  }
}

// fp32 accumulator layout: dQ tile (b, h, block of 128 rows), or dK / dV tile of a part -> 4 row quads -> acc_d / 4 (D / 4) pieces of 4 columns -> 32 rows: the 16-byte stores of a
// drain warp (a row per lane) are contiguous.  A thread converts 8 columns of four rows of dQ, or adds the parts of 8 columns of a row of dK or dV.
template <int D, bool CUT>
__global__ void ma_convert_kernel(const __grid_constant__ BwdParams pp) {
  grid_go();
  grid_wait();
  const MaParams& p = pp.w.f;
  const long long threads = (long long)gridDim.x * blockDim.x;
  long long start = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  const int n_mblocks = (p.Sq + 127) / 128;
  if constexpr (CUT) {
    const int lane = threadIdx.x & 31;
    constexpr int G = D / 8;
    const int n_nblk = (p.Sk + 127) / 128, rep = p.hq / p.hkv, pairs = p.hkv * p.B;
    const long long pieces = (pp.items ? 2LL * p.hkv * pp.n_items[1] : 2LL * pairs * n_nblk) * 4 * G;
    for (; start < 32 * pieces; start += threads) {            // (dK or dV, key block, pair, quad, 8 columns)
      const long long w = start >> 5;
      const int g = (int)(w % G), quad = (int)((w / G) & 3);
      const long long tile = w / (4 * G);
      int pair = (int)(tile % pairs), block = (int)((tile / pairs) % n_nblk), dv = (int)(tile / pairs / n_nblk);
      if (pp.items) {
        const long long of = tile / p.hkv;                     // (key blocks in several pieces alone)
        const int e = pp.cut_blocks[of >> 1];
        dv = (int)(of & 1);
        block = e % n_nblk;
        pair = e / n_nblk * p.hkv + (int)(tile % p.hkv);
      }
      const int b = pair / p.hkv;
      const int row = block * 128 + quad * 32 + lane;
      if (row >= p.Sk || g * 8 >= p.d) continue;
      int used;
      long long first, apart = 1;                              // place of the first part, and from one to the next
      if (pp.items) {
        const int2 j = pp.joined[b * n_nblk + block];
        used = j.y;
        apart = p.hkv;
        first = (long long)j.x * p.hkv + pair % p.hkv;
      } else {
        const int2 mb = query_blocks(p, b, block * 128, false);
        const int its = (mb.y - mb.x) * rep, share = (its + pp.parts - 1) / pp.parts;
        used = share ? (its + share - 1) / share : 0;
        first = ((long long)block * pairs + pair) * pp.parts;
      }
      const float4* from = reinterpret_cast<const float4*>(dv ? pp.dv_acc : pp.dk_acc) + first * (32 * D) + (quad * (D / 4) + 2 * g) * 32 + lane;
      float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      for (int part = 0; part < used; part += 4) {
        float4 x[4][2];
#pragma unroll
        for (int u = 0; u < 4; u++)
          if (part + u < used) { x[u][0] = from[(part + u) * apart * (32 * D)]; x[u][1] = from[(part + u) * apart * (32 * D) + 32]; }
#pragma unroll
        for (int u = 0; u < 4; u++)
          if (part + u < used) {
#pragma unroll
            for (int k = 0; k < 2; k++) { f[4 * k] += x[u][k].x; f[4 * k + 1] += x[u][k].y; f[4 * k + 2] += x[u][k].z; f[4 * k + 3] += x[u][k].w; }
          }
      }
      const MaStrides& st = dv ? pp.w.dvs : pp.w.dks;
      *reinterpret_cast<uint4*>((dv ? pp.w.dv : pp.w.dk) + b * st.b + row * st.s + (pair % p.hkv) * st.h + g * 8) = pack8(f);
    }
    start -= 32 * pieces;                                      // dQ's pieces come next
  }
  // A warp takes RW rows at a time, whole: its stores are whole lines, its loads 16 bytes of RW neighbouring rows, all of four rounds in flight.  (A lane per row with 32
  // columns, contiguous loads but stores of 16 bytes in 32 rows: 8 x 2048, 32 heads, d 64 54 us.)
  constexpr int TPR = D / 8, RW = 32 / TPR, UNITS = 128 / (4 * RW);
  const int lane = threadIdx.x & 31, c = lane % TPR, sub = lane / TPR;
  const long long total = (long long)p.B * p.hq * n_mblocks * UNITS;
  for (long long w = start >> 5; w < total; w += threads >> 5) {
    const long long tile = w / UNITS;
    const int first = (int)(w % UNITS) * 4 * RW + sub;          // row of the tile
    const int mblock = (int)(tile % n_mblocks), h = (int)(tile / n_mblocks % p.hq), b = (int)(tile / n_mblocks / p.hq);
    const float4* at = reinterpret_cast<const float4*>(pp.dq_acc) + tile * (32 * pp.acc_d) + 2 * c * 32;
    float4 x[4][2];
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const int r = first + k * RW;
      if (mblock * 128 + r < p.Sq && c * 8 < p.d) {
        const float4* a = at + (r >> 5) * (8 * pp.acc_d) + (r & 31);
        x[k][0] = __ldcs(a);
        x[k][1] = __ldcs(a + 32);
      }
    }
    bf16* o = pp.w.dq + b * pp.w.dqs.b + h * pp.w.dqs.h + c * 8;
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const int row = mblock * 128 + first + k * RW;
      if (row < p.Sq && c * 8 < p.d) *reinterpret_cast<uint4*>(o + row * pp.w.dqs.s) = pack8(reinterpret_cast<const float*>(x[k]));
    }
  }
}

template <int D, int FORM, bool CAP, bool BIAS>
__global__ void __launch_bounds__(512, 1)
ma_bwd_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, const __grid_constant__ CUtensorMap tdo,
              const __grid_constant__ CUtensorMap tdk, const __grid_constant__ CUtensorMap tdv, const __grid_constant__ BwdParams pp) {
  using C = Cfg<D>;
  const MaParams& p = pp.w.f;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + C::NBAR);
  int* s_abort = reinterpret_cast<int*>(tmem_slot + 1);     // {abort, extra wait in ms}: see bw::mbar_wait

  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;   // (uniform over the warp)
  const uint32_t sbase = smem_u32(smem);
  if (sbase & 1023u) {                                       // the swizzled tiles need it; nothing has been started yet
    if (threadIdx.x == 0) atomicExch(&g_mab_status[0], 4u);
    return;
  }
  const uint32_t bar0 = smem_u32(bars);
  const uint32_t kv_full = bar0;
  auto q_full = [&](int s) { return bar0 + 8u * (1 + s); };
  auto q_empty = [&](int s) { return bar0 + 8u * (1 + C::QS + s); };
  auto do_full = [&](int s) { return bar0 + 8u * (1 + 2 * C::QS + s); };
  auto do_empty = [&](int s) { return bar0 + 8u * (1 + 2 * C::QS + C::DS + s); };
  const uint32_t bar1 = bar0 + 8u * (1 + 2 * C::QS + 2 * C::DS);
  const uint32_t s_full = bar1, dp_full = bar1 + 8, p_full = bar1 + 16, ds_full = bar1 + 24, dq_full = bar1 + 32, dq_free = bar1 + 40;

  // The first key blocks of all (batch, kv head) pairs of a group first: under a causal mask they take longest (with documents: in the order that has been
  // found).  In parts: those of the first key block of all pairs, then the next.
  const int n_nblk = (p.Sk + C::BN - 1) / C::BN;
  int nblk, pair, part = 0;
  if constexpr (FORM == PARTS) {
    const int pairs = p.hkv * p.B, t = (int)blockIdx.x / pp.parts;
    part = (int)blockIdx.x % pp.parts;
    pair = t % pairs;
    nblk = t / pairs;
  } else {
    // (under a window all walks are as long, and a pair's share most when they run together)
    const int group = p.window ? 1 : GROUP;
    const int grp = (int)blockIdx.x / (n_nblk * group);
    const int in_grp = (int)blockIdx.x - grp * n_nblk * group;
    const int gsize = min(group, p.hkv * p.B - grp * group);
    nblk = in_grp / gsize;
    pair = grp * group + in_grp % gsize;
  }
  const int off = p.Sk - p.Sq;
  const int rep = p.hq / p.hkv;
  const int n_mblocks = (p.Sq + C::BM - 1) / C::BM;

  if (threadIdx.x == 0) {
    s_abort[0] = s_abort[1] = 0;
    mbar_init(kv_full, 1);
    for (int s = 0; s < C::QS; s++) { mbar_init(q_full(s), 1); mbar_init(q_empty(s), 1); }
    for (int s = 0; s < C::DS; s++) { mbar_init(do_full(s), 1); mbar_init(do_empty(s), 1); }
    mbar_init(s_full, 1);
    mbar_init(dp_full, 1);
    mbar_init(p_full, 8);
    mbar_init(ds_full, 8);
    mbar_init(dq_full, 1);
    mbar_init(dq_free, 4);
    mbar_init_fence();
    prefetch_tmap(&tq); prefetch_tmap(&tk); prefetch_tmap(&tv); prefetch_tmap(&tdo); prefetch_tmap(&tdk); prefetch_tmap(&tdv);
  }
  if (warp == 1) tmem_alloc(smem_u32(tmem_slot), 512);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  volatile int* abort_flag = s_abort;
  grid_wait();

  [[maybe_unused]] int4 piece = make_int4(0, 0, 0, 0);          // (a CTA without one leaves nothing)
  if constexpr (FORM == LIST) {
    const int2 at = entry_and_head((int)blockIdx.x, (int)gridDim.x, p.hkv, pp.n_items[2]);
    if (at.x < pp.n_items[0]) piece = pp.items[at.x];
    nblk = piece.x % n_nblk;
    pair = piece.x / n_nblk * p.hkv + at.y;
  }
  if (FORM == WHOLE && pp.order) {
    const int2 at = entry_and_head((int)blockIdx.x, (int)gridDim.x, p.hkv, pp.lead);
    const int e = pp.order[at.x];
    nblk = e % n_nblk;
    pair = e / n_nblk * p.hkv + at.y;
  }
  const int hk = pair % p.hkv, b = pair / p.hkv;
  const int n0 = nblk * C::BN;
  // query blocks of every head of the group, head by head; a part takes an equal share of them
  const int2 seen_by = query_blocks(p, b, n0, FORM == ALONE);
  const int mb_first = seen_by.x, mb_end = seen_by.y, per_head = mb_end - mb_first;
  int total_it = per_head * rep, it_first = 0;
  if constexpr (FORM == PARTS) {
    const int share = (total_it + pp.parts - 1) / pp.parts;
    it_first = min(total_it, part * share);
    total_it = min(share, total_it - it_first);
  }
  if constexpr (FORM == LIST) {
    it_first = piece.y;
    total_it = piece.z;
  }
  constexpr bool CUT = FORM == PARTS || FORM == LIST;
  const int h_first = hk * rep + (CUT && total_it ? it_first / per_head : 0);
  const int mb_start = mb_first + (CUT && total_it ? it_first % per_head : 0);
  const bool leaves_sums = FORM == PARTS || (FORM == LIST && piece.w >= 0);

  if (warp < 4) reg_dec<C::REGS_ISSUE>();
  if (warp == 0) {
    // ------------------------------- TMA producer -------------------------------
    if (total_it > 0 && elect_one()) {
      mbar_expect_tx(kv_full, 2 * C::TILE_BYTES);
#pragma unroll
      for (int a = 0; a < C::ATOMS; a++) {
        tma_load_4d(sbase + C::OFF_K + a * C::ATOM_BYTES, &tk, a * 64, hk, n0, b, kv_full);
        tma_load_4d(sbase + C::OFF_V + a * C::ATOM_BYTES, &tv, a * 64, hk, n0, b, kv_full);
      }
      bool ok = true;
      int h = h_first, mb = mb_start, st = 0, dst = 0;
      uint32_t ph = 1u, dph = 1u;
      for (int it = 0; it < total_it; it++) {
        if (!mbar_wait(q_empty(st), ph, abort_flag)) { ok = false; break; }
        mbar_expect_tx(q_full(st), C::TILE_BYTES + 1024);
#pragma unroll
        for (int a = 0; a < C::ATOMS; a++)
          tma_load_4d(sbase + C::OFF_Q + st * C::TILE_BYTES + a * C::ATOM_BYTES, &tq, a * 64, h, mb * C::BM, b, q_full(st));
        bulk_load(sbase + C::OFF_ST + st * 1024, pp.w.stats + (((long long)b * p.hq + h) * n_mblocks + mb) * 256, 1024, q_full(st));
        if (!mbar_wait(do_empty(dst), dph, abort_flag)) { ok = false; break; }
        mbar_expect_tx(do_full(dst), C::TILE_BYTES);
#pragma unroll
        for (int a = 0; a < C::ATOMS; a++)
          tma_load_4d(sbase + C::OFF_DO + dst * C::TILE_BYTES + a * C::ATOM_BYTES, &tdo, a * 64, h, mb * C::BM, b, do_full(dst));
        if (++mb == mb_end) { mb = mb_first; h++; }
        if (++st == C::QS) { st = 0; ph ^= 1u; }
        if (++dst == C::DS) { dst = 0; dph ^= 1u; }
      }
      if (!ok) atomicExch(&g_mab_status[0], 1u);
    }
  } else if (warp == 1) {
    // ------------------------------- MMA issuer -------------------------------
    if (total_it > 0 && elect_one()) {
      const uint32_t idesc_s = make_idesc(128, 128, 0, 0);     // S^T, dP^T: K-major A and B
      const int slices = (p.d + 15) / 16;                      // of 16 columns: those past head_dim are zeros, and left out of all products
      const uint32_t idesc_kv = make_idesc(128, slices * 16, 0, 1);      // dV, dK: A in TMEM, MN-major B
      const uint32_t idesc_dq = make_idesc(128, slices * 16, 1, 1);      // dQ: MN-major A and B
      const uint64_t kK = make_desc(sbase + C::OFF_K, 16, 1024), kV = make_desc(sbase + C::OFF_V, 16, 1024);
      const uint64_t kQ = make_desc(sbase + C::OFF_Q, 16, 1024), kDO = make_desc(sbase + C::OFF_DO, 16, 1024);
      const uint64_t mK = make_desc(sbase + C::OFF_K, C::ATOM_BYTES, 1024), mDS = make_desc(sbase + C::OFF_DS, C::ATOM_BYTES, 1024);
      const uint64_t mQ = make_desc(sbase + C::OFF_Q, C::ATOM_BYTES, 1024), mDO = make_desc(sbase + C::OFF_DO, C::ATOM_BYTES, 1024);
      auto scores = [&](int col, uint64_t a, uint64_t bq) {      // [128 keys x 128 queries] over d
#pragma unroll
        for (int s = 0; s < D / 16; s++) {
          const uint64_t o = (uint64_t)(((s >> 2) * C::ATOM_BYTES + (s & 3) * 32) >> 4);
          if (s < slices) umma_bf16(tmem_base + col, a + o, bq + o, idesc_s, s ? 1u : 0u);
        }
      };
      // A (P^T or dS^T): 16 queries of a warpgroup's 64 are 8 columns; the second warpgroup's start 64 columns on
      auto grad_kv = [&](int col, int acol, uint64_t bop, uint32_t acc) {
#pragma unroll
        for (int s = 0; s < C::BM / 16; s++)
          umma_bf16_ta(tmem_base + col, tmem_base + acol + (s >> 2) * 64 + (s & 3) * 8, bop + (uint64_t)(s * 128), idesc_kv, s ? 1u : acc);
      };
      auto issue_s = [&](uint64_t so) {                          // (Q is there)
        scores(C::COL_S, kK, kQ + so);
        umma_commit(s_full);
      };
      auto issue_dp = [&](uint64_t so) {                         // (dO is there, dQ has left the columns)
        scores(C::COL_DP, kV, kDO + so);
        umma_commit(dp_full);
      };
      bool ok = mbar_wait(kv_full, 0, abort_flag) && mbar_wait(q_full(0), 0, abort_flag);
      if (ok) { fence_after(); issue_s(0); ok = mbar_wait(do_full(0), 0, abort_flag); }
      if (ok) { fence_after(); issue_dp(0); }
      int st = 0, dst = 0;
      uint32_t ph = 0, dph = 0;
      for (int it = 0; it < total_it && ok; it++) {
        const bool more = it + 1 < total_it;
        const int sn = st + 1 == C::QS ? 0 : st + 1, dn = dst + 1 == C::DS ? 0 : dst + 1;       // stages of the next block
        const uint32_t phn = sn ? ph : ph ^ 1u, dphn = dn ? dph : dph ^ 1u;
        if (more && !(ok = mbar_wait(q_full(sn), phn, abort_flag))) break;
        if (!(ok = mbar_wait(p_full, (uint32_t)it & 1u, abort_flag))) break;
        fence_after();
        grad_kv(C::COL_DV, C::COL_S, mDO + (uint64_t)((dst * C::TILE_BYTES) >> 4), it ? 1u : 0u);       // dV += P^T dO
        umma_commit(do_empty(dst));
        if (more) issue_s((uint64_t)((sn * C::TILE_BYTES) >> 4));        // P^T has been read: S^T of the next block
        if (!C::DQ_ALIAS && more && !(ok = mbar_wait(do_full(dn), dphn, abort_flag))) break;
        if (!C::DQ_ALIAS && it > 0 && !(ok = mbar_wait(dq_free, (uint32_t)(it - 1) & 1u, abort_flag))) break;
        if (!(ok = mbar_wait(ds_full, (uint32_t)it & 1u, abort_flag))) break;
        fence_after();
        grad_kv(C::COL_DK, C::COL_DP, mQ + (uint64_t)((st * C::TILE_BYTES) >> 4), it ? 1u : 0u);        // dK += dS^T Q
        umma_commit(q_empty(st));
        if (!C::DQ_ALIAS && more) issue_dp((uint64_t)((dn * C::TILE_BYTES) >> 4));
#pragma unroll
        for (int s = 0; s < C::BN / 16; s++)                             // dQ = dS K
          umma_bf16(tmem_base + C::COL_DQ, mDS + (uint64_t)(s * 128), mK + (uint64_t)(s * 128), idesc_dq, s ? 1u : 0u);
        umma_commit(dq_full);
        if (C::DQ_ALIAS && more) {
          if (!(ok = mbar_wait(do_full(dn), dphn, abort_flag))) break;
          if (!(ok = mbar_wait(dq_free, (uint32_t)it & 1u, abort_flag))) break;
          fence_after();
          issue_dp((uint64_t)((dn * C::TILE_BYTES) >> 4));
        }
        st = sn; ph = phn;
        dst = dn; dph = dphn;
      }
      if (!ok) atomicExch(&g_mab_status[0], 2u);
    }
  } else if (warp >= 12) {
    if constexpr (C::REGS_DRAIN > 128) reg_inc<C::REGS_DRAIN>(); else reg_dec<C::REGS_DRAIN>();
    // ------------------------------- dQ drain -------------------------------
    const int quad = warp & 3;
    const uint32_t tdq = tmem_base + ((uint32_t)(quad * 32) << 16) + C::COL_DQ;
    uint8_t* stg = smem + C::OFF_STG + quad * 2 * C::STG_BYTES;
    bool ok = true;
    int h = h_first, mb = mb_start;
    for (int it = 0; it < total_it; it++) {
      if (!mbar_wait(dq_full, (uint32_t)it & 1u, abort_flag)) { ok = false; break; }
      fence_after();
      uint32_t r[D];
#pragma unroll
      for (int c = 0; c < D / 32; c++) tmem_ld32(tdq + c * 32, r + c * 32);
      tmem_ld_wait();
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(dq_free);
      if constexpr (FORM == ALONE) {
        // the query block's dQ is complete: a row per lane
        const int row = mb * C::BM + quad * 32 + lane;
        if (row < p.Sq) {
          bf16* o = pp.w.dq + b * pp.w.dqs.b + row * pp.w.dqs.s + h * pp.w.dqs.h;
#pragma unroll
          for (int k = 0; k < D / 8; k++)
            if (k * 8 < p.d) *reinterpret_cast<uint4*>(o + k * 8) = pack8(reinterpret_cast<const float*>(r) + k * 8);
        }
      } else {
        float* tile = pp.dq_acc + (((long long)b * p.hq + h) * n_mblocks + mb) * (128 * pp.acc_d) + quad * (32 * pp.acc_d);
#pragma unroll
        for (int c = 0; c < D / 32; c++) {
          if (c * 32 >= p.d) break;
          uint8_t* sp = stg + (c & 1) * C::STG_BYTES;
          // This half of the staging has been read.  (Where a block has an odd number of chunks, its first waits for both halves: the last block's last chunk left from the same one.
          // Counting the halves through all blocks instead took registers: 68 -> 96 bytes spilled at 128 columns, in parts.)
          if (lane == 0) {
            if (c == 0 && ((p.d + 31) & 32)) bulk_wait_read_but<0>(); else bulk_wait_read_but<1>();
          }
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 8; k++)
            *reinterpret_cast<uint4*>(sp + k * 512 + lane * 16) =
                make_uint4(r[c * 32 + k * 4], r[c * 32 + k * 4 + 1], r[c * 32 + k * 4 + 2], r[c * 32 + k * 4 + 3]);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            bulk_reduce_add_f32(tile + c * 1024, smem_u32(sp), C::STG_BYTES);
            bulk_commit();
          }
        }
      }
      if (++mb == mb_end) { mb = mb_first; h++; }
    }
    if (lane == 0) bulk_wait_read_but<0>();
    if (!ok && lane == 0) atomicExch(&g_mab_status[0], 5u);
  } else if (warp >= 4) {
    reg_inc<C::REGS_MATH>();
    // ------------------------------- math warps -------------------------------
    const int quad = warp & 3;
    const int wg = (warp - 4) >> 2;                 // which 64 of the 128 query columns
    const int rit = quad * 32 + lane;               // key row inside the block
    const int key = n0 + rit;
    const uint32_t lane_addr = tmem_base + ((uint32_t)(quad * 32) << 16);
    const uint32_t ts = lane_addr + C::COL_S + wg * 64, tdp = lane_addr + C::COL_DP + wg * 64;
    uint8_t* sds = smem + C::OFF_DS + wg * C::ATOM_BYTES;
    const int2 see = key < p.Sk ? ma_queries(p, b, key) : make_int2(0, 0);
    [[maybe_unused]] bool behind_only = true;       // no key of the warp is seen by a query ahead of it
    if constexpr (BIAS) behind_only = __all_sync(0xffffffffu, see.x >= see.y || see.x + off >= key);
    bool ok = true;
    int h = h_first, mb = mb_start, qs = 0;
    uint32_t qph = 0;
    for (int it = 0; it < total_it; it++) {
      const int m0 = mb * C::BM + wg * 64;          // first query of these columns
      const float4* st = reinterpret_cast<const float4*>(smem + C::OFF_ST + qs * 1024) + wg * 16;
      [[maybe_unused]] float slope2 = 0.f;
      if constexpr (BIAS) slope2 = p.slopes[h] * LOG2E;
      if (!mbar_wait(q_full(qs), qph, abort_flag) ||        // the statistics
          !mbar_wait(s_full, (uint32_t)it & 1u, abort_flag)) { ok = false; break; }
      fence_after();
      float pf[64];                                 // P, then P times the cap's derivative
      {
        // the key is seen by queries lo to hi - 1 of these columns
        const int lo = see.x - m0, hi = see.y - m0;
        const bool need_mask = __any_sync(0xffffffffu, lo > 0 || hi < 64);
        // distance to the columns' places: 1 all behind the key, -1 all ahead of it, 0 both
        const int first = m0 + off - key;
        int side = 1;
        if constexpr (BIAS) side = behind_only || m0 + off >= n0 + quad * 32 + 31 ? 1 : m0 + off + 63 <= n0 + quad * 32 ? -1 : 0;
        const float slope = side > 0 ? -slope2 : slope2;
        const f32x2 step = pack2(2.f * slope, 2.f * slope);
        // 32 columns at a time.  With 128 columns of head_dim they are loaded so, too: all 64 do not fit into the registers beside P (1 x 8192, capped, both ways in
        // turn: 1675 to 1692 us, now 1605 to 1626).  What a warp decides for all columns is decided outside of their loops, which would else be one pair after the other.
        constexpr int AT_ONCE = (D == 64) ? 64 : 32;
        uint32_t all[AT_ONCE];
#pragma unroll
        for (int w = 0; w < 64; w += 32) {
          uint32_t pp_[16];
          if (w % AT_ONCE == 0) {
#pragma unroll
            for (int c = 0; c < AT_ONCE; c += 32) tmem_ld32(ts + w + c, all + c);
            tmem_ld_wait();
          }
          uint32_t* const sr = all + w % AT_ONCE;
          if constexpr (CAP) {                      // tanh
            float top[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 32; i += 2) top[(i >> 1) & 3] = max3abs(top[(i >> 1) & 3], __uint_as_float(sr[i]), __uint_as_float(sr[i + 1]));
            if (__all_sync(0xffffffffu, max2(max2(top[0], top[1]), max2(top[2], top[3])) <= pp.f.limit)) {
#pragma unroll
              for (int i = 0; i < 32; i += 2) {
                const f32x2 x = pack2(__uint_as_float(sr[i]), __uint_as_float(sr[i + 1])), u = mul2(x, x);
                float t0, t1;
                unpack2(mul2(x, fma2(u, fma2(u, fma2(u, pp.f.c[3], pp.f.c[2]), pp.f.c[1]), pp.f.c[0])), t0, t1);
                sr[i] = __float_as_uint(t0);
                sr[i + 1] = __float_as_uint(t1);
              }
            } else {
#pragma unroll
              for (int i = 0; i < 32; i++)          // tanh u = 1 - 2 / (exp 2u + 1)
                sr[i] = __float_as_uint(1.f - __fdividef(2.f, exp2f(__uint_as_float(sr[i]) * pp.f.by2) + 1.f));
            }
          }
          auto weights = [&](auto both) {           // both: the columns are on both sides of the key
            f32x2 add = pack2(0.f, 0.f);
            if constexpr (BIAS) { const float base = slope * (float)(first + w); add = pack2(base, base + slope); }
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              const float2 nl = reinterpret_cast<const float2*>(st)[(w + i) >> 1];
              const f32x2 x = pack2(__uint_as_float(sr[i]), __uint_as_float(sr[i + 1]));
              f32x2 to = pack2(nl.x, nl.y);
              if constexpr (BIAS && !decltype(both)::value) {
                to = add2(to, add);
                add = add2(add, step);
              } else if constexpr (BIAS) {
                to = pack2(fmaf(-slope2, fabsf((float)(first + w + i)), nl.x), fmaf(-slope2, fabsf((float)(first + w + i + 1)), nl.y));
              }
              unpack2(fma2(x, CAP ? pp.f.cap : pp.f.scale, to), pf[w + i], pf[w + i + 1]);
              pf[w + i] = exp2f(pf[w + i]);
              pf[w + i + 1] = exp2f(pf[w + i + 1]);
            }
          };
          if (BIAS && side == 0) weights(std::true_type{}); else weights(std::false_type{});
          const uint32_t bits = ma_bits(lo, hi, w);
          if (need_mask) {
#pragma unroll
            for (int i = 0; i < 32; i++)
              if (!(bits >> i & 1u)) pf[w + i] = 0.f;
          }
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            bf162 pb = __floats2bfloat162_rn(pf[w + i], pf[w + i + 1]);
            pp_[i >> 1] = *reinterpret_cast<uint32_t*>(&pb);
          }
          tmem_st16(ts + w / 2, pp_);
          if constexpr (CAP) {
#pragma unroll
            for (int i = 0; i < 32; i += 2) {       // P (1 - t^2)
              const f32x2 e = pack2(pf[w + i], pf[w + i + 1]), t = pack2(__uint_as_float(sr[i]), __uint_as_float(sr[i + 1]));
              unpack2(sub2(e, mul2(mul2(e, t), t)), pf[w + i], pf[w + i + 1]);
            }
            if (need_mask) {                        // (a hidden NaN is one still)
#pragma unroll
              for (int i = 0; i < 32; i++)
                if (!(bits >> i & 1u)) pf[w + i] = 0.f;
            }
          }
        }
        tmem_st_wait();
      }
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full);
      if (!mbar_wait(dp_full, (uint32_t)it & 1u, abort_flag)) { ok = false; break; }
      fence_after();
      uint32_t dd[32];
#pragma unroll
      for (int half = 0; half < 2; half++) {
        uint32_t dr[32];
        tmem_ld32(tdp + half * 32, dr);
        tmem_ld_wait();
#pragma unroll
        for (int c = 0; c < 8; c++) {
          const float4 nd = st[32 + half * 8 + c];
          const int i = half * 32 + c * 4;
          const f32x2 d01 = mul2(pack2(pf[i], pf[i + 1]),
                                 fma2(pack2(__uint_as_float(dr[c * 4]), __uint_as_float(dr[c * 4 + 1])), pp.scale2, pack2(nd.x, nd.y)));
          const f32x2 d23 = mul2(pack2(pf[i + 2], pf[i + 3]),
                                 fma2(pack2(__uint_as_float(dr[c * 4 + 2]), __uint_as_float(dr[c * 4 + 3])), pp.scale2, pack2(nd.z, nd.w)));
          float d[4];
          unpack2(d01, d[0], d[1]);
          unpack2(d23, d[2], d[3]);
          bf162 a = __floats2bfloat162_rn(d[0], d[1]), e = __floats2bfloat162_rn(d[2], d[3]);
          dd[i >> 1] = *reinterpret_cast<uint32_t*>(&a);
          dd[(i >> 1) + 1] = *reinterpret_cast<uint32_t*>(&e);
        }
      }
      tmem_st32(tdp, dd);
      // the shared copy may be rewritten once dQ of the previous block has read it
      if (it > 0 && !mbar_wait(dq_full, (uint32_t)(it - 1) & 1u, abort_flag)) { ok = false; break; }
#pragma unroll
      for (int c = 0; c < 8; c++)
        *reinterpret_cast<uint4*>(sds + sw128_off(rit, c)) = make_uint4(dd[c * 4], dd[c * 4 + 1], dd[c * 4 + 2], dd[c * 4 + 3]);
      tmem_st_wait();
      fence_before();
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(ds_full);
      if (++mb == mb_end) { mb = mb_first; h++; }
      if (++qs == C::QS) { qs = 0; qph ^= 1u; }
    }
    // dQ of the last block is the last MMA: everything has finished
    if (ok && total_it > 0) ok = mbar_wait(dq_full, (uint32_t)(total_it - 1) & 1u, abort_flag);
    if (CUT && leaves_sums && ok && total_it > 0) {
      // to this CTA's place, 32 columns at a time
      fence_after();
      const long long place = FORM == LIST ? (long long)piece.w * p.hkv + hk : ((long long)nblk * p.hkv * p.B + pair) * pp.parts + part;
      float* sum = (wg ? pp.dk_acc : pp.dv_acc) + place * (128 * D) + quad * (32 * D);
      uint8_t* out = smem + (wg ? C::OFF_V : C::OFF_K) + quad * C::STG_BYTES;
#pragma unroll 1
      for (int c = 0; c < D / 32 && c * 32 < p.d; c++) {
        uint32_t r[32];
        tmem_ld32(lane_addr + (wg ? C::COL_DK : C::COL_DV) + c * 32, r);
        tmem_ld_wait();
        if (lane == 0) bulk_wait_read_but<0>();
        __syncwarp();
#pragma unroll
        for (int k = 0; k < 8; k++)
          *reinterpret_cast<uint4*>(out + k * 512 + lane * 16) = make_uint4(r[k * 4], r[k * 4 + 1], r[k * 4 + 2], r[k * 4 + 3]);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          bulk_store(sum + c * 1024, smem_u32(out), C::STG_BYTES);
          bulk_commit();
        }
      }
      if (lane == 0) bulk_wait_read_but<0>();        // nothing reads shared memory after the CTA's end
    } else if (FORM != PARTS && !leaves_sums && ok && total_it > 0) {
      // through shared memory (K's tile for dV, V's for dK: nothing reads them any more), 64 columns of 32 keys at a time
      fence_after();
#pragma unroll 1
      for (int a = 0; a < C::ATOMS; a++) {
        uint8_t* out = smem + (wg ? C::OFF_V : C::OFF_K) + a * C::ATOM_BYTES + quad * 4096;
        uint32_t r[64];
        tmem_ld32(lane_addr + (wg ? C::COL_DK : C::COL_DV) + a * 64, r);
        tmem_ld32(lane_addr + (wg ? C::COL_DK : C::COL_DV) + a * 64 + 32, r + 32);
        tmem_ld_wait();
#pragma unroll
        for (int g = 0; g < 8; g++) {
          float f[8];
#pragma unroll
          for (int i = 0; i < 8; i++) f[i] = __uint_as_float(r[g * 8 + i]);
          *reinterpret_cast<uint4*>(out + sw128_off(lane, g)) = pack8(f);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0 && n0 + quad * 32 < p.Sk) {
          tma_store_4d(wg ? &tdk : &tdv, smem_u32(out), a * 64, hk, n0 + quad * 32, b);
          bulk_commit();
        }
      }
      if (lane == 0) bulk_wait_read_but<0>();        // nothing reads shared memory after the CTA's end
    } else if (FORM != PARTS && !leaves_sums && total_it == 0 && key < p.Sk) {
      // no query sees these keys: their gradients are zero
      const MaStrides& s = wg ? pp.w.dks : pp.w.dvs;
      bf16* orow = (wg ? pp.w.dk : pp.w.dv) + b * s.b + key * s.s + hk * s.h;
      for (int c = 0; c < p.d / 8; c++) *reinterpret_cast<uint4*>(orow + c * 8) = make_uint4(0, 0, 0, 0);
    }
    if (!ok && lane == 0) atomicExch(&g_mab_status[0], 3u);
  }

  fence_before();
  __syncthreads();
  if (warp == 1) {
    fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

template <int D, int FORM, bool CAP, bool BIAS>
int launch(const CUtensorMap* m, const BwdParams& p, unsigned grid, cudaStream_t s) {
  using C = Cfg<D>;
  auto fn = ma_bwd_kernel<D, FORM, CAP, BIAS>;
  static MaOnce once;
  bool* const set = once.here();
  if (!set) return LB_ERR_LAUNCH;
  if (!*set) {
    // the register split must fit in what the launch allocates, or it would wait for registers that nobody gives back
    cudaFuncAttributes fa;
    if (cudaFuncGetAttributes(&fa, fn) != cudaSuccess || (fa.numRegs + 7) / 8 * 8 != 128) return LB_ERR_LAUNCH;
    cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    *set = true;
  }
  return lb_launch(fn, grid, C::NTHREADS, C::SMEM, s, m[0], m[1], m[2], m[3], m[4], m[5], p);
}
template <int D, int FORM>
int launch_form(const CUtensorMap* m, const BwdParams& p, unsigned grid, cudaStream_t s) {
  const bool cap = p.w.f.softcap > 0.f, bias = p.w.f.slopes != nullptr;
  if (cap) return bias ? launch<D, FORM, true, true>(m, p, grid, s) : launch<D, FORM, true, false>(m, p, grid, s);
  return bias ? launch<D, FORM, false, true>(m, p, grid, s) : launch<D, FORM, false, false>(m, p, grid, s);
}

long long order_ints(const MaParams& p) { return (long long)p.B * ((p.Sk + 127) / 128); }

// CTAs of a key block, for its walk over query blocks of all heads of the group.  In query blocks: a CTA's fixed part is some 6, leaving dK / dV in fp32 instead of
// writing them 3 and their conversion 2 more (the figures of the causal backward's model); where the mask comes from the device its lengths are not known
// here, and those of a causal mask are taken.  Whole / parts, all kernels as a graph, us, causal: 2 x 2000, 16 / 2 heads, d 64 213 / 78; 1 x 2000, 16 / 4, d 128 156 / 79; 1 x 8192, 8 / 2, d 128
// 577 / 341; 4 x 500, 16 / 4, d 64 41 / 35; 2 x 1000, 16 / 4, d 96 80 / 51; 1 x 300, 8 / 2, d 64 30 / 14; left whole 8 x 2048, 32 / 4, d 64.
int parts_of(int B, int Sq, int Sk, int hq, int hkv, int causal, int sms) {
  const int n_mblocks = (Sq + 127) / 128, n_nblk = (Sk + 127) / 128, rep = hq / hkv, off = Sk - Sq;
  const long long pairs = (long long)hkv * B;
  if (Sk <= 128 || n_nblk * pairs > 4LL * sms) return 1;      // (several CTAs per SM, longest first)
  const int longest = n_mblocks * rep;
  long long total = 0;
  for (int k = 0; k < n_nblk; k++) total += (n_mblocks - (causal ? std::max(k * 128 - off, 0) / 128 : 0)) * (long long)rep;
  double best_time = 0.9 * std::max(longest + 6.0, 1.1 * (double)(total + 6LL * n_nblk) * pairs / sms);
  int best = 1;
  for (int parts = 2; parts <= std::min(longest, 32); parts++) {
    const double time = std::max((longest + parts - 1) / parts + 9.0, 1.1 * (double)(total + 9LL * n_nblk * parts) * pairs / sms) + 2.0;
    if (time < best_time) { best_time = time; best = parts; }
  }
  return best;
}

long long stats_floats(const MaParams& p) { return (long long)p.B * p.hq * ((p.Sq + 127) / 128) * 256; }
int acc_columns(int d) { return (d + 31) / 32 * 32; }
long long dq_floats(const MaParams& p) { return p.Sk <= 128 ? 0 : stats_floats(p) / 2 * acc_columns(p.d); }

// Under a window: the longest piece of a walk, how many pieces there may be beyond one per key block, and how many leave sums (of one kv head).  By the model of parts_of(), for keys that queries near
// them see and for blocks of sinks, which all queries behind them see.  Without a mask that is what the walks are at most; documents cut them shorter, and make more, shorter ones of sinks: then there is
// room for more pieces, and where it does not do the list makes them twice as long.  What pieces leave takes no more memory than dQ's sums, or 64 MB.  Without pieces there is no list; key blocks are
// sorted then by their walks where these differ.
// Without a mask, with several kv heads and two CTAs for each SM or more, the rest of the walks go head by head: 148 CTAs then work on two heads or three, whose Q, dO and dQ's sums stay in L2.  What is
// longer, of the sinks, goes head by head, too, and what begins with the last head may end behind all others; or it comes first, of all heads, and is slower, most where it is cut, for pieces that are
// at different queries share nothing.  The whole backward, us, in the order: longest first of all heads / head by head / the sinks' first and the rest head by head, for lengths of pieces in query blocks;
// 32 / 8 heads, d 128: 2 x 8208, window 103, 1 sink, 8 blocks 553 / 519 / 519, 65 508 / 589 / 514, 130 596 / 742 / 590, whole 887 / 1016 / 870; 1 x 8192, window 128, 1024 sinks, 32 blocks 547 / 496 / 548,
// 128 500 / 619 / 502, whole 725 / 828 / 684; 1 x 8192, window 1024, 4 sinks, 36 blocks 542 / 512 / 510, 128 516 / 724 / 508, whole 768 / 970 / 771; 1 x 32768, window 512, 4096 sinks, 20 blocks
// 9524 / 7947 / 7839, 256 7058 / 6215 / 6457, whole 6270 / 6669 / 5764; 4 x 8192, window 128, 4096 sinks, 43 blocks 6505 / 5609 / 6651, whole 5077 / 5024 / 4768; 16 x 742, 64 / 8 heads, window 337,
// 4 sinks, 32 blocks 890 / 792 / 827, whole 880 / 802 / 837.  With a mask, 32 / 8 heads, d 128, whole and sorted / in pieces: 1 x 8192, window 1024, 4 sinks, one document 740 / 493, documents of 3000
// 672 / 473; 32 / 4 heads, d 64: 8 x 2048, window 512, documents of 900, where none is cut, 330 / 340.
struct Pieces { int length, extra, sums, ordinary, lead; bool sorted; };
Pieces pieces_of(const MaParams& p, bool masked, int sms) {
  const int n_mblocks = (p.Sq + 127) / 128, n_nblk = (p.Sk + 127) / 128, rep = p.hq / p.hkv;
  const long long pairs = (long long)p.hkv * p.B, span = 128 + (p.causal ? 1LL : 2LL) * (p.window - 1LL);
  // (key and query blocks that begin at the same places meet in one block fewer)
  const long long most = (span + 127) / 128 + ((p.Sk - p.Sq) % 128 || !p.causal ? 1 : 0);
  const long long near = std::min<long long>(most, n_mblocks) * rep, far = (long long)n_mblocks * rep;
  const long long n_far = std::min<long long>((p.sinks + 127) / 128, n_nblk), n_near = n_nblk - n_far;
  const long long room = std::max(dq_floats(p), 1LL << 24) / (2LL * p.hkv * 128 * (p.d <= 64 ? 64 : 128));      // pieces that leave sums
  const bool heads = !masked && p.hkv > 1 && n_nblk * pairs >= 2LL * sms;
  double best_time = 0.0;
  Pieces best{(int)far, 0, 0, 0, 0, false};
  if (p.Sk <= 128) return best;
  auto look = [&](long long length) {
    const long long a = (near + length - 1) / length, b = (far + length - 1) / length;
    long long extra = (n_near * (a - 1) + n_far * (b - 1)) * p.B, sums = extra + ((a > 1 ? n_near : 0) + (b > 1 ? n_far : 0)) * p.B;
    if (sums > room) return;
    const double work = (double)(n_near * (near + a * (a > 1 ? 9 : 6))) * pairs / sms, sinks = (double)(n_far * (far + b * (b > 1 ? 9 : 6))) * pairs / sms;
    const double other = (double)((near + a - 1) / a), sink = n_far ? (double)((far + b - 1) / b) : 0.0, longest = std::max(other, sink);
    const double apart = 1.045 * (work + sinks) + std::max(0.0, longest - std::max(other, (work + sinks) / p.hkv));
    const double first = heads ? std::max(std::max(other, 1.2 * sink) + 9.0, 1.045 * work + (b > 1 ? 1.4 : 1.1) * sinks) : std::max(longest + 9.0, 1.1 * (work + sinks));
    const bool by_head = heads && (longest == other || apart <= first);
    const double time = (by_head ? apart : first) + (extra ? 1.0 : 0.0);
    if (best_time != 0.0 && time >= best_time) return;
    best_time = time;
    if (masked && extra) {
      extra = std::min(2 * extra + (p.sinks ? 4LL * p.B : 0), room / 2);
      sums = extra + std::min(extra, (long long)p.B * n_nblk);
    }
    best = Pieces{(int)length, (int)std::min(extra, 1LL << 24), (int)std::min(sums, 1LL << 25), by_head ? INT_MAX : heads ? (int)other : 0, 0, false};
  };
  for (long long parts = 1; parts <= std::min<long long>(far, 64); parts++) look((far + parts - 1) / parts);
  for (long long parts = 1; parts <= std::min<long long>(near, 32); parts++) look((near + parts - 1) / parts);
  // (walks differ where there are sinks, and where a window is so long that many of them end with the queries; both passes, in order of their places / sorted, us: 16 x 1500, 8 / 1 heads, d 64, window 800
  // 278 / 234, 400 left 234; 8 x 2000, 8 / 2 heads, window 1900, 4 sinks 275 / 217)
  best.sorted = masked || (n_nblk * pairs > sms && ((n_far > 0 && far > near) || 2 * near > far));
  best.lead = (int)((best.ordinary == INT_MAX ? 0 : heads ? n_far : n_nblk) * p.B);
  return best;
}

template <int D>
int launch_bwd(BwdParams& p, cudaStream_t s) {
  const MaParams& a = p.w.f;
  const MaBwdParams& w = p.w;
  CUtensorMap m[6];      // q, k, v, dout, dk, dv
  int rc;
  const uint64_t B = a.B, Sq = a.Sq, Sk = a.Sk, hq = a.hq, hkv = a.hkv, d = a.d;
  if ((rc = make_map_bf16_4d(m, a.q, d, hq, Sq, B, a.qs.h, a.qs.s, a.qs.b, 128))) return rc;
  if ((rc = make_map_bf16_4d(m + 1, a.k, d, hkv, Sk, B, a.ks.h, a.ks.s, a.ks.b, 128))) return rc;
  if ((rc = make_map_bf16_4d(m + 2, a.v, d, hkv, Sk, B, a.vs.h, a.vs.s, a.vs.b, 128))) return rc;
  if ((rc = make_map_bf16_4d(m + 3, w.dout, d, hq, Sq, B, w.dos.h, w.dos.s, w.dos.b, 128))) return rc;
  if ((rc = make_map_bf16_4d(m + 4, w.dk, d, hkv, Sk, B, w.dks.h, w.dks.s, w.dks.b, 32))) return rc;
  if ((rc = make_map_bf16_4d(m + 5, w.dv, d, hkv, Sk, B, w.dvs.h, w.dvs.s, w.dvs.b, 32))) return rc;
  // Up to 128 keys a query block's dQ comes from one CTA, which writes it: nothing to clear, to add to and to convert.  Added / written, as a graph, us: 4 x 128, 12 heads, d 64 13.2 / 10.3,
  // 8 x 128, 32 heads 24.6 / 18.5, 32 x 128, 32 / 8 heads 54 / 41; 8 x 100, 16 heads, d 128 18.6 / 14.4.
  const bool alone = a.Sk <= 128;
  const long long grid = p.items ? (order_ints(a) + p.extra) * a.hkv : (long long)((a.Sk + 127) / 128) * a.hkv * a.B * p.parts;
  if (grid > 2147483647LL) return LB_ERR_SHAPE;
  const long long rows = (long long)a.B * ((a.Sq + 127) / 128 * 128) * a.hq;
  const long long rows_per_block = 256 / (D / 8), cap = lb_num_sms() * 16;
  const long long pblocks = (rows + rows_per_block - 1) / rows_per_block;
  LB_LAUNCH((p.items ? ma_bwd_prep_kernel<D, true> : ma_bwd_prep_kernel<D, false>), (int)(pblocks < cap ? pblocks : cap) + (p.order || p.items ? 1 : 0), 256, 0, s, p, !alone);
  rc = p.items ? launch_form<D, LIST>(m, p, (unsigned)grid, s) : p.parts > 1 ? launch_form<D, PARTS>(m, p, (unsigned)grid, s) : alone ? launch_form<D, ALONE>(m, p, (unsigned)grid, s) : launch_form<D, WHOLE>(m, p, (unsigned)grid, s);
  if (rc || alone) return rc;
  const bool cut = p.parts > 1 || p.items;
  const long long part_rows = cut ? 2LL * a.B * ((a.Sk + 127) / 128 * 128) * a.hkv : 0;
  const long long cblocks = (rows * (D / 32) + part_rows * (D / 8) + 255) / 256;      // (a thread takes 32 values of dQ)
  LB_LAUNCH(cut ? ma_convert_kernel<D, true> : ma_convert_kernel<D, false>, (int)(cblocks < cap ? cblocks : cap), 256, 0, s, p);
  return LB_OK;
}

long long part_floats(const MaParams& p, int parts) {
  return parts > 1 ? (long long)p.B * p.hkv * ((p.Sk + 127) / 128) * parts * 128 * (p.d <= 64 ? 64 : 128) : 0;
}
long long piece_floats(const MaParams& p, const Pieces& c) { return (long long)c.sums * p.hkv * 128 * (p.d <= 64 ? 64 : 128); }

}  // namespace

// Bytes of the workspace: row statistics, fp32 dQ (up to 128 keys: none), fp32 dK and dV of parts or pieces, the order of the key blocks or the list of the pieces.
long long ma_bwd_ws_bytes(const MaParams& p, bool masked) {
  const long long all = stats_floats(p) + dq_floats(p);
  if (p.window > 0) {
    const Pieces c = pieces_of(p, masked, lb_num_sms());
    return (all + (c.extra ? 2 * piece_floats(p, c) + 4 * (order_ints(p) + c.extra) + 3 * order_ints(p) + 4 : order_ints(p))) * (long long)sizeof(float);
  }
  return (all + 2 * part_floats(p, parts_of(p.B, p.Sq, p.Sk, p.hq, p.hkv, p.causal, lb_num_sms())) + order_ints(p)) * (long long)sizeof(float);
}

int ma_launch_bwd(const MaBwdParams& w, cudaStream_t s) {
  const MaParams& a = w.f;
  BwdParams p;
  p.w = w;
  p.items = nullptr;
  p.acc_d = acc_columns(a.d);
  p.dq_acc = w.stats + stats_floats(a);
  p.dk_acc = p.dq_acc + dq_floats(a);
  p.f.set(a, false, twice);
  p.scale2 = twice(a.scale);
  const Pieces c = a.window > 0 ? pieces_of(a, a.qb != nullptr, lb_num_sms()) : Pieces{};
  p.parts = 1;
  p.order = nullptr;
  if (c.extra) {
    p.chunk = c.length;
    p.extra = c.extra;
    p.sums = c.sums;
    p.ordinary = c.ordinary;
    p.dv_acc = p.dk_acc + piece_floats(a, c);
    p.items = reinterpret_cast<int4*>(p.dv_acc + piece_floats(a, c));
    p.joined = reinterpret_cast<int2*>(p.items + order_ints(a) + c.extra);
    p.n_items = reinterpret_cast<int*>(p.joined + order_ints(a));
    p.cut_blocks = p.n_items + 4;
    return a.d <= 64 ? launch_bwd<64>(p, s) : launch_bwd<128>(p, s);
  }
  if (!a.window) p.parts = parts_of(a.B, a.Sq, a.Sk, a.hq, a.hkv, a.causal, lb_num_sms());
  p.dv_acc = p.dk_acc + part_floats(a, p.parts);
  p.lead = a.window > 0 ? c.lead : (int)order_ints(a);
  p.order = (a.window > 0 ? c.sorted : a.kb && p.parts == 1) && a.Sk > 128 ? reinterpret_cast<int*>(p.dv_acc + part_floats(a, p.parts)) : nullptr;
  return a.d <= 64 ? launch_bwd<64>(p, s) : launch_bwd<128>(p, s);
}

// Copies the status words of the backward to host memory and clears them.
extern "C" int lb_masked_attn_bwd_status(void* out) {
  cudaError_t e = cudaMemcpyFromSymbol(out, g_mab_status, sizeof(unsigned int) * 4);
  if (e != cudaSuccess) { g_lb_last_cuda_error = (int)e; return LB_ERR_LAUNCH; }
  unsigned int zeros[4] = {0, 0, 0, 0};
  cudaMemcpyToSymbol(g_mab_status, zeros, sizeof(zeros));
  return LB_OK;
}
