// Forward of attention under interval masks (attn_masked.cuh) on the 5th-generation tensor cores, head_dim up to 128 (a multiple of 8, in
// tiles of 64 or 128 columns).
//
// A CTA works on one tile of 128 queries of one (batch, head) at a time, two CTAs per SM; S = Q K^T and O += P V by tcgen05.mma with S, P and O in tensor
// memory, K and V by TMA through a ring of 16 KB slots, further tiles by cluster launch control: the pipeline of the causal
// forward (flash_fwd_tcgen05.cu has what each part of it is worth).  What is different here:
//   * a row is two threads', 64 columns of a key block each, in eight softmax warps, which tell each other maxima and sums through shared memory.  (One thread a row / two, 8 x 2048,
//     32 / 4 heads, d 64: causal 268 / 254 us, bias 470 / 312, cap 363 / 305, documents 178 / 134; 1 x 8192, 32 / 8 heads, d 128: 632 / 595, bias 974 / 727, cap 720 / 722.)
//   * the keys of a tile run from the first key of its first row to the last key of its last (the ends never fall), from exactly there: blocks start
//     at any key, so that a document of n keys takes ceil(n / 128) of them wherever it lies.  Blocks inside all 32 intervals of a warp are not masked.
//   * with a cap the scores are known to lie within it.  Up to softcap * log2(e) = 80 exponentials are taken relative to zero instead of the running
//     maximum: 2^+-80 and sums of them are far inside fp32 (and bf16 has the same exponents), and nothing is ever rescaled (8 x 2048, d 64 with the maximum / without 400 / 304 us, 1 x 8192, d 128 828 / 566).  With 128 columns the two halves of a
//     block then have nothing to tell each other, and their scores, P and products run apart (d 128, cap: 700 -> 640 us).  Above 80 the maximum is kept.
//   * tanh: where no score of 32 rows x 64 columns is above 0.6 caps (33 at caps above 55: MaTerms), x times a polynomial in x^2 on the FMA pipe, two at a time
//     (7e-5 of a score at most, at caps above 550 1.3e-7 caps); else by its definition with exp2, whose units the softmax needs itself.
//   * the bias is an addend of the FMA that scales a score (or evaluates its polynomial), counted up along the columns; only where a block holds keys on both sides of a row is its
//     distance made per column.  Without a cap the exponentials' reference is a bound, not the maximum itself: what they are relative to cancels, as long as it is within 2^60
//     or so of the maximum.  The nearest key blocks come first, or the maximum would grow from block to block and O be rescaled in each (both together: 1 x 8192, 32 / 8 heads,
//     d 128 780 -> 632 us, 8 x 2048, 32 / 4 heads, d 64 303 -> 287).
//   * slopes below zero, whose scores rise with distance, are told apart on the device, by head: the bound takes the largest distance, and what exponentials under a cap are
//     relative to is the bias at the row's farthest key instead of zero.  (For all biased forms under a cap 0 to 3 %: 1 x 4096, 32 / 8 heads, d 128, cap 50 210 -> 216 us, without
//     gradients 177 -> 178, 4 x 2048, 32 / 4 heads, d 64 191 -> 193; without a cap nothing.)
//   * o is divided by the sum of the weights as they are rounded for P V.  A row that all but one key leave cold has o = v of that key then, and a D = do . o whose
//     error is as small as the differences dP - D that the backward lives on (the weight's own rounding, 2^-9 of dP, would drown them); lse is of the sum of the
//     unrounded ones, from which the backward's P are made.
//   * few tiles share their key blocks between CTAs, which leave O in fp32 with its reference and sums; another kernel joins them.
//   * o leaves twice: rounded, and what the rounding left (for the backward's row sums).
// What bounds it: latency, with instructions close behind.  Of the active cycles 61 % of the issue slots and 41 to 52 % of the exponentials' unit (d 64, two tiles per SM), 39 %
// of the tensor pipe (d 128); a block takes 1960 (d 64) / 2400 cycles (d 128, cap) of an SM, 2530 with documents, whose loops are short and whose blocks are nearly all masked.
// All waits are bounded; on expiry a status word is set and the CTA drains and frees its TMEM.
#include "attn_masked.cuh"
#include "tcgen05.cuh"

static __device__ unsigned int g_ma_status[4] = {0, 0, 0, 0};

namespace {
using namespace bw;

constexpr int THREADS = 384;
// Registers per thread of the issuing and of the two softmax warpgroups (two CTAs of 384 threads leave 80 per thread at launch).
constexpr int REGS_LAUNCH = 80, REGS_ISSUE = 48, REGS_SOFTMAX = 96;
static_assert(REGS_ISSUE + 2 * REGS_SOFTMAX <= 3 * REGS_LAUNCH, "a CTA has 384 x 80 registers");
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

struct FwdParams {
  MaParams a;
  int tiles_x;                   // query tiles (128 rows) per (batch, head)
  int steal;                     // CTAs go on with entries that have not been started
  int group;                     // (batch, head) pairs whose tiles are ordered together
  FastDiv by_grp, by_group, by_last, by_hq, by_rep;    // entries of a group, heads of a group / of the last one, hq, hq / hkv
  MaTerms f;
  int splits;                    // CTAs of a tile, each with a share of its key blocks, which leave parts
  float *part_o, *part_s;        // [tile][split] x [D / 4][128 rows][4] fp32, and x [reference, sum, rounded sum][128 rows]
};

enum : int { NO_CAP, CAP_ZERO, CAP_MAX };      // CAP_ZERO: exponentials relative to zero, CAP_MAX: to the running maximum

template <int D>
struct Cfg {
  static constexpr int BM = 128, BN = 128;
  static constexpr int ATOMS = D / 64;
  static constexpr int SLOT_BYTES = 128 * 128;          // K: 128 keys x 64 columns; V: 128 keys x 64 columns or 64 keys x 128 columns
  static constexpr int SLOTS = 4;
  static constexpr int OUT_BYTES = (D == 64) ? 4096 : 2048;      // of a softmax warp
  static constexpr int UNITS = 2 * ATOMS;               // slots that a key block takes, K before V
  // TMEM columns: S fp32 [128], O fp32 [D], P packed bf16 [64]; with 128 columns of O, P takes the first half of S's
  static constexpr bool P_ALIAS = (D == 128);
  static constexpr int COL_S = 0, COL_O = 128, COL_P = P_ALIAS ? 0 : 192, TMEM_COLS = 256;
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_RING = OFF_Q + ATOMS * SLOT_BYTES;
  // 2 KB per softmax warp: 32 rows x 32 columns of O on their way out, and before that what the rows' two threads tell each other
  static constexpr int OFF_OUT = OFF_RING + SLOTS * SLOT_BYTES;
  static constexpr int OFF_BAR = OFF_OUT + 8 * OUT_BYTES;
  static constexpr int NBAR = 2 + 2 * SLOTS + 14;
  static constexpr int SMEM = OFF_BAR + 288;
};
static_assert(Cfg<64>::SMEM <= 115712 && Cfg<128>::SMEM <= 115712, "two CTAs per SM");

// 64 raw scores to units of log2, capped and lowered with distance.  `first`: key of column 0 less the row's position; `side`: the columns lie on the row's left (1),
// on its right (-1) or on both sides (0), the same for all lanes; `at`: what the row's exponentials are relative to, taken off with the bias.
template <int CAP, bool BIAS>
__device__ __forceinline__ void scores64(uint32_t* r, const FwdParams& p, float slope2, int side, int first, float at) {
  bool small = true;
  if constexpr (CAP != NO_CAP) {
    float top[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 64; i += 2) top[(i >> 1) & 3] = max3abs(top[(i >> 1) & 3], __uint_as_float(r[i]), __uint_as_float(r[i + 1]));
    small = __all_sync(0xffffffffu, max2(max2(top[0], top[1]), max2(top[2], top[3])) <= p.f.limit);
  }
  const float slope = side < 0 ? -slope2 : slope2;
  const float step1 = side ? 2.f * slope : 0.f;
  const f32x2 step = pack2(step1, step1);
#pragma unroll
  for (int c0 = 0; c0 < 64; c0 += 32) {
    // (counted up anew every 32 columns: its rounding errors do not pile up)
    const float base = fmaf(slope, (float)(first + c0), -at);
    f32x2 add = !BIAS ? pack2(0.f, 0.f) : side ? pack2(base, base + slope) : pack2(-at, -at);
    if (CAP == NO_CAP || small) {
#pragma unroll
      for (int i = c0; i < c0 + 32; i += 2) {
        const f32x2 x = pack2(__uint_as_float(r[i]), __uint_as_float(r[i + 1]));
        f32x2 f = p.f.c[0];
        if constexpr (CAP != NO_CAP) {
          const f32x2 w = mul2(x, x);
          f = fma2(w, fma2(w, fma2(w, p.f.c[3], p.f.c[2]), p.f.c[1]), p.f.c[0]);
        }
        f32x2 y;
        if constexpr (BIAS) {
          y = fma2(x, f, add);
          add = add2(add, step);
        } else {
          y = mul2(x, f);
        }
        float y0, y1;
        unpack2(y, y0, y1);
        r[i] = __float_as_uint(y0);
        r[i + 1] = __float_as_uint(y1);
      }
    } else if constexpr (CAP != NO_CAP) {
      const float by = p.f.by2;
#pragma unroll
      for (int i = c0; i < c0 + 32; i += 2) {
        float a0, a1;
        unpack2(add, a0, a1);
        if constexpr (BIAS) add = add2(add, step);
        // tanh u = 1 - 2 / (exp 2u + 1)
        const float t0 = 1.f - __fdividef(2.f, exp2f(__uint_as_float(r[i]) * by) + 1.f), t1 = 1.f - __fdividef(2.f, exp2f(__uint_as_float(r[i + 1]) * by) + 1.f);
        r[i] = __float_as_uint(fmaf(p.f.cap1, t0, a0));
        r[i + 1] = __float_as_uint(fmaf(p.f.cap1, t1, a1));
      }
    }
  }
  if (BIAS && side == 0) {
    const float d0 = (float)first;
#pragma unroll
    for (int i = 0; i < 64; i++) r[i] = __float_as_uint(fmaf(-slope2, fabsf(d0 + (float)i), __uint_as_float(r[i])));
  }
}

// GRAD: o_lo and lse are wanted
template <int D, int CAP, bool BIAS, bool GRAD>
__global__ void __launch_bounds__(THREADS, 2)
ma_fwd_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, const __grid_constant__ CUtensorMap to,
              const __grid_constant__ CUtensorMap to_lo, const __grid_constant__ FwdParams pp) {
  using C = Cfg<D>;
  constexpr bool MADE = CAP != NO_CAP;                // scores are made in units of log2 ahead of the softmax
  constexpr bool LINEAR = BIAS && !MADE;              // the bias is added where the exponentials are taken
  constexpr bool SPLIT = D == 128 && CAP == CAP_ZERO;
  constexpr bool BACKWARDS = BIAS && CAP != CAP_ZERO;      // the nearest keys first: on the way to them the maximum would grow in every block, and O be rescaled
  const MaParams& p = pp.a;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + C::NBAR + 5);     // behind two 16-byte answers
  int* s_abort = reinterpret_cast<int*>(tmem_slot + 1);     // {abort, extra wait in ms}: see bw::mbar_wait

  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;   // (uniform over the warp)
  const uint32_t sbase = smem_u32(smem);
  if (sbase & 1023u) {                                       // the swizzled tiles need it; nothing has been started yet
    if (threadIdx.x == 0) atomicExch(&g_ma_status[0], 4u);
    return;
  }
  const uint32_t bar0 = smem_u32(bars);
  const uint32_t q_full = bar0, q_empty = bar0 + 8;
  auto full = [&](int s) { return bar0 + 8u * (2 + s); };
  auto empty = [&](int s) { return bar0 + 8u * (2 + C::SLOTS + s); };
  const uint32_t bar1 = bar0 + 8u * (2 + 2 * C::SLOTS);
  const uint32_t s_full = bar1, s_free = bar1 + 8, p_full = bar1 + 16, pv_done = bar1 + 24;
  auto next_full = [&](int i) { return bar1 + 32u + 8u * i; };
  auto next_empty = [&](int i) { return bar1 + 48u + 8u * i; };
  auto pair_bar = [&](int quad) { return bar1 + 64u + 8u * quad; };
  // SPLIT: scores and P of the second 64 keys of a block have barriers of their own
  auto s_full_of = [&](int half) { return SPLIT && half ? bar1 + 96u : s_full; };
  auto p_full_of = [&](int half) { return SPLIT && half ? bar1 + 104u : p_full; };
  const uint32_t next_slot = (bar0 + 8u * C::NBAR + 15u) & ~15u;

  // One entry per (batch, head, query tile): the last tiles, which see most under a causal mask, of all heads of a group first; a group is as many heads as keep
  // their K / V in L2 together.  A resident CTA goes on with entries that have not been started (cluster launch control).
  volatile int* abort_flag = s_abort;
  const int off = p.Sk - p.Sq;
  struct Tile { int m0, b, h, hk, key0, nb, split; };
  auto tile_of = [&](int cid) {
    Tile t;
    t.split = 0;
    if (pp.splits > 1) { t.split = cid % pp.splits; cid /= pp.splits; }
    const int grp = pp.by_grp.div(cid);
    const int in_grp = cid - grp * (int)pp.by_grp.d;
    const FastDiv& heads = (grp + 1) * pp.group <= p.hq * p.B ? pp.by_group : pp.by_last;
    const int row = heads.div(in_grp);
    const int bh = grp * pp.group + in_grp - row * (int)heads.d;
    t.m0 = (pp.tiles_x - 1 - row) * C::BM;
    t.b = pp.by_hq.div(bh);
    t.h = bh - t.b * p.hq;
    t.hk = pp.by_rep.div(t.h);
    t.key0 = ma_keys(p, t.b, t.m0).x;
    // (a tile whose rows see nothing takes one block, all of it hidden)
    t.nb = max((ma_keys(p, t.b, min(t.m0 + C::BM, p.Sq) - 1).y - t.key0 + C::BN - 1) / C::BN, 1);
    if (pp.splits > 1) {
      // (a share behind the tile's last block is one block that all rows' intervals hide)
      const int share = (t.nb + pp.splits - 1) / pp.splits, first = min(t.split * share, t.nb);
      t.key0 += first * C::BN;
      t.nb = max(min(share, t.nb - first), 1);
    }
    return t;
  };
  // Entry n + 1 of this CTA: the answer to request n, or -1 at the end.
  auto next_cta = [&](int n) -> int {
    if (!pp.steal || !mbar_wait(next_full(n & 1), (uint32_t)(n >> 1) & 1u, abort_flag)) return -1;
    const int cta = cancel_result(next_slot + 16u * (n & 1));
    fence_proxy_async_smem();
    return cta;
  };

  if (threadIdx.x == 0) {
    s_abort[0] = s_abort[1] = 0;
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int s = 0; s < C::SLOTS; s++) { mbar_init(full(s), 1); mbar_init(empty(s), 1); }
    mbar_init(s_full, 1);
    mbar_init(pv_done, 1);
    mbar_init(s_free, 8);
    mbar_init(p_full, SPLIT ? 4 : 8);
    mbar_init(s_full_of(1), 1);
    mbar_init(p_full_of(1), SPLIT ? 4 : 8);
    for (int i = 0; i < 4; i++) mbar_init(pair_bar(i), 2);
    for (int i = 0; i < 2; i++) { mbar_init(next_full(i), 1); mbar_init(next_empty(i), 9); }   // the issuer and eight softmax warps read
    mbar_init_fence();
    prefetch_tmap(&tq); prefetch_tmap(&tk); prefetch_tmap(&tv); prefetch_tmap(&to); prefetch_tmap(&to_lo);
  }
  if (warp == 1) tmem_alloc(smem_u32(tmem_slot), C::TMEM_COLS);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  if (!pp.steal) grid_go();
  grid_wait();

  if (warp < 4) {
    reg_dec<REGS_ISSUE>();
    if (warp == 0) {
      // ------------------------------- TMA producer -------------------------------
      if (elect_one()) {
        bool ok = true;
        int slot = 0;
        uint32_t phase = 0;
        int asked = 0;
        for (int n = 0, cta = (int)blockIdx.x; ok && cta >= 0; n++) {
          if (pp.steal) {
            if (!mbar_wait(next_empty(n & 1), ((uint32_t)(n >> 1) & 1u) ^ 1u, abort_flag)) { ok = false; break; }
            mbar_expect_tx(next_full(n & 1), 16);
            cancel_next(next_slot + 16u * (n & 1), next_full(n & 1));
            asked = n + 1;
          }
          const Tile t = tile_of(cta);
          if (!mbar_wait(q_empty, (uint32_t)(n & 1) ^ 1u, abort_flag)) { ok = false; break; }
          mbar_expect_tx(q_full, C::ATOMS * C::SLOT_BYTES);
#pragma unroll
          for (int a = 0; a < C::ATOMS; a++) tma_load_4d(sbase + C::OFF_Q + a * C::SLOT_BYTES, &tq, a * 64, t.h, t.m0, t.b, q_full);
          for (int j = 0; j < t.nb && ok; j++) {
            const int key0 = t.key0 + (BACKWARDS ? t.nb - 1 - j : j) * C::BN;
#pragma unroll
            for (int u = 0; u < C::UNITS; u++) {
              if (ok && !mbar_wait(empty(slot), phase ^ 1u, abort_flag)) ok = false;
              if (!ok) break;
              const uint32_t dst = sbase + C::OFF_RING + slot * C::SLOT_BYTES, bar = full(slot);
              mbar_expect_tx(bar, C::SLOT_BYTES);
              if (u < C::ATOMS) {
                tma_load_4d(dst, &tk, u * 64, t.hk, key0, t.b, bar);              // box 128 keys x 64 columns
              } else {
                const int half = u - C::ATOMS;                                    // 128 columns: keys 0-63, then 64-127
#pragma unroll
                for (int a = 0; a < 2; a++)                                       // boxes 64 keys x 64 columns
                  tma_load_4d(dst + a * 8192, &tv, D == 128 ? a * 64 : 0, t.hk, key0 + (D == 128 ? half * 64 : a * 64), t.b, bar);
              }
              if (++slot == C::SLOTS) { slot = 0; phase ^= 1u; }
            }
          }
          if (ok) cta = next_cta(n);
        }
        if (!ok) {
          atomicExch(&g_ma_status[0], 1u);
          if (asked) mbar_wait(next_full((asked - 1) & 1), (uint32_t)((asked - 1) >> 1) & 1u, abort_flag);   // nothing arrives after the CTA's end
        }
      }
    } else if (warp == 1) {
      // ------------------------------- MMA issuer -------------------------------
      // Per tile S(0); then per key block, 64 columns: S(j+1) as soon as the softmax threads hold S(j) in registers, and P(j) V when P(j) is there; 128
      // columns: P(j) V, then S(j+1) into the columns that P(j) leaves.
      if (elect_one()) {
        const uint32_t idesc_s = make_idesc(C::BM, C::BN, 0, 0);
        const int slices = (p.d + 15) / 16;             // of 16 columns: those past head_dim are zeros, and left out of both products
        const uint32_t idesc_o = make_idesc(C::BM, slices * 16, 0, 1);
        const uint64_t qa = make_desc(sbase + C::OFF_Q, 16, 1024);
        const uint64_t dk0 = make_desc(sbase + C::OFF_RING, 16, 1024);
        const uint64_t dv0 = make_desc(sbase + C::OFF_RING, 8192, 1024);
        const uint32_t s_dst = tmem_base + C::COL_S, o_dst = tmem_base + C::COL_O, pa = tmem_base + C::COL_P;
        bool ok = true;
        // slots are taken in load order: K (ATOMS slots), then V of every block
        auto ring = [&](int& slot, uint32_t& phase, int step) { slot += step; if (slot >= C::SLOTS) { slot -= C::SLOTS; phase ^= 1u; } };
        int ks = 0, vs = C::ATOMS;                      // next slot of K and of V, and their phases
        uint32_t kp = 0, vp = 0;
        uint32_t g = 0;                                 // key blocks so far, over all tiles: the phase of the per-block barriers
        auto k_ready = [&]() -> bool {                  // the next block's K has arrived
          if (!mbar_wait(full(ks), kp, abort_flag)) return false;
          if (C::ATOMS == 1) return true;
          const bool wrap = ks + 1 == C::SLOTS;
          return mbar_wait(full(wrap ? 0 : ks + 1), wrap ? kp ^ 1u : kp, abort_flag);
        };
        // SPLIT: S of the next block's keys 64 * half and on, into the columns that P of such keys has left; the second half releases K (and Q)
        const uint32_t idesc_half = make_idesc(C::BM, 64, 0, 0);
        auto issue_half = [&](int half, bool last) {
#pragma unroll
          for (int a = 0; a < C::ATOMS; a++) {
            const int slot = ks + a >= C::SLOTS ? ks + a - C::SLOTS : ks + a;
            const uint64_t ka = dk0 + (uint64_t)((slot * C::SLOT_BYTES + half * 8192) >> 4);
#pragma unroll
            for (int s = 0; s < 4; s++)
              if (a * 4 + s < slices)
                umma_bf16(s_dst + 64 * half, qa + (uint64_t)((a * C::SLOT_BYTES + s * 32) >> 4), ka + (uint64_t)((s * 32) >> 4), idesc_half, (a | s) ? 1u : 0u);
          }
          umma_commit(s_full_of(half));
          if (half) {
#pragma unroll
            for (int a = 0; a < C::ATOMS; a++) {
              umma_commit(empty(ks));
              ring(ks, kp, a == C::ATOMS - 1 ? C::UNITS - C::ATOMS + 1 : 1);
            }
            if (last) umma_commit(q_empty);
          }
        };
        auto issue_s = [&](bool last) {                 // S = Q K^T of the next block (K is there), then release its slots of K (and Q)
          fence_after();
          if constexpr (SPLIT) {
            issue_half(0, last);
            issue_half(1, last);
          } else {
#pragma unroll
            for (int a = 0; a < C::ATOMS; a++) {
              const uint64_t ka = dk0 + (uint64_t)((ks * C::SLOT_BYTES) >> 4);
#pragma unroll
              for (int s = 0; s < 4; s++)
                if (a * 4 + s < slices)
                  umma_bf16(s_dst, qa + (uint64_t)((a * C::SLOT_BYTES + s * 32) >> 4), ka + (uint64_t)((s * 32) >> 4), idesc_s, (a | s) ? 1u : 0u);
              if (a == C::ATOMS - 1) umma_commit(s_full);
              umma_commit(empty(ks));
              ring(ks, kp, a == C::ATOMS - 1 ? C::UNITS - C::ATOMS + 1 : 1);
            }
            if (last) umma_commit(q_empty);
          }
        };
        // SPLIT: O += P V by halves of 64 keys, each with S of the next block's behind it: the softmax threads of one half work while the products of the other run.
        // (The first P V of a tile waits for both: until then the last tile's O is still being read.)
        auto issue_halves = [&](bool first, bool last, bool last_s) -> bool {
#pragma unroll
          for (int half = 0; half < 2; half++) {
            if (!mbar_wait(full(vs), vp, abort_flag)) return false;
            if (half == 0 && !last && !k_ready()) return false;
            if (half == 0 && first && !mbar_wait(p_full_of(1), g & 1u, abort_flag)) return false;
            if (!mbar_wait(p_full_of(half), g & 1u, abort_flag)) return false;
            fence_after();
            const uint64_t va = dv0 + (uint64_t)((vs * C::SLOT_BYTES) >> 4);
#pragma unroll
            for (int s = 0; s < 4; s++)
              umma_bf16_ta(o_dst, pa + 64u * half + 8u * s, va + (uint64_t)((s * 2048) >> 4), idesc_o, (half | s) ? 1u : (first ? 0u : 1u));
            if (half && last) umma_commit(pv_done);
            umma_commit(empty(vs));
            ring(vs, vp, half ? C::ATOMS + 1 : 1);
            if (!last) issue_half(half, last_s);
          }
          return true;
        };
        auto issue_pv = [&](bool first, bool last) -> bool {      // O += P V of block g, then release its slots of V
#pragma unroll
          for (int half = 0; half < 2; half++) {
            if (half == 0 && !mbar_wait(full(vs), vp, abort_flag)) return false;
            if (half == 0) {
              if (D == 128) {                           // the second half of V, ahead of the wait that is the last to come
                const bool wrap = vs + 1 == C::SLOTS;
                if (!mbar_wait(full(wrap ? 0 : vs + 1), wrap ? vp ^ 1u : vp, abort_flag)) return false;
              }
              if (C::P_ALIAS && !last && !k_ready()) return false;
              if (!mbar_wait(p_full, g & 1u, abort_flag)) return false;
              fence_after();
            }
            const uint64_t va = dv0 + (uint64_t)((vs * C::SLOT_BYTES + (D == 128 ? 0 : half * 8192)) >> 4);
#pragma unroll
            for (int s = 0; s < 4; s++)
              umma_bf16_ta(o_dst, pa + 8u * (half * 4 + s), va + (uint64_t)((s * 2048) >> 4), idesc_o, (half | s) ? 1u : (first ? 0u : 1u));
            if (half && (!C::P_ALIAS || last)) umma_commit(pv_done);
            if (D == 128 || half) {
              umma_commit(empty(vs));
              ring(vs, vp, half ? C::ATOMS + 1 : 1);
            }
          }
          return true;
        };
        Tile t = tile_of((int)blockIdx.x);
        for (int n = 0; ok; n++) {
          ok = k_ready() && mbar_wait(q_full, (uint32_t)n & 1u, abort_flag);
          if (ok && !C::P_ALIAS && n > 0) ok = mbar_wait(s_free, (g - 1) & 1u, abort_flag);
          if (ok) issue_s(t.nb == 1);
          // (the next tile's size is on its way while this one is worked on)
          const int cta = ok ? next_cta(n) : -1;
          Tile next = t;
          if (cta >= 0) {
            mbar_arrive(next_empty(n & 1));
            next = tile_of(cta);
          }
          for (int j = 0; j < t.nb && ok; j++, g++) {
            const bool last = j + 1 == t.nb;
            if constexpr (SPLIT) {
              ok = issue_halves(j == 0, last, j + 2 == t.nb);
              continue;
            }
            if (!C::P_ALIAS && !last) {
              ok = k_ready() && mbar_wait(s_free, g & 1u, abort_flag);
              if (ok) issue_s(j + 2 == t.nb);
            }
            if (ok) ok = issue_pv(j == 0, last);
            if (C::P_ALIAS && ok && !last) issue_s(j + 2 == t.nb);
          }
          if (cta < 0) break;
          t = next;
        }
        if (!ok) atomicExch(&g_ma_status[0], 2u);
      }
    }
  } else {
    // ------------------------------- softmax warps -------------------------------
    // A row is two threads', in the warps quad and quad + 4 of the eight: 64 columns of a key block each, and half of the columns of O.
    reg_inc<REGS_SOFTMAX>();
    const int quad = warp & 3, set = warp >= 8 ? 1 : 0;
    const uint32_t lane_addr = tmem_base + ((uint32_t)(quad * 32) << 16);
    const uint32_t ts_addr = lane_addr + C::COL_S + set * 64, to_addr = lane_addr + C::COL_O + set * (D / 2), tp_addr = lane_addr + C::COL_P + set * (SPLIT ? 64 : 32);
    [[maybe_unused]] const f32x2 scale2 = MADE ? 0 : kept(pp.f.scale);
    uint8_t* const out = smem + C::OFF_OUT + (warp - 4) * C::OUT_BYTES;
    float2* const mine = reinterpret_cast<float2*>(out) + lane;
    const float2* const other = reinterpret_cast<float2*>(smem + C::OFF_OUT + ((warp - 4) ^ 4) * C::OUT_BYTES) + lane;
    bool ok = true;
    uint32_t turn = 0;
    // The row's two threads meet (in a wait that ends, as all do); what the other one has in y.  Two places in turn: nobody is more than one meeting ahead.
    auto meet = [&](float2 x, float2& y) {
      mine[turn * 32] = x;
      __syncwarp();
      if (lane == 0) mbar_arrive(pair_bar(quad));
      if (!mbar_wait(pair_bar(quad), turn, abort_flag)) ok = false;
      y = other[turn * 32];
      turn ^= 1u;
    };
    auto arrive = [&](uint32_t bar) {              // once per warp
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    uint32_t g = 0;                                // key blocks so far, over all tiles
    bool s_ready = false;                          // S of the next block was seen complete
    Tile t = tile_of((int)blockIdx.x);
    // (rows past the last one are never stored: they are left unmasked)
    auto keys_of = [&](const Tile& at) { const int row = at.m0 + quad * 32 + lane; return row < p.Sq ? ma_keys(p, at.b, row) : make_int2(0, 0x7fffffff); };
    int2 see = keys_of(t);
    for (int n = 0; ok; n++) {
      const int nb = t.nb, row = t.m0 + quad * 32 + lane, warp_at = t.m0 + quad * 32 + off;      // the row's place is row + off
      [[maybe_unused]] float slope2 = 0.f;
      [[maybe_unused]] bool left_only = true;      // no row of the warp sees a key behind its own
      if constexpr (BIAS) {
        slope2 = p.slopes ? p.slopes[t.h] * LOG2E : 0.f;
        left_only = __all_sync(0xffffffffu, row >= p.Sq || see.y <= row + off + 1);
      }
      if (lane == 0) bulk_wait_read_but<0>();      // the last tile's O has left the place of the meetings
      __syncwarp();
      [[maybe_unused]] float top = 0.f;
      // (a slope below zero lifts scores over the cap, up to its value at the farthest key that the row sees: exponentials are relative to that, and one of them is 2^-80 or more)
      if constexpr (BIAS && CAP == CAP_ZERO)
        if (slope2 < 0.f && row < p.Sq) top = -slope2 * (float)max(max(row + off - see.x, see.y - 1 - (row + off)), 0);
      float m_i = -INFINITY, m_s = top, l_i = 0.f, lp_i = 0.f;      // the row's running maximum, what exponentials are relative to, this thread's sums of them
      for (int j = 0; j < nb; j++, g++) {
        if (!s_ready && !mbar_wait(s_full_of(set), g & 1u, abort_flag)) { ok = false; break; }
        fence_after();
        uint32_t r[64];
        const int c0 = t.key0 + (BACKWARDS ? nb - 1 - j : j) * C::BN + set * 64, lo = see.x - c0, hi = see.y - c0;       // visible columns
        const bool need_mask = __any_sync(0xffffffffu, lo > 0 || hi < 64);
        tmem_ld32(ts_addr, r);
        tmem_ld32(ts_addr + 32, r + 32);
        tmem_ld_wait();
        if (!C::P_ALIAS) arrive(s_free);                 // S may be overwritten by the next key block
        const bool pv_ready = !C::P_ALIAS && j > 0 && mbar_test_wait(pv_done, (g - 1) & 1u);   // asked ahead of its use
        if constexpr (MADE) {
          const int side = left_only || c0 + 63 <= warp_at ? 1 : c0 >= warp_at + 31 ? -1 : 0;
          scores64<CAP, BIAS>(r, pp, slope2, side, c0 - (row + off), top);
        }
        if (need_mask) {
#pragma unroll
          for (int w = 0; w < 64; w += 32) {
            const uint32_t bits = ma_bits(lo, hi, w);
#pragma unroll
            for (int i = 0; i < 32; i++)
              if (!(bits >> i & 1u)) r[w + i] = 0xff800000u;           // -inf
          }
        }
        // LINEAR: bias at column i is slope * (c0 + i - place); with keys on both sides of a row (slope 0) it is in r from here on
        [[maybe_unused]] float slope = 0.f;
        if constexpr (LINEAR) {
          slope = left_only || c0 + 63 <= warp_at ? slope2 : c0 >= warp_at + 31 ? -slope2 : 0.f;
          if (slope == 0.f) {
            const float by = -__fdividef(slope2, pp.f.scale1), d0 = (float)(c0 - (row + off));
#pragma unroll
            for (int i = 0; i < 64; i++) r[i] = __float_as_uint(fmaf(by, fabsf(d0 + (float)i), __uint_as_float(r[i])));
          }
        }
        bool rescale = false;
        float corr = 1.f;
        if constexpr (CAP != CAP_ZERO) {
          // Lazy reference maximum: the old one stays unless the new maximum is more than 2^8 above it, so that O and l rarely need rescaling.
          const float unit = MADE || LINEAR ? 1.f : pp.f.scale1;
          const float from = LINEAR ? -INFINITY : m_i;
          float mx4[4] = {from, from, from, from};       // four independent chains
          float m_new = m_i;
          if constexpr (LINEAR) {
            // A bound instead of the maximum: of 32 columns the largest score with the smallest distance (with the largest where the slope is below zero and scores rise with
            // it), at most 31 slopes above it.  (Where that is more than 2^60 the biased scores are looked at one by one.)
#pragma unroll
            for (int w = 0; w < 64; w += 32) {
              const int to_left = row + off - (c0 + w + 31), to_right = c0 + w - (row + off);
              const float steep = fabsf(slope), rise = slope2 < 0.f ? steep : -steep;      // (0 where the bias is in r)
              if (steep <= 60.f / 31.f) {
                float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int i = w; i < w + 32; i += 2) top[(i >> 1) & 1] = max3(top[(i >> 1) & 1], __uint_as_float(r[i]), __uint_as_float(r[i + 1]));
                m_new = max2(m_new, fmaf(max2(top[0], top[1]), pp.f.scale1, rise * (float)(slope2 < 0.f ? max(to_left, to_right) + 31 : max(max(to_left, to_right), 0))));
              } else {
#pragma unroll
                for (int i = w; i < w + 32; i++) m_new = max2(m_new, fmaf(__uint_as_float(r[i]), pp.f.scale1, rise * fabsf((float)(to_right + (i - w)))));
              }
            }
          } else {
#pragma unroll
            for (int i = 0; i < 64; i += 2) mx4[(i >> 1) & 3] = max3(mx4[(i >> 1) & 3], __uint_as_float(r[i]), __uint_as_float(r[i + 1]));
            m_new = max2(max2(mx4[0], mx4[1]), max2(mx4[2], mx4[3]));
          }
          float2 theirs;
          meet(make_float2(m_new, 0.f), theirs);
          m_new = max2(m_new, theirs.x);
          const bool grow = !(m_i != -INFINITY && (m_new - m_i) * unit <= 8.f);
          if (__any_sync(0xffffffffu, grow)) {
            // (where a row has seen nothing yet there is nothing to rescale)
            rescale = __any_sync(0xffffffffu, grow && m_i != -INFINITY);
            if (!grow) m_new = m_i;
            const float m_r = m_s;
            // (a row with a score of +inf has no softmax: NaN, as inf - inf gives)
            m_s = (m_new == -INFINITY) ? 0.f : (m_new == INFINITY ? __int_as_float(0x7fffffff) : LINEAR ? fmaf(fabsf(m_new), 0x1p-22f, m_new) : m_new);
            corr = (m_i == -INFINITY) ? 0.f : exp2f((m_r - m_s) * unit);
            l_i *= corr;
            lp_i *= corr;
            m_i = m_new;
          }
        }
        // exponentials, packed as bf16 pairs (column c of P holds keys 2c, 2c+1)
        uint32_t pr[32];
        f32x2 sum = pack2(0.f, 0.f);
        float p0 = 0.f, p1 = 0.f;
        const f32x2 nms2 = pack2(-m_s, -m_s);
        [[maybe_unused]] f32x2 add = nms2, step = nms2;
        if constexpr (LINEAR) step = pack2(2.f * slope, 2.f * slope);
#pragma unroll
        for (int c = 0; c < 32; c++) {
          float e0 = __uint_as_float(r[2 * c]), e1 = __uint_as_float(r[2 * c + 1]);
          // (the difference first: with the maximum scaled ahead and a fused product, what its rounding left would be the exponent of scores far from zero)
          if constexpr (LINEAR) {
            if (c % 16 == 0) {                           // (counted up anew every 32 columns: its rounding errors do not pile up)
              const float base = fmaf(slope, (float)(c0 + 2 * c - (row + off)), -m_s);
              add = pack2(base, base + slope);
            }
            unpack2(fma2(pack2(e0, e1), scale2, add), e0, e1);
            add = add2(add, step);
          } else if constexpr (CAP != CAP_ZERO) {
            f32x2 x = add2(pack2(e0, e1), nms2);
            if constexpr (!MADE) x = mul2(x, scale2);
            unpack2(x, e0, e1);
          }
          e0 = exp2f(e0);
          e1 = exp2f(e1);
          bf162 pk = __floats2bfloat162_rn(e0, e1);
          pr[c] = *reinterpret_cast<uint32_t*>(&pk);
          if constexpr (GRAD) sum = add2(sum, pack2(e0, e1));
          add_halves(pr[c], p0, p1);
        }
        if (j > 0) {
          // previous P V finished: O is stable and the P columns may be overwritten.  (128 columns: S(j) was issued behind it by the same thread, so
          // its completion says that P V has completed too.)
          if (!C::P_ALIAS) {
            if (!pv_ready && !mbar_wait(pv_done, (g - 1) & 1u, abort_flag)) { ok = false; break; }
            fence_after();
          }
          if (CAP != CAP_ZERO && rescale) {
#pragma unroll 1
            for (int c = 0; c < D / 2; c += 16) {
              uint32_t o[16];
              tmem_ld16(to_addr + c, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
              tmem_st16(to_addr + c, o);
            }
          }
        }
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        // (128 columns: P takes columns of S that the row's other thread reads; both have, where maxima were exchanged.  SPLIT: its own.)
        tmem_st32(tp_addr, pr);
        tmem_st_wait();
        arrive(p_full_of(set));
        s_ready = !C::P_ALIAS && j + 1 < nb && mbar_test_wait(s_full, (g + 1) & 1u);
        float s0, s1;
        unpack2(sum, s0, s1);
        l_i += s0 + s1;
        lp_i += p0 + p1;
      }
      if (!ok) break;
      const int cta = next_cta(n);
      __syncwarp();
      Tile next = t;
      int2 see_next = see;
      if (cta >= 0) {
        if (lane == 0) mbar_arrive(next_empty(n & 1));
        next = tile_of(cta);
        see_next = keys_of(next);
      }
      float2 theirs;
      meet(make_float2(l_i, lp_i), theirs);
      l_i += theirs.x;
      lp_i += theirs.y;
      float2 none;
      meet(theirs, none);                          // (O takes the place of what the other one has read by now)
      if (!ok || !mbar_wait(pv_done, C::P_ALIAS ? (uint32_t)n & 1u : (g - 1) & 1u, abort_flag)) ok = false;
      if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
      fence_after();
      if (pp.splits > 1) {                         // (one tile per CTA)
        const long long part = (((long long)t.b * p.hq + t.h) * pp.tiles_x + t.m0 / C::BM) * pp.splits + t.split;
        float4* o = reinterpret_cast<float4*>(pp.part_o + part * (C::BM * D)) + set * (D / 8) * C::BM + quad * 32 + lane;
#pragma unroll 1
        for (int c = 0; c < D / 2; c += 32) {
          uint32_t r[32];
          tmem_ld32(to_addr + c, r);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 8; i++) o[(c / 4 + i) * C::BM] = reinterpret_cast<const float4*>(r)[i];
        }
        if (set == 0) {
          float* s = pp.part_s + part * (3 * C::BM) + quad * 32 + lane;
          s[0] = lp_i != 0.f ? m_s * (MADE || LINEAR ? 1.f : pp.f.scale1) : -INFINITY;
          s[C::BM] = l_i;
          s[2 * C::BM] = lp_i;
        }
        break;
      }
      const float inv = lp_i != 0.f ? 1.f / lp_i : 0.f;
      // 32 columns at a time through shared memory and TMA stores, which leave out rows past the last and columns past head_dim
      auto leave = [&](const CUtensorMap* map, const uint4* v, int col, int at) {      // v: 32 columns of the lane's row
        if (C::OUT_BYTES == 2048) {
          if (lane == 0) bulk_wait_read_but<0>();
          __syncwarp();
        }
#pragma unroll
        for (int i = 0; i < 4; i++) *reinterpret_cast<uint4*>(out + at + lane * 64 + ((i ^ ((lane >> 1) & 3)) << 4)) = v[i];      // (64-byte swizzle)
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0 && t.m0 + quad * 32 < p.Sq) {
          tma_store_4d(map, smem_u32(out) + at, col, t.h, t.m0 + quad * 32, t.b);
          bulk_commit();
        }
      };
#pragma unroll 1
      for (int c = 0; c < D / 2 && set * (D / 2) + c < p.d; c += 32) {
        uint32_t r[32];
        uint4 hi[4];
        tmem_ld32(to_addr + c, r);
        tmem_ld_wait();
#pragma unroll
        for (int g8 = 0; g8 < 4; g8++) {
          float f[8], back[8];
#pragma unroll
          for (int i = 0; i < 8; i++) f[i] = __uint_as_float(r[g8 * 8 + i]) * inv;
          hi[g8] = pack8(f);
          unpack8(hi[g8], back);
#pragma unroll
          for (int i = 0; i < 8; i++) r[g8 * 8 + i] = __float_as_uint(f[i] - back[i]);
        }
        leave(&to, hi, set * (D / 2) + c, 0);
        if constexpr (GRAD) {
#pragma unroll
          for (int g8 = 0; g8 < 4; g8++) hi[g8] = pack8(reinterpret_cast<const float*>(r) + g8 * 8);
          leave(&to_lo, hi, set * (D / 2) + c, C::OUT_BYTES - 2048);
        }
      }
      if (GRAD && set == 0 && row < p.Sq) p.lse[((long long)t.b * p.hq + t.h) * p.Sq + row] = l_i != 0.f ? m_s * (MADE || LINEAR ? LN2 : p.scale) + logf(l_i) : -INFINITY;
      if (cta < 0) break;
      t = next;
      see = see_next;
    }
    if (lane == 0) bulk_wait_read_but<0>();        // nothing reads shared memory after the CTA's end
    if (!ok && lane == 0) atomicExch(&g_ma_status[0], 3u);
  }

  fence_before();
  __syncthreads();
  if (warp == 1) {
    fence_after();
    tmem_dealloc(tmem_base, C::TMEM_COLS);
  }
}

// Adds up the parts of a tile's rows: weights by their references, the order of the splits.  A thread has 8 columns of a row; a warp's stores are whole rows.
template <int D>
__global__ void ma_join_kernel(const __grid_constant__ FwdParams pp) {
  grid_go();
  grid_wait();
  const MaParams& p = pp.a;
  constexpr int TPR = D / 8;
  const int c = threadIdx.x % TPR, rows = blockDim.x / TPR;
  const long long total = (long long)p.B * p.hq * p.Sq;
  for (long long at = (long long)blockIdx.x * rows + threadIdx.x / TPR; at < total; at += (long long)gridDim.x * rows) {
    const int i = (int)(at % p.Sq), h = (int)(at / p.Sq % p.hq), b = (int)(at / p.Sq / p.hq), r = i & 127;
    const long long part = (((long long)b * p.hq + h) * pp.tiles_x + i / 128) * pp.splits;
    const float* s = pp.part_s + part * 384 + r;
    float m = -INFINITY;
    for (int k = 0; k < pp.splits; k++) m = max2(m, s[k * 384]);
    float l = 0.f, lp = 0.f, f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    const float4* o = reinterpret_cast<const float4*>(pp.part_o + part * (128 * D)) + 2 * c * 128 + r;
    for (int k = 0; k < pp.splits; k++) {
      const float from = s[k * 384];
      if (from == -INFINITY) continue;                       // (has seen nothing)
      const float w = exp2f(from - m);
      const float4 x = o[(long long)k * (32 * D)], y = o[(long long)k * (32 * D) + 128];
      l += w * s[k * 384 + 128];
      lp += w * s[k * 384 + 256];
      f[0] += w * x.x; f[1] += w * x.y; f[2] += w * x.z; f[3] += w * x.w;
      f[4] += w * y.x; f[5] += w * y.y; f[6] += w * y.z; f[7] += w * y.w;
    }
    const float inv = lp != 0.f ? 1.f / lp : 0.f;
    if (c * 8 < p.d) {
      const long long to = (((long long)b * p.Sq + i) * p.hq + h) * p.d + c * 8;
      float back[8];
#pragma unroll
      for (int k = 0; k < 8; k++) f[k] *= inv;
      const uint4 hi = pack8(f);
      *reinterpret_cast<uint4*>(p.o + to) = hi;
      if (p.o_lo) {
        unpack8(hi, back);
#pragma unroll
        for (int k = 0; k < 8; k++) f[k] -= back[k];
        *reinterpret_cast<uint4*>(p.o_lo + to) = pack8(f);
      }
    }
    if (p.lse && c == 0) p.lse[at] = l != 0.f ? m * LN2 + logf(l) : -INFINITY;
  }
}

// CTAs of a tile: one where there is a tile for each SM, else as many as find room (two per SM), with four key blocks or more each.  Whole / split, us, causal: 8192 queries and keys, 1 head,
// d 64 97 / 45; 2 heads, d 128, cap 121 / 74; 4 x 4096 of 4 heads, d 128, cap 68 / 46; 2048, 4 heads, d 64 27 / 22; one query, 32 / 8 heads, d 128, 8192 keys 118 / 37, 4 x 32768 keys
// 557 / 296; left whole 1024, 8 heads, d 128 19.7 / 20.4 and 2 x 1024, 8 heads, d 64 19.5 / 19.2.  (Where the mask comes from the device the length of the walks is not known here: that of all keys is taken.)
int splits_of(int B, int Sq, int Sk, int hq, int sms) {
  const long long tiles = (long long)((Sq + 127) / 128) * hq * B;
  const int blocks = (Sk + 127) / 128;
  if (tiles > sms || blocks <= 8) return 1;
  const long long room = 2LL * sms / tiles;
  return (int)(room < blocks / 4 ? room : blocks / 4);
}
long long part_floats(int B, int Sq, int hq, int d, int splits) {
  return splits > 1 ? (long long)((Sq + 127) / 128) * hq * B * splits * 128 : 0;
}

template <int D, int CAP, bool BIAS, bool GRAD>
int launch_form(const CUtensorMap* maps, const FwdParams& p, unsigned grid, cudaStream_t s) {
  using C = Cfg<D>;
  auto fn = ma_fwd_kernel<D, CAP, BIAS, GRAD>;
  static MaOnce once;
  bool* const set = once.here();
  if (!set) return LB_ERR_LAUNCH;
  if (!*set) {
    // the register split must fit in what the launch allocates, or it would wait for registers that nobody gives back
    cudaFuncAttributes fa;
    if (cudaFuncGetAttributes(&fa, fn) != cudaSuccess || (fa.numRegs + 7) / 8 * 8 < REGS_LAUNCH) return LB_ERR_LAUNCH;
    cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    *set = true;
  }
  LB_LAUNCH(fn, grid, THREADS, C::SMEM, s, maps[0], maps[1], maps[2], maps[3], maps[4], p);
  if (p.splits > 1) {
    const long long blocks = ((long long)p.a.B * p.a.hq * p.a.Sq * (D / 8) + 255) / 256, cap = lb_num_sms() * 16;
    LB_LAUNCH(ma_join_kernel<D>, (unsigned)(blocks < cap ? blocks : cap), 256, 0, s, p);
  }
  return LB_OK;
}

// (Without gradients the sum of the unrounded weights, lse and o_lo are left out: 2 x 4099 both ways, cap 30, 16 heads, d 64 118.7 -> 115.3 us, 8 x 2048, documents of 300, 32 / 4 heads,
// d 64 137 -> 121.)
template <int D, int CAP, bool BIAS>
int launch(const CUtensorMap* maps, const FwdParams& p, unsigned grid, cudaStream_t s) {
  return p.a.o_lo ? launch_form<D, CAP, BIAS, true>(maps, p, grid, s) : launch_form<D, CAP, BIAS, false>(maps, p, grid, s);
}

template <int D>
int launch_fwd(const MaParams& a, void* ws, long long ws_bytes, cudaStream_t s) {
  CUtensorMap maps[5];      // q, k, v, o, o_lo
  int rc;
  const uint64_t B = a.B, Sq = a.Sq, Sk = a.Sk, hq = a.hq, hkv = a.hkv, d = a.d;
  if ((rc = make_map_bf16_4d(maps, a.q, d, hq, Sq, B, a.qs.h, a.qs.s, a.qs.b, 128))) return rc;
  if ((rc = make_map_bf16_4d(maps + 1, a.k, d, hkv, Sk, B, a.ks.h, a.ks.s, a.ks.b, 128))) return rc;
  if ((rc = make_map_bf16_4d(maps + 2, a.v, d, hkv, Sk, B, a.vs.h, a.vs.s, a.vs.b, 64))) return rc;
  if ((rc = make_map_bf16_4d(maps + 3, a.o, d, hq, Sq, B, d, hq * d, Sq * hq * d, 32, 32))) return rc;
  if ((rc = make_map_bf16_4d(maps + 4, a.o_lo ? a.o_lo : a.o, d, hq, Sq, B, d, hq * d, Sq * hq * d, 32, 32))) return rc;
  FwdParams p;
  p.a = a;
  p.tiles_x = (a.Sq + 127) / 128;
  // heads ordered together: as many as have their K / V in 48 MB (of 126 MB of L2), whole GQA groups
  const long long kv_bytes = 4LL * D * a.Sk, pairs = (long long)a.hq * a.B;
  const long long kv_heads = kv_bytes >= (48LL << 20) ? 1 : (48LL << 20) / kv_bytes;
  p.group = (int)(kv_heads * (a.hq / a.hkv) < pairs ? kv_heads * (a.hq / a.hkv) : pairs);
  p.splits = ws_bytes > 0 && ws_bytes >= ma_fwd_ws_bytes(a) ? splits_of(a.B, a.Sq, a.Sk, a.hq, lb_num_sms()) : 1;
  p.part_o = (float*)ws;
  p.part_s = p.part_o + part_floats(a.B, a.Sq, a.hq, a.d, p.splits) * D;
  const long long grid = p.tiles_x * pairs * p.splits;
  if (grid > 2147483647LL) return LB_ERR_SHAPE;
  p.by_grp.set((unsigned)(p.tiles_x * p.group));
  p.by_group.set((unsigned)p.group);
  p.by_last.set((unsigned)(pairs % p.group ? pairs % p.group : p.group));
  p.by_hq.set((unsigned)a.hq);
  p.by_rep.set((unsigned)(a.hq / a.hkv));
  p.steal = p.splits == 1 && grid > 2 * lb_num_sms();      // (with all tiles resident at once there is none to take)
  p.f.set(a, true, twice);
  const bool bias = a.slopes != nullptr;
  if (a.softcap <= 0.f) return bias ? launch<D, NO_CAP, true>(maps, p, (unsigned)grid, s) : launch<D, NO_CAP, false>(maps, p, (unsigned)grid, s);
  if (p.f.cap1 <= 80.f) return bias ? launch<D, CAP_ZERO, true>(maps, p, (unsigned)grid, s) : launch<D, CAP_ZERO, false>(maps, p, (unsigned)grid, s);
  // (above 55 the running maximum is kept, with and without slopes by the form that has the bias: such caps are rare, and four forms fewer are built.  Without slopes a form of its own
  // is faster: cap 200, this one / its own, 8 x 2048, 32 / 4 heads, d 64 412 / 362 us, both ways 710 / 645; 1 x 8192, 32 / 8 heads, d 128 830 / 740, both ways 1710 / 1585.)
  return launch<D, CAP_MAX, true>(maps, p, (unsigned)grid, s);
}

}  // namespace

// Bytes of the parts' workspace: 0 where tiles are not split.
long long ma_fwd_ws_bytes(const MaParams& p) {
  const int splits = splits_of(p.B, p.Sq, p.Sk, p.hq, lb_num_sms());
  return part_floats(p.B, p.Sq, p.hq, p.d, splits) * ((p.d <= 64 ? 64 : 128) + 3) * (long long)sizeof(float);
}

int ma_launch_fwd(const MaParams& p, void* ws, long long ws_bytes, cudaStream_t s) {
  return p.d <= 64 ? launch_fwd<64>(p, ws, ws_bytes, s) : launch_fwd<128>(p, ws, ws_bytes, s);
}

// Copies the status words of the forward to host memory and clears them.
extern "C" int lb_masked_attn_status(void* out) {
  cudaError_t e = cudaMemcpyFromSymbol(out, g_ma_status, sizeof(unsigned int) * 4);
  if (e != cudaSuccess) { g_lb_last_cuda_error = (int)e; return LB_ERR_LAUNCH; }
  unsigned int zeros[4] = {0, 0, 0, 0};
  cudaMemcpyToSymbol(g_ma_status, zeros, sizeof(zeros));
  return LB_OK;
}
