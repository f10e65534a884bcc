// Cross entropy over a vocabulary without the logits, and its gradient.
//
//   z = X W^T             X [n][d] f16 hidden states, W [v][d] f16 vocabulary weights
//   lse_i  = log sum_v exp z_iv
//   loss_i = lse_i - z_{i,t_i}                        0 where t_i is outside [0, v)
//   g_iv   = dl_i (exp(z_iv - lse_i) - [v = t_i]);    dX = g W,  dW = g^T X
//
// A map-map-reduce contraction whose result is consumed by a (maximum, sum) reduction.  The logits stay in
// tensor memory: the contraction's epilogue folds each 256 x 256 tile to one (maximum, sum) pair per
// row, and a small kernel (in small calls the last CTA) folds the v/256 pairs of a row.  The gradient works the vocabulary off in pieces: a
// piece's logits are computed again (by the same instructions; sums of more than 2048 products in one
// accumulator where the losses had two, which was 1.4e-6 of a logit over 4096 products and grows with their number), turned into g in
// binary16 in the epilogue, and that piece of g meets W (summed over the pieces in f32) and X.
//
// Rounding of g to 11 bits.  With q_i = 1 - exp(-loss_i) the row is kept as
//   G_iv = 2^13 (exp(z_iv - lse_i) - [v = t_i]) / q_i,  G_{i,t_i} = -2^13 exactly,  and  w_i = dl_i q_i  aside:
//   dX_i = 2^-13 w_i sum_v G_iv W_v                 w_i in f32, after the sum
//   dW_v = 2^(E-14-13) sum_i G_iv (X_i w_i 2^(14-E))  E the largest exponent of any |X_ij w_i|
// The target's term, the largest of its row by far, is thus exact in dX; the others round relative to
// themselves (2^13 keeps probabilities down to 2^-27 out of binary16's subnormals, and the sum over the others is q_i,
// so |G| <= 2^13 up to the rounding of the losses).  In dW the scaled X is rounded once more to binary16: half
// a unit in the last place of each element, independent of the others, of the size of the result's own rounding.
// All of binary16's range is used for it: X_ij w_i keeps its 11 bits down to 2^-28 of the largest, and below that an absolute 2^(E-39),
// which is no more than what the result itself is rounded to (2^-25) unless the largest is 2^15 or more and the result about
// to overflow.  Both products accumulate in f32.
//
// The products run on one kernel (vocab_mma_kernel): pairs of CTAs on 256 x 256 tiles with
// tcgen05.mma.cta_group::2 (single CTAs on 128 x 256 for small batches), operands by bulk tensor copies through a ring of stages, two accumulators in tensor
// memory so that the epilogue of a tile runs under the next tile's instructions.  The operands are taken
// as they lie in memory, contiguous along the summed axis or across it: no transposition.
//
// 4096 x 65536 x 2048, one at a time: logits folded 707 us (1556 Tflop/s), G 733 to 760, dX 749 to 772 (128 tiles on 74 pairs: two rounds), dW 745 to 757;
// bound by the tensor cores, and one after the other by the power they draw (3.2 to 3.6 ms for the four).  64 x 131072 x 4096: the
// weights are read once, in 169 us (6.3 TB/s), bound by HBM.
#include <cuda_fp16.h>
#include <math.h>

#include <type_traits>

#include "kernels.h"
#include "tcgen.cuh"

namespace fb {

constexpr int VT = 256;                                // tile edge of a CTA pair
constexpr int VK = 64;                                 // summed elements of a block
constexpr int V_OPERAND = 128 * VK * 2;                // 128 rows of an operand in one block: 16 KiB
constexpr int V_SLAB = VK * 64 * 2;                    // 64 x 64 block of an operand that is contiguous across the sum
constexpr int V_EPI_BUF = 32 * 128;                    // 32 rows of 128 bytes
constexpr int V_GROUP = 16;                            // row tiles that share the columns' operand before it moves on
constexpr float V_LOG2E = 1.4426950408889634f;
constexpr float V_GSCALE = 8192.f;                     // 2^13, see above
// Longest sum, in blocks of VK, that a logit is accumulated in at once.  The tensor cores truncate the running sum at every
// step, so a logit's error grows with the number of steps and has the logit's sign: over 4096 products the logarithm of the sum was
// 1.4e-6 off relative to itself.  Longer sums run in two accumulators that the epilogue adds, which halves that; both halves of tensor
// memory then belong to one tile, and the next one begins when they have been read.
constexpr int V_ONE_SUM = 32;

enum VocabEpilogue : int {
  VE_SOFTMAX = 0,      // (maximum, sum) of the tile's columns per row, and the target's logit
  VE_GRAD = 1,         // G in binary16
  VE_SLAB = 2,         // f32 partial products, one slab per part of the summed axis
  VE_HALF = 3,         // binary16, times a factor from device memory
  VE_ROWS = 4,         // binary16, times 2^-13 and the row's weight: dX where the sum is in one part
};

// Sixteen epilogue warps, four per SM partition, each with a row and 64 of the tile's columns per thread.  One warp
// per partition cannot hide its own latencies: it issued every 4.5 clocks and took 7400 clocks for a tile of which the
// exponentials need 2048.  Folding stages nothing and leaves room for another stage of operands.
constexpr int V_WARPS = 16, V_COLS = VT / (V_WARPS / 4), V_THREADS = 64 + 32 * V_WARPS;
template <bool PAIR, int EPI> struct VocabShape {
  static constexpr int rows = PAIR ? 256 : 128;                     // of a tile
  static constexpr int room = (EPI == VE_SOFTMAX ? 12 : PAIR ? 10 : 9) * V_OPERAND;      // of the ring of stages
  static constexpr int staging = EPI == VE_SOFTMAX ? 2 * (V_WARPS / 4) * 128 * (int)sizeof(float2) : V_WARPS * V_EPI_BUF;
  static constexpr int smem = room + 1024 /*alignment*/ + 1024 /*barriers*/ + staging;
};

struct VocabArgs {
  int M, N, kblocks;            // extents; the summed axis in blocks of VK
  int nt;                       // columns of a tile: a multiple of 32 up to 256
  int arows;                    // rows of A that a CTA brings per stage
  int block, sub, stages;       // bytes of a block of the sum, blocks of a stage, stages of the ring
  int halves;                   // VE_SOFTMAX: the sum in two accumulators
  int splits, kps;              // parts of the summed axis and the blocks of each
  int tiles_m, tiles_n;
  const int32_t *targets;       // VE_SOFTMAX, VE_GRAD
  int v, v0;                    // size of the vocabulary, first word of the piece
  float2 *part;                 // VE_SOFTMAX: [M][tiles_n] (maximum, sum of exp(logit - maximum))
  float *ztarget;
  float *loss, *lse;            // and the results, where small calls finish them,
  uint32_t *ticket;             // with a word that is 0 between launches
  const float *cexp;            // VE_GRAD: per row the exponent's constant term, or, in small calls, what it comes from
  const float *losses, *lses;
  const float *factor;          // VE_HALF
  const float *w;               // VE_ROWS
  int add;                      // VE_SLAB: add to the slab instead of writing it
  int *failure;
};

constexpr int V_MAX_STAGES = 12;
struct VocabBarriers {
  uint64_t full[V_MAX_STAGES];   // used in the pair's first CTA only
  uint64_t empty[V_MAX_STAGES];
  uint64_t tmem_full[2];
  uint64_t tmem_empty[2];        // used in the pair's first CTA only
  uint64_t met[2][4];            // VE_SOFTMAX: three shares of 32 rows are in shared memory
  uint32_t tmem_base;
  uint32_t last;                 // whether this CTA is the one that ends last
};

// Tiles in the order the pairs take them: V_GROUP row tiles by all column tiles, the rows first.  74 pairs then
// work on about 16 x 5 tiles at a time, whose operands come from HBM once and from L2 for every further tile.
__device__ __forceinline__ void vocab_tile(const VocabArgs &a, uint32_t t, int &split, int &tm, int &tn) {
  const uint32_t per = (uint32_t)a.tiles_m * (uint32_t)a.tiles_n, gsize = (uint32_t)V_GROUP * (uint32_t)a.tiles_n;
  const uint32_t sp = a.splits > 1 ? t / per : 0, r = t - sp * per;
  const uint32_t g = r / gsize, in = r - g * gsize;
  const uint32_t rows = min((uint32_t)V_GROUP, (uint32_t)a.tiles_m - g * V_GROUP);
  const uint32_t n = in / rows;
  split = (int)sp;
  tn = (int)n;
  tm = (int)(g * V_GROUP + in - n * rows);
}

// A row's loss by L neighbouring lanes: fold of its (maximum, sum) pairs, eight per lane in flight; the last step in f64, where a loss near 0 is
// a difference.  All lanes of the warp come here, those of rows that do not exist with valid = false.
__device__ __forceinline__ void row_loss(const float2 *part, int tiles, const float *ztarget, const int32_t *targets, float *loss, float *lse, int64_t row,
                                         bool valid, int64_t v, int L) {
  const int lane = threadIdx.x & (L - 1);
  float m = -INFINITY, s = 0.f;
  for (int t0 = lane; t0 < tiles; t0 += 8 * L) {
    float2 p[8];
#pragma unroll
    for (int j = 0; j < 8; j++) p[j] = valid && t0 + L * j < tiles ? __ldcg(part + row * tiles + t0 + L * j) : make_float2(-INFINITY, 0.f);
    float mn = m;
#pragma unroll
    for (int j = 0; j < 8; j++) mn = fmaxf(mn, p[j].x);
    const float ref = mn == -INFINITY ? 0.f : mn;
    s *= exp2f((m - ref) * V_LOG2E);
#pragma unroll
    for (int j = 0; j < 8; j++) s += p[j].y * exp2f((p[j].x - ref) * V_LOG2E);
    m = mn;
  }
  for (int o = L >> 1; o > 0; o >>= 1) {
    const float pm = __shfl_xor_sync(kFull, m, o), ps = __shfl_xor_sync(kFull, s, o);
    const float mn = fmaxf(m, pm), ref = mn == -INFINITY ? 0.f : mn;
    s = s * exp2f((m - ref) * V_LOG2E) + ps * exp2f((pm - ref) * V_LOG2E);
    m = mn;
  }
  if (lane == 0 && valid) {
    const double l = (double)m + log((double)s);
    const int64_t t = targets[row];
    lse[row] = (float)l;
    loss[row] = t >= 0 && t < v ? (float)(l - (double)__ldcg(ztarget + row)) : 0.f;
  }
}
// Lanes of a row where one CTA makes all losses.
static __host__ __device__ __forceinline__ int join_lanes(int64_t n) {
  int L = 32;
  while (L > 1 && n * L > V_THREADS) L >>= 1;
  return L;
}

// q_i and the constant term of G's exponent.  Near 0 a loss is the logarithm of a sum of f32 numbers that begins with 1 (the target's logit is the
// maximum, and goes out exactly).  It is off by the roundings of a few dozen additions, 2^-24 each, whatever lse is: a q below 2^-22 is as
// good as that.
__device__ __forceinline__ float row_q(float loss) {
  const float least = 0x1p-22f, q = -expm1f(-loss);
  return q < least ? least : q;
}
__device__ __forceinline__ float row_exponent(float loss, float lse) { return 13.f - log2f(row_q(loss)) - lse * V_LOG2E; }

// A_MN / B_MN: the operand is contiguous across the summed axis ([K][M], [K][N]) instead of along it.
// PAIR: two CTAs per tile of 256 rows; otherwise one per tile of 128 rows, for batches of at most 128 tokens.  Of a pair's 256
// rows those would leave half or more to zeros: 64 tokens against 131072 x 4096 weights took 185 us, which is what the tensor
// cores need for 256 rows, where the weights can be read in 164.
// SMALL: folding also makes the losses, G's exponents come from the losses and not from a kernel before it.  Either in every call
// made the loops 2 to 3 % slower, by other registers alone (2048 x 50000 x 256: G 59.7 -> 61.7 us).
template <bool PAIR, bool A_MN, bool B_MN, int EPI, bool SMALL>
__device__ __forceinline__ void vocab_mma_body(const CUtensorMap &tmA, const CUtensorMap &tmB, const CUtensorMap &tmC, const VocabArgs &a, uint32_t block,
                                               uint32_t blocks) {
  constexpr int MT = VocabShape<PAIR, EPI>::rows, ROOM = VocabShape<PAIR, EPI>::room;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  VocabBarriers *bars = reinterpret_cast<VocabBarriers *>(smem + ROOM);
  uint8_t *epi = smem + ROOM + 1024;

  const int tid = threadIdx.x, warp = __shfl_sync(kFull, tid >> 5, 0), lane = tid & 31;
  const uint32_t rank = PAIR ? cluster_ctarank() : 0;
  const uint32_t pair = PAIR ? block >> 1 : block, npairs = PAIR ? blocks >> 1 : blocks;
  const uint32_t num_tiles = (uint32_t)a.tiles_m * (uint32_t)a.tiles_n * (uint32_t)a.splits;     // below 2^31

  if (tid == 0) {
    prefetch_map(&tmA);
    prefetch_map(&tmB);
    if (EPI != VE_SOFTMAX) prefetch_map(&tmC);
    for (int s = 0; s < a.stages; s++) { mbar_init(&bars->full[s], 1); mbar_init(&bars->empty[s], 1); }
    for (int i = 0; i < 2; i++) { mbar_init(&bars->tmem_full[i], 1); mbar_init(&bars->tmem_empty[i], (PAIR ? 2 : 1) * V_WARPS); }
    for (int i = 0; i < 8; i++) mbar_init(&bars->met[i >> 2][i & 3], V_WARPS / 4 - 1);
    fence_mbar_init();
  }
  if (!PAIR && !A_MN) {
    // rows of the tile that no token has are 0, in every stage and from now on: the card runs at its power limit even where HBM is the bound, and
    // products of what else lies there cost clocks (64 x 131072 x 4096, call after call: 197 us, with zeros 190)
    const int per = (128 - a.arows) * 8;
    for (int i = tid; i < a.stages * a.sub * per; i += V_THREADS) {
      const int st = i / per;
      *reinterpret_cast<uint4 *>(smem + st * a.block + a.arows * 128 + (i - st * per) * 16) = make_uint4(0, 0, 0, 0);
    }
    fence_proxy_async_smem();
  }
  if (warp == 1) {
    if (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars->tmem_base)), "r"(512) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      tmem_alloc(&bars->tmem_base, 512);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync_all();                        // both CTAs' barriers exist before either signals the other's
  tc_fence_after();
  const uint32_t tmem_base = bars->tmem_base;
  chain_wait();
  const bool poisoned = ld_failure(a.failure) != FAIL_NONE;

  if (!poisoned) {
    if (warp == 0) {
      // ---------------- producer: this CTA's half of each operand ----------------
      if (elect_one()) {
        auto produce = [&](auto blocks_of_stage) {
          constexpr int SUB = decltype(blocks_of_stage)::value;
          int s = 0;
          uint32_t ph = 0;
          for (uint32_t t = pair; t < num_tiles; t += npairs) {
            int split, tm, tn;
            vocab_tile(a, t, split, tm, tn);
            const int m0 = tm * MT + (int)rank * 128, n0 = tn * a.nt + (int)rank * (a.nt >> 1);
            const int kb1 = min(a.kblocks, (split + 1) * a.kps);
            for (int kb = split * a.kps; kb < kb1; kb += SUB) {
              if (!mbar_wait_bounded(&bars->empty[s], ph ^ 1)) return false;
              uint64_t *full = &bars->full[s];
              const uint32_t full0 = PAIR ? map_to_cta(smem_u32(full), 0) : 0;
              auto load = [&](void *dst, const CUtensorMap *tm, int x, int y) {
                if (PAIR) tma_load_3d_pair(dst, tm, x, y, 0, full0);
                else tma_load_3d(dst, tm, x, y, 0, full);
              };
              // both CTAs' bytes
              if (rank == 0) mbar_expect_tx(full, min(SUB, kb1 - kb) * ((PAIR ? 2 : 1) * a.arows + a.nt) * (VK * 2));
#pragma unroll
              for (int u = 0; u < SUB; u++) {
                if (kb + u >= kb1) break;
                uint8_t *sa = smem + (s * SUB + u) * a.block, *sb = sa + V_OPERAND;
                const int k0 = (kb + u) * VK;
                if (A_MN) {
                  load(sa, &tmA, m0, k0);
                  load(sa + V_SLAB, &tmA, m0 + 64, k0);
                } else {
                  load(sa, &tmA, k0, m0);
                }
                if (B_MN) {
                  const int slabs = a.nt / (PAIR ? 128 : 64);
                  for (int j = 0; j < slabs; j++) load(sb + j * V_SLAB, &tmB, n0 + j * 64, k0);
                } else {
                  load(sb, &tmB, k0, n0);
                }
              }
              if (++s == a.stages) { s = 0; ph ^= 1; }
            }
          }
          return true;
        };
        const bool ok = a.sub == 2 ? produce(std::integral_constant<int, 2>()) : produce(std::integral_constant<int, 1>());
        if (!ok) atomicCAS(a.failure, FAIL_NONE, FAIL_MMA_TIMEOUT);
      }
    } else if (warp == 1) {
      // ---------------- MMA issuer: one thread of the first CTA ----------------
      if (rank == 0 && elect_one()) {
        // D = f32, A = B = f16, M the tile's rows, N its columns
        const uint32_t idesc = (1u << 4) | ((A_MN ? 1u : 0u) << 15) | ((B_MN ? 1u : 0u) << 16) | ((uint32_t)(a.nt >> 3) << 17) | ((uint32_t)(MT >> 4) << 24);
        // along the sum: rows of 128 bytes, 8-row groups 1024 bytes apart, a step of 16 is 32 bytes inside the
        // swizzled row; across it: 64-wide slabs (leading), 8-row groups 1024 bytes apart, a step is 16 rows
        const uint32_t sa = smem_u32(smem), sb = sa + V_OPERAND;
        const uint64_t adesc0 = A_MN ? make_smem_desc(sa, V_SLAB, 1024) : make_smem_desc(sa, 16, 1024);
        const uint64_t bdesc0 = B_MN ? make_smem_desc(sb, V_SLAB, 1024) : make_smem_desc(sb, 16, 1024);
        auto issue = [&](auto blocks_of_stage) {
          constexpr int SUB = decltype(blocks_of_stage)::value;
          const uint32_t step = a.block >> 4;              // of a block, in a descriptor
          int s = 0;
          uint32_t ph = 0, tile_it = 0;
          uint64_t adesc = adesc0, bdesc = bdesc0;
          for (uint32_t t = pair; t < num_tiles; t += npairs, tile_it++) {
            int split, tm, tn;
            vocab_tile(a, t, split, tm, tn);
            const bool halves = EPI == VE_SOFTMAX && a.halves;
            const uint32_t acc = halves ? 0 : tile_it & 1, acc_ph = (halves ? tile_it : tile_it >> 1) & 1;
            if (!mbar_wait_bounded(&bars->tmem_empty[acc], acc_ph ^ 1)) return false;
            tc_fence_after();
            uint32_t d_tmem = tmem_base + acc * VT, more = 0;
            const int kb0 = split * a.kps, kb1 = min(a.kblocks, kb0 + a.kps), turn = halves ? (kb0 + kb1) / 2 : kb1;
            for (int kb = kb0; kb < kb1; kb += SUB) {
              if (!mbar_wait_bounded(&bars->full[s], ph)) return false;
              tc_fence_after();
#pragma unroll
              for (int u = 0; u < SUB; u++) {
                if (kb + u >= kb1) break;
                if (kb + u == turn) { d_tmem += VT; more = 0; }      // the second half starts from nothing
                const uint64_t au = adesc + (uint64_t)(u * step), bu = bdesc + (uint64_t)(u * step);
#pragma unroll
                for (int k = 0; k < VK / 16; k++) {
                  const uint64_t ad = au + (uint64_t)(k * (A_MN ? 128 : 2)), bd = bu + (uint64_t)(k * (B_MN ? 128 : 2));
                  if (PAIR) tc2_mma_f16(d_tmem, ad, bd, idesc, k > 0 ? 1u : more);
                  else tc_mma_f16(d_tmem, ad, bd, idesc, k > 0 ? 1u : more);
                }
                more = 1;
              }
              if (PAIR) tc2_commit_both(&bars->empty[s]);
              else tc_commit(&bars->empty[s]);
              adesc += SUB * step;
              bdesc += SUB * step;
              if (++s == a.stages) { s = 0; ph ^= 1; adesc = adesc0; bdesc = bdesc0; }
            }
            if (PAIR) tc2_commit_both(&bars->tmem_full[acc]);
            else tc_commit(&bars->tmem_full[acc]);
          }
          return true;
        };
        const bool ok = a.sub == 2 ? issue(std::integral_constant<int, 2>()) : issue(std::integral_constant<int, 1>());
        if (!ok) atomicCAS(a.failure, FAIL_NONE, FAIL_MMA_TIMEOUT);
      }
    } else {
      // ---------------- epilogue: this CTA's 128 rows of the tile, one row and V_COLS columns per thread ----------------
      const int quarter = warp & 3, share = (warp - 2) >> 2, cbase = share * V_COLS;
      uint32_t tile_it = 0;
      bool ok = true;
      uint8_t *stg = epi + (warp - 2) * V_EPI_BUF;
      const float factor = EPI == VE_HALF ? *a.factor : 1.f;
      // what a tile needs of its row is fetched while the tile before it is worked on
      int tm = 0, tn = 0, split = 0, next_target = -1;
      float next_c = 0.f;
      constexpr bool PER_ROW = EPI == VE_SOFTMAX || EPI == VE_GRAD || EPI == VE_ROWS;
      auto fetch = [&](uint32_t t, int &sp, int &m, int &n) {
        if (t >= num_tiles) return;
        vocab_tile(a, t, sp, m, n);
        const int r = m * MT + (int)rank * 128 + quarter * 32 + lane;
        if (PER_ROW && r < a.M) {
          next_target = a.targets[r];
          if (EPI == VE_GRAD) next_c = SMALL ? row_exponent(a.losses[r], a.lses[r]) : a.cexp[r];
          if (EPI == VE_ROWS) next_c = a.w[r];
        }
      };
      fetch(pair, split, tm, tn);
      for (uint32_t t = pair; t < num_tiles && ok; t += npairs, tile_it++) {
        const int row0 = tm * MT + (int)rank * 128 + quarter * 32, n0 = tn * a.nt;
        const int row = row0 + lane;
        const bool halves = EPI == VE_SOFTMAX && a.halves;
        const uint32_t acc = halves ? 0 : tile_it & 1, acc_ph = (halves ? tile_it : tile_it >> 1) & 1;
        const int ncols = min(a.nt, a.N - n0);
        int tcol = -1;                                     // the target's column in this tile, if it has it
        const float c = next_c;
        const bool counts = next_target >= 0 && next_target < a.v && row < a.M;
        if ((EPI == VE_SOFTMAX || EPI == VE_GRAD) && counts) {
          const int tl = next_target - a.v0 - n0;
          if (tl >= 0 && tl < ncols) tcol = tl;
        }
        const int this_split = split, this_tn = tn;
        if (!__all_sync(kFull, mbar_wait_bounded(&bars->tmem_full[acc], acc_ph))) { ok = false; break; }
        tc_fence_after();
        fetch(t + npairs, split, tm, tn);
        const uint32_t taddr0 = tmem_base + ((uint32_t)(quarter * 32) << 16) + acc * VT;
        float m = -INFINITY, sum = 0.f;

        // 32 columns of a row: running maximum and sum.  The maximum is subtracted before the scaling: scaled first it would be rounded,
        // by up to |m| 2^-24, which leaves the exponents' range for logits above 2^30
        auto fold = [&](uint32_t (&v)[32], int c0) {
          if (c0 >= ncols) return;
          if (c0 + 32 > ncols) {
#pragma unroll
            for (int j = 0; j < 32; j++) if (c0 + j >= ncols) v[j] = 0xff800000u;     // columns that do not exist
          }
          float mx[4];
#pragma unroll
          for (int j = 0; j < 4; j++) mx[j] = __uint_as_float(v[j]);
#pragma unroll
          for (int j = 4; j < 32; j++) mx[j & 3] = fmaxf(mx[j & 3], __uint_as_float(v[j]));
          const float cm = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
          const float mn = fmaxf(m, cm);
          const float ref = mn == -INFINITY ? 0.f : mn;    // a row of -inf so far: the sum stays 0
          const float2 scale = make_float2(V_LOG2E, V_LOG2E), nr = make_float2(-ref, -ref);
          float2 s0 = make_float2(sum * ex2((m - ref) * V_LOG2E), 0.f), s1 = make_float2(0.f, 0.f);
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            const float2 e = mul2(add2(make_float2(__uint_as_float(v[j]), __uint_as_float(v[j + 1])), nr), scale);
            const float2 f = mul2(add2(make_float2(__uint_as_float(v[j + 2]), __uint_as_float(v[j + 3])), nr), scale);
            s0 = add2(s0, make_float2(ex2(e.x), ex2(e.y)));
            s1 = add2(s1, make_float2(ex2(f.x), ex2(f.y)));
          }
          sum = (s0.x + s0.y) + (s1.x + s1.y);
          m = mn;
          const int tj = tcol - c0;
          if (tj >= 0 && tj < 32) {
            float zt = 0.f;
#pragma unroll
            for (int j = 0; j < 32; j++) if (j == tj) zt = __uint_as_float(v[j]);
            a.ztarget[row] = zt;
          }
        };
        // 32 columns of G (or of the scaled product) as 16 pairs of binary16
        auto to_half = [&](const uint32_t (&v)[32], int c0, uint32_t (&h)[16]) {
          const bool none = (EPI == VE_GRAD || EPI == VE_ROWS) && !counts;
          const float2 by = EPI == VE_GRAD ? make_float2(V_LOG2E, V_LOG2E) : EPI == VE_ROWS ? make_float2(c, c) : make_float2(factor, factor);
          const __half2 most = __float2half2_rn(65504.f);
#pragma unroll
          for (int j = 0; j < 16; j++) {
            float2 f = make_float2(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]));
            __half2 p;
            if (EPI == VE_GRAD) {
              f = fma2(f, by, make_float2(c, c));
              p = __hmin2_nan(__floats2half2_rn(ex2(f.x), ex2(f.y)), most);        // NaN stays
            } else {
              if (EPI == VE_ROWS) f = mul2(f, make_float2(1.f / V_GSCALE, 1.f / V_GSCALE));
              f = mul2(f, by);
              p = __floats2half2_rn(f.x, f.y);
            }
            h[j] = none ? 0u : *reinterpret_cast<const uint32_t *>(&p);
          }
          if (EPI == VE_GRAD) {
            const int tj = tcol - c0;
            if (tj >= 0 && tj < 32) {                      // the target's, exactly
              const uint32_t g = __half_as_ushort(__float2half_rn(-V_GSCALE));
#pragma unroll
              for (int j = 0; j < 16; j++) {
                if (tj == 2 * j) h[j] = (h[j] & 0xffff0000u) | g;
                if (tj == 2 * j + 1) h[j] = (h[j] & 0x0000ffffu) | (g << 16);
              }
            }
          }
        };
        // 128 bytes of a row are staged as the 128-byte swizzle wants them (16-byte piece q of row r at q ^ (r & 7))
        // and leave by one bulk tensor store, which has read the buffer before it is written again.
        auto half_pieces = [&](const uint32_t (&h)[16], int q0) {
#pragma unroll
          for (int q = 0; q < 4; q++)
            *reinterpret_cast<uint4 *>(stg + lane * 128 + (((q0 + q) ^ (lane & 7)) << 4)) =
                make_uint4(h[4 * q], h[4 * q + 1], h[4 * q + 2], h[4 * q + 3]);
        };
        auto acquire = [&] {
          if (lane == 0) bulk_wait_read0();
          __syncwarp();
        };
        auto release = [&](int c0) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            if (c0 < ncols) {                              // the tile's, and not behind the last column
              if (EPI == VE_SLAB && a.add) tma_add_3d(&tmC, stg, n0 + c0, row0, this_split);
              else tma_store_3d(&tmC, stg, n0 + c0, row0, this_split);
            }
            bulk_commit();
          }
        };
        auto slab = [&](const uint32_t (&v)[32], int c0) {
          acquire();
#pragma unroll
          for (int q = 0; q < 8; q++)
            *reinterpret_cast<uint4 *>(stg + lane * 128 + ((q ^ (lane & 7)) << 4)) = make_uint4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
          release(c0);
        };

        // the accumulator may be written again
        auto give_back = [&] {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if (PAIR) mbar_arrive_pair(map_to_cta(smem_u32(&bars->tmem_empty[acc]), 0));
            else mbar_arrive(&bars->tmem_empty[acc]);
          }
        };
        const bool mine = row0 < a.M && cbase < ncols;     // uniform over the warp
        if (halves && !mine) give_back();
        if (mine) {
          uint32_t va[32], vb[32];
          tmem_ld_32x32(taddr0 + cbase, va);
          if (halves) {                                    // each 32 columns from both accumulators
            tmem_ld_32x32(taddr0 + VT + cbase, vb);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; j++) va[j] = __float_as_uint(__uint_as_float(va[j]) + __uint_as_float(vb[j]));
            fold(va, cbase);
            tmem_ld_32x32(taddr0 + cbase + 32, va);
            tmem_ld_32x32(taddr0 + VT + cbase + 32, vb);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; j++) vb[j] = __float_as_uint(__uint_as_float(va[j]) + __uint_as_float(vb[j]));
            give_back();
          } else {
            tmem_ld_wait();
            tmem_ld_32x32(taddr0 + cbase + 32, vb);
            if (EPI == VE_SOFTMAX) fold(va, cbase);
            else if (EPI == VE_SLAB) slab(va, cbase);
            else { uint32_t h[16]; to_half(va, cbase, h); acquire(); half_pieces(h, 0); }
            tmem_ld_wait();
          }
          if (EPI == VE_SOFTMAX) fold(vb, cbase + 32);
          else if (EPI == VE_SLAB) slab(vb, cbase + 32);
          else { uint32_t h[16]; to_half(vb, cbase + 32, h); half_pieces(h, 4); release(cbase); }
        }
        if (EPI == VE_SOFTMAX) {
          // the four shares of a row meet in shared memory, at the first one's warp.  The tile after the next one uses the same
          // places: it begins when this warp has given back the next tile's accumulator, or this one's where there are two
          float2 *meet = reinterpret_cast<float2 *>(epi) + (tile_it & 1) * (V_WARPS / 4) * 128 + quarter * 32 + lane;
          if (share != 0) {
            meet[share * 128] = make_float2(m, sum);
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->met[tile_it & 1][quarter]);
          } else {
            if (!__all_sync(kFull, mbar_wait_bounded(&bars->met[tile_it & 1][quarter], (tile_it >> 1) & 1))) { ok = false; break; }
#pragma unroll
            for (int w = 1; w < V_WARPS / 4; w++) {
              const float2 o = meet[w * 128];
              const float mn = fmaxf(m, o.x), ref = mn == -INFINITY ? 0.f : mn;
              sum = sum * ex2((m - ref) * V_LOG2E) + o.y * ex2((o.x - ref) * V_LOG2E);
              m = mn;
            }
          }
        }
        if (!halves) give_back();
        if (EPI == VE_SOFTMAX && share == 0 && row < a.M) a.part[(int64_t)row * a.tiles_n + this_tn] = make_float2(m, sum);
      }
      if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
      if (!ok) atomicCAS(a.failure, FAIL_NONE, FAIL_MMA_TIMEOUT);
    }
  }
  // ---------------- teardown: every thread of both CTAs arrives here, whatever happened ----------------
  // A role that gave up has waited its whole limit after the last copy it issued; stores are waited for above.
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_meet();                            // nobody signals into a partner that has left
  if (EPI == VE_SOFTMAX && SMALL) {
    // the CTA that ends last makes the losses
    if (tid == 0) {
      __threadfence();
      bars->last = atomicAdd(a.ticket, 1u) == blocks - 1;
    }
    __syncthreads();
    if (bars->last) {
      __threadfence();
      const int L = join_lanes(a.M), row = tid / L;      // in one turn
      if (L == 32) row_loss(a.part, a.tiles_n, a.ztarget, a.targets, a.loss, a.lse, row, row < a.M, a.v, 32);
      else row_loss(a.part, a.tiles_n, a.ztarget, a.targets, a.loss, a.lse, row, row < a.M, a.v, L);
      if (tid == 0) *a.ticket = 0;
    }
  }
  if (warp == 1) {
    tc_fence_after();
    if (!PAIR) tmem_dealloc(tmem_base, 512);
    else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512) : "memory");
  }
}

struct VocabRows {
  const __half *x;
  int64_t n, dp, v;
  const int32_t *targets;
  const float *loss, *lse, *dl;
  int *tops;                                         // E of the rows of each of `top_ctas` CTAs of a kernel before
  int top_ctas;                                      // 0: there was none
  float *w, *factor;
  float *cexp;                                       // or nullptr
  __half *out;
};
// w_i = dl_i q_i and the constant term of G's exponent; false for a token without a target
__device__ __forceinline__ bool row_weight(const VocabRows &a, int64_t i, float &w, float &c) {
  const int64_t t = a.targets[i];
  const float ls = a.loss[i], l = a.lse[i], d = a.dl[i];
  const bool counts = t >= 0 && t < a.v;
  w = counts ? d * row_q(ls) : 0.f;
  c = counts ? row_exponent(ls, l) : 0.f;
  return counts;
}
// E over all rows takes a kernel of its own, since every scaled element waits for it (2.3 us: 777 x 32003 x 1000 gradient 175 instead of 173 us
// with an E that need not look at X).  Where X is at most this many elements, the CTAs that need E find it for themselves: gradient of
// 16 x 500 x 64 13 instead of 16 us, 100 x 2000 x 360 19.8 instead of 18.5, 1000 x 1000 x 200 71 instead of 17.
constexpr int64_t V_OWN_TOPS = 32768;
constexpr int V_NO_TOP = -1000;                      // below the exponent of any product of an f32 and a binary16 number
constexpr int V_TOP_THREADS = 256, V_TOP_CTAS = 8;   // CTAs per SM
// The largest exponent of |X_ij w_i| that `warps` warps find, this one the `warp`-th: 1024 elements of a row at a time, so that few
// long rows are shared out too.  Elements and weights that are not finite do not count: what they lead to is not finite either.
__device__ __forceinline__ int rows_top(const VocabRows &a, int64_t warp, int64_t warps) {
  const int lane = threadIdx.x & 31;
  const int64_t per = a.dp / 8, chunks = (per + 127) / 128, items = a.n * chunks;
  int top = V_NO_TOP;
  for (int64_t at = warp; at < items; at += warps) {
    const int64_t i = at / chunks, c = (at - i * chunks) * 128 + lane;
    const uint4 *x = reinterpret_cast<const uint4 *>(a.x + i * a.dp);
    uint4 v[4];
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = c + 32 * j < per ? x[c + 32 * j] : make_uint4(0, 0, 0, 0);
    float w, ci;
    row_weight(a, i, w, ci);
    if (w == 0.f || !isfinite(w)) continue;          // uniform over the warp
    uint32_t m = 0;                                  // bit patterns of sizes order like the sizes
    auto pair = [&](uint32_t u) { u &= 0x7fff7fffu; m = __vmaxu2(m, u & __vcmpltu2(u, 0x7c007c00u)); };
#pragma unroll
    for (int j = 0; j < 4; j++) { pair(v[j].x); pair(v[j].y); pair(v[j].z); pair(v[j].w); }
    m = __reduce_max_sync(kFull, max(m & 0xffffu, m >> 16));
    if (m != 0) top = max(top, ilogb((double)fabsf(w) * (double)__half2float(__ushort_as_half((unsigned short)m))));   // the product is exact
  }
  return top;
}
template <int THREADS>
__device__ __forceinline__ int cta_max(int x) {
  __shared__ int of_warp[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  x = __reduce_max_sync(kFull, x);
  if (lane == 0) of_warp[warp] = x;
  __syncthreads();
  return __reduce_max_sync(kFull, of_warp[lane < THREADS / 32 ? lane : 0]);
}
__global__ void __launch_bounds__(V_TOP_THREADS) vocab_tops_kernel(const VocabRows a) {
  constexpr int warps = V_TOP_THREADS / 32;
  chain_wait();
  const int top = cta_max<V_TOP_THREADS>(rows_top(a, (int64_t)blockIdx.x * warps + (threadIdx.x >> 5), (int64_t)gridDim.x * warps));
  if (threadIdx.x == 0) a.tops[blockIdx.x] = top;
}
// Per row w_i, the exponent's constant, and X_i w_i 2^(14-E) in binary16 (0 without a target), a warp per row, whose first one is on its way
// while E is found.  *factor = 2^(E-14-13).
template <int THREADS>
__device__ __forceinline__ void vocab_rows(const VocabRows &a, uint32_t block, uint32_t blocks) {
  constexpr int warps = THREADS / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t per = a.dp / 8, first = (int64_t)block * warps + warp;
  chain_wait();
  uint4 ahead[4];                                    // of the warp's first row, while E is found
#pragma unroll
  for (int j = 0; j < 4; j++)
    if (first < a.n && lane + 32 * j < per) ahead[j] = reinterpret_cast<const uint4 *>(a.x + first * a.dp)[lane + 32 * j];
  int top = V_NO_TOP;
  if (a.top_ctas == 0) top = rows_top(a, warp, warps);
  else for (int i = threadIdx.x; i < a.top_ctas; i += THREADS) top = max(top, a.tops[i]);
  top = cta_max<THREADS>(top);
  const int e = top == V_NO_TOP ? 14 : top;
  if (block == 0 && threadIdx.x == 0) *a.factor = ldexpf(1.f, e - 14 - 13);
  for (int64_t i = first; i < a.n; i += (int64_t)blocks * warps) {
    float wi, ci;
    const bool counts = row_weight(a, i, wi, ci);
    if (lane == 0) {
      a.w[i] = wi;
      if (a.cexp != nullptr) a.cexp[i] = ci;
    }
    float f = ldexpf(wi, 14 - e);
    if (isinf(f) && isfinite(wi)) f = copysignf(3.4e38f, wi);        // of a row of zeros, which stay zeros
    const uint4 *x = reinterpret_cast<const uint4 *>(a.x + i * a.dp);
    uint4 *out = reinterpret_cast<uint4 *>(a.out + i * a.dp);
    auto scaled = [&](const uint4 &v) {
      __align__(16) __half h[8];
      *reinterpret_cast<uint4 *>(h) = v;
#pragma unroll
      for (int j = 0; j < 8; j++) h[j] = __float2half_rn(__half2float(h[j]) * f);
      return counts ? *reinterpret_cast<const uint4 *>(h) : make_uint4(0, 0, 0, 0);
    };
    if (i == first) {
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (lane + 32 * j < per) out[lane + 32 * j] = scaled(ahead[j]);
    }
    for (int64_t c = lane + (i == first ? 128 : 0); c < per; c += 128) {
      uint4 some[4];                                 // all in flight before the first is written
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (c + 32 * j < per) some[j] = x[c + 32 * j];
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (c + 32 * j < per) out[c + 32 * j] = scaled(some[j]);
    }
  }
}
constexpr int V_ROW_THREADS = 1024;
__global__ void __launch_bounds__(V_ROW_THREADS) vocab_rows_kernel(const VocabRows a) { vocab_rows<V_ROW_THREADS>(a, blockIdx.x, gridDim.x); }

template <bool PAIR, bool A_MN, bool B_MN, int EPI, bool SMALL = false>
__global__ void __cluster_dims__(PAIR ? 2 : 1, 1, 1) __launch_bounds__(V_THREADS, 1)
vocab_mma_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                 const __grid_constant__ CUtensorMap tmC, const VocabArgs a) {
  vocab_mma_body<PAIR, A_MN, B_MN, EPI, SMALL>(tmA, tmB, tmC, a, blockIdx.x, gridDim.x);
}

// G of a small call, and in the CTAs behind the first `blocks`, which it leaves idle, the rows' weights and the scaled X that the products need.
template <bool PAIR>
__global__ void __cluster_dims__(PAIR ? 2 : 1, 1, 1) __launch_bounds__(V_THREADS, 1)
vocab_grad_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmG,
                  const VocabArgs a, const uint32_t blocks, const VocabRows r) {
  if (blockIdx.x < blocks) vocab_mma_body<PAIR, false, false, VE_GRAD, true>(tmX, tmW, tmG, a, blockIdx.x, blocks);
  else vocab_rows<V_THREADS>(r, blockIdx.x - blocks, gridDim.x - blocks);
}

// Both products of a small call side by side: dX in the first `blocks` CTAs, dW in the others.
template <int EPI>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(V_THREADS, 1)
vocab_products_kernel(const __grid_constant__ CUtensorMap tmGk, const __grid_constant__ CUtensorMap tmWn, const __grid_constant__ CUtensorMap tmX,
                      const VocabArgs ax, const uint32_t blocks, const __grid_constant__ CUtensorMap tmGm, const __grid_constant__ CUtensorMap tmXn,
                      const __grid_constant__ CUtensorMap tmD, const VocabArgs aw) {
  if (blockIdx.x < blocks) vocab_mma_body<true, false, true, EPI, true>(tmGk, tmWn, tmX, ax, blockIdx.x, blocks);
  else vocab_mma_body<true, true, true, VE_HALF, true>(tmGm, tmXn, tmD, aw, blockIdx.x - blocks, gridDim.x - blocks);
}

// ---- the small kernels around it ------------------------------------------------------------------
__global__ void __launch_bounds__(256)
vocab_loss_kernel(const float2 *part, int tiles, const float *ztarget, const int32_t *targets,
                  float *loss, float *lse, int64_t n, int64_t v) {
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  chain_wait();
  row_loss(part, tiles, ztarget, targets, loss, lse, row, row < n, v, 32);
}

// Rows of up to two matrices in another pitch, what is behind the narrower of the two 0 or left out; 8 elements of a result per thread.
struct PitchJob {
  const __half *in;
  __half *out;
  int64_t rows;
};
__global__ void __launch_bounds__(256)
vocab_pitch_kernel(const PitchJob a, const PitchJob b, int64_t in_cols, int64_t out_cols) {
  const int64_t first = (a.rows * out_cols + 7) / 8, groups = first + (b.rows * out_cols + 7) / 8;
  chain_wait();
  for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < groups; at += (int64_t)gridDim.x * 256) {
    const PitchJob &job = at < first ? a : b;
    const int64_t o = (at < first ? at : at - first) * 8, total = job.rows * out_cols;
    int64_t i = total < (1ll << 32) ? (int64_t)((uint32_t)o / (uint32_t)out_cols) : o / out_cols, c = o - i * out_cols;
    __align__(16) __half h[8];
    const int64_t src = i * in_cols + c;
    if (c + 8 <= in_cols && c + 8 <= out_cols && src > 0 && src + 9 <= job.rows * in_cols) {
      // 8 neighbours from any place: the words they lie in, shifted by half a word where they start in the middle of one
      const uint32_t *w = reinterpret_cast<const uint32_t *>((uintptr_t)(job.in + src) & ~(uintptr_t)3);
      const bool odd = ((uintptr_t)(job.in + src) & 2) != 0;
      uint32_t *hw = reinterpret_cast<uint32_t *>(h);
      uint32_t lo = w[0];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const uint32_t next = j < 3 || odd ? w[j + 1] : 0u;
        hw[j] = odd ? __funnelshift_r(lo, next, 16) : lo;
        lo = next;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++) {
        h[j] = c < in_cols && o + j < total ? job.in[i * in_cols + c] : __half(0.f);
        if (++c == out_cols) { c = 0; i++; }
      }
    }
    if (o + 8 <= total && ((uintptr_t)(job.out + o) & 15) == 0) *reinterpret_cast<uint4 *>(job.out + o) = *reinterpret_cast<const uint4 *>(h);
    else for (int j = 0; j < 8 && o + j < total; j++) job.out[o + j] = h[j];
  }
}

// dX_i = 2^-13 w_i times the sum of the slabs, in f32, rounded once.
__global__ void __launch_bounds__(256)
vocab_dx_kernel(const float *slabs, int splits, int64_t n, int64_t d, int64_t dp, const int32_t *targets, int64_t v,
                const float *w, __half *dx) {
  const int64_t per = dp / 4, total = n * per;
  chain_wait();
  for (int64_t o = (int64_t)blockIdx.x * 256 + threadIdx.x; o < total; o += (int64_t)gridDim.x * 256) {
    const int64_t i = o / per, c = (o - i * per) * 4;
    const int64_t t = targets[i];
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (t >= 0 && t < v) {
      for (int k = 0; k < splits; k++) {
        const float4 p = *reinterpret_cast<const float4 *>(slabs + ((int64_t)k * n + i) * dp + c);
        s.x += p.x; s.y += p.y; s.z += p.z; s.w += p.w;
      }
      const float f = w[i];
      constexpr float g = 1.f / V_GSCALE;
      s.x *= g; s.y *= g; s.z *= g; s.w *= g;
      s.x *= f; s.y *= f; s.z *= f; s.w *= f;
    }
    const __half2 lo = __floats2half2_rn(s.x, s.y), hi = __floats2half2_rn(s.z, s.w);
    if (d == dp) {
      uint2 r;
      r.x = *reinterpret_cast<const uint32_t *>(&lo); r.y = *reinterpret_cast<const uint32_t *>(&hi);
      *reinterpret_cast<uint2 *>(dx + i * d + c) = r;
    } else {
      if (c + 0 < d) dx[i * d + c + 0] = __low2half(lo);
      if (c + 1 < d) dx[i * d + c + 1] = __high2half(lo);
      if (c + 2 < d) dx[i * d + c + 2] = __low2half(hi);
      if (c + 3 < d) dx[i * d + c + 3] = __high2half(hi);
    }
  }
}

__global__ void __launch_bounds__(256)
vocab_fill_kernel(float *loss, float *lse, int64_t n, float l) {
  chain_wait();
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) { loss[i] = 0.f; lse[i] = l; }
}

// ---- host side ------------------------------------------------------------------------------------------
static inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
static inline size_t align256(size_t b) { return (b + 255) & ~(size_t)255; }
static inline int elementwise_grid(int64_t items, int num_sms) {
  const int64_t g = ceil_div(items, 256);
  return (int)(g < 1 ? 1 : g < (int64_t)num_sms * 16 ? g : (int64_t)num_sms * 16);
}

// Batches of at most 128 tokens go to single CTAs, where the tokens are the rows of the product.
static inline bool small_batch(int64_t n) { return n <= 128; }
// Whether the contraction's last CTA makes the losses: in one turn, which costs
// less than a kernel's launch (200 x 2000 x 512 forward: 17.1 us instead of 19.2).  Two turns cost more: 1000 x 2000 x 512, 20.4 to 21.9 us instead of 19.5.
static bool last_makes_losses(int64_t n, int64_t tiles_n) {
  const int64_t L = join_lanes(n);
  return ceil_div(n, V_THREADS / L) * ceil_div(tiles_n, 8 * L) <= 1;
}
// The ring: blocks of 128 rows of the first operand and a CTA's share of the tile's columns, in stages of two blocks where there is room for four of
// those.  Half as many barriers and commits then: 1000 x 1000 x 8192 forward 28 us instead of 33.  With fewer stages than that they come too
// late: three of two blocks instead of six took 3.9 ms instead of 3.75 for 4096 x 65536 x 2048.
static inline int block_bytes(bool pair, int cols) { return V_OPERAND + (pair ? cols / 2 : cols) * VK * 2; }
static inline int ring_blocks(int room, int block) { return room / block >= 8 ? 2 : 1; }
static inline int ring_stages(int room, int stage) { return room / stage < V_MAX_STAGES ? room / stage : V_MAX_STAGES; }
// Clocks of a block of 64 summed elements of a tile of `cols` columns: on pairs 512 for 256 columns at the tensor cores'
// rate and a fifth of that for the rows' operand; on single CTAs what 148 of them leave each other of HBM, 24 bytes per clock.
// However narrow the tile, a block takes its issuer 330, in stages of two blocks 230.
static inline double block_clocks(bool pair, int cols) {
  const double c = pair ? (cols + 64) * 1.6 : cols * 5.3, least = ring_blocks(10 * V_OPERAND, block_bytes(pair, cols)) == 2 ? 230 : 330;
  return c < least ? least : c;
}

// Columns of a tile.  A tile of fewer columns reuses its rows less, but a number of tiles that is just above a multiple of
// the number of CTAs or pairs leaves most of them idle in the last round; and where there are few tiles, narrow ones put more CTAs to work (down to
// 32 instead of 128 columns: 8 x 4000 x 8192 forward 25.5 us instead of 33, 1317 x 271 x 2729 in both directions 59 instead of 62).  `losses`: a
// kernel that folds more partial results than the last CTA does in a turn costs 8000.
static int tile_columns(bool pair, int64_t rows, int64_t cols, int64_t kblocks, int step, int least, bool losses, int num_sms) {
  int best = VT;
  double best_cost = 0;
  const int64_t workers = pair ? num_sms / 2 : num_sms;
  for (int nt = VT; nt >= least; nt -= step) {
    const int64_t tiles = ceil_div(rows, pair ? 256 : 128) * ceil_div(cols, nt);
    const double cost = (double)ceil_div(tiles, workers) * (kblocks * block_clocks(pair, nt) + 1500.0) +
                        (losses && !last_makes_losses(rows, ceil_div(cols, nt)) ? 8000.0 : 0.0);
    if (nt == VT || cost < 0.97 * best_cost) { best = nt; best_cost = cost; }
  }
  return best;
}

// Parts of the summed axis of dX = G W.  A small batch has fewer tiles than there are SMs, while its sum runs over the
// vocabulary; each part costs a slab of f32 written and read again.  The estimate is in clocks, as above, with
// 3000 per tile for its epilogue where nothing hides it, 6000 for the kernel that adds the slabs and 3600 bytes of HBM per clock.
static int dx_splits(bool pair, int64_t workers, int64_t n, int64_t dp, int64_t kblocks, int *nt) {
  int best = 1;
  double best_cost = 0;
  for (int w = VT; w >= 128; w -= 128) {
    const int64_t tiles = ceil_div(n, pair ? 256 : 128) * ceil_div(dp, w);
    const int most = (int)(kblocks < 128 ? kblocks : 128);
    for (int want = 1; want <= most && (want == 1 || tiles * want < 4 * workers); want += 1 + want / 8) {
      const int64_t kps = ceil_div(kblocks, want), s = ceil_div(kblocks, kps);      // parts that all have something to add
      const double cost = (double)ceil_div(tiles * s, workers) * (kps * block_clocks(pair, w) + 3000.0) + (s > 1 ? 6000.0 + (double)s * n * dp * 8 / 3600.0 : 0.0);
      if ((want == 1 && w == VT) || cost < best_cost) { best = (int)s; *nt = w; best_cost = cost; }
    }
  }
  return best;
}

VocabPlan vocab_plan(int64_t n, int64_t v, int64_t d, bool x_aligned, bool w_aligned, bool grad, int num_sms) {
  VocabPlan p = {};
  if (n <= 0 || v <= 0 || (grad && d <= 0)) return p;           // nothing will run
  p.dp = d <= 0 ? 8 : (d + 7) & ~(int64_t)7;
  const bool padded = p.dp != d;
  const bool pair = !small_batch(n);
  size_t off = 0;
  auto take = [&](size_t bytes) { const size_t at = off; off += align256(bytes); return at; };
  p.copy_x = padded || !x_aligned;
  p.copy_w = padded || !w_aligned;
  p.xp = p.copy_x ? take((size_t)(n * p.dp) * 2) : 0;
  p.wp = p.copy_w ? take((size_t)(v * p.dp) * 2) : 0;
  if (!grad) {
    p.nt = tile_columns(pair, n, v, ceil_div(p.dp, VK), 32, 32, true, num_sms);
    p.part = take((size_t)(n * ceil_div(v, p.nt)) * sizeof(float2));
    p.zt = take((size_t)n * 4);
  } else {
    // pieces of the vocabulary whose part of G is at most 1 GiB: 65536 words for 8192 tokens
    const int64_t most = (int64_t)1 << 29;
    const int64_t want = ceil_div(v, VT) * VT;
    int64_t words = most / (n > 0 ? n : 1) / VT * VT;
    if (words < VT) words = VT;
    if (words > want) words = want;
    p.piece = ceil_div(ceil_div(v, ceil_div(v, words)), VT) * VT;       // equal pieces
    p.nt = tile_columns(pair, n, p.piece < v ? p.piece : v, ceil_div(p.dp, VK), 64, 64, false, num_sms);
    p.pieces = (int)ceil_div(v, p.piece);
    p.ntw = tile_columns(true, p.piece < v ? p.piece : v, p.dp, ceil_div(n, VK), 128, 128, false, num_sms);
    // Small calls: what the products need besides G is made beside it, and the products side by side, on CTAs that have nothing else
    // to do.  Both products are then pairs' work, since all tensor-core instructions of a kernel are of one kind.  Both directions of 16 x 500
    // x 64 take 34 us instead of 38.5, 1000 x 1000 x 200 36.5 instead of 40.5, 500 x 8000 x 1024 60.5 instead of 65.5.
    const int64_t gtiles = ceil_div(n, pair ? 256 : 128) * ceil_div(v, p.nt), gctas = pair ? 2 * gtiles : gtiles;
    const int64_t rctas = ceil_div(n, V_THREADS / 32), idle = pair ? (num_sms - gctas) / 2 * 2 : num_sms - gctas, wtiles = ceil_div(v, VT) * ceil_div(p.dp, p.ntw), pairs = num_sms / 2;
    const int64_t want_rows = pair ? (rctas + 1) / 2 * 2 : rctas;
    p.row_ctas = p.pieces == 1 && rctas <= 4 * idle ? (int)(want_rows < idle ? want_rows : idle) : 0;
    p.together = p.pieces == 1 && wtiles + ceil_div(n, VT) * ceil_div(p.dp, VT) <= pairs;
    const int64_t free = p.together ? pairs - wtiles : pair ? pairs : num_sms;
    p.splits = dx_splits(pair || p.together, free, n, p.dp, ceil_div(p.piece < v ? p.piece : v, VK), &p.ntd);
    p.w = take((size_t)n * 4);
    p.cexp = take((size_t)n * 4);
    p.scalars = take(256);
    const int64_t top_ctas = ceil_div(n * ceil_div(p.dp, 1024), V_TOP_THREADS / 32), most_tops = (int64_t)num_sms * V_TOP_CTAS;
    p.top_ctas = n * p.dp <= V_OWN_TOPS ? 0 : (int)(top_ctas < most_tops ? top_ctas : most_tops);
    p.tops = take((size_t)p.top_ctas * 4);
    p.xs = take((size_t)(n * p.dp) * 2);
    p.g = take((size_t)(n * p.piece) * 2);
    p.direct = p.splits == 1 && p.pieces == 1;
    if (p.direct) p.dxp = padded ? take((size_t)(n * p.dp) * 2) : 0;
    else p.slabs = take((size_t)p.splits * (size_t)(n * p.dp) * 4);
    p.dwp = padded ? take((size_t)((p.piece < v ? p.piece : v) * p.dp) * 2) : 0;
  }
  p.bytes = off;
  return p;
}

// Fills in the tiles of a product; the CTAs that work on them, of at most `most`.
static int tile_ctas(bool pair, int room, VocabArgs &a, int most) {
  a.block = block_bytes(pair, a.nt);
  a.sub = ring_blocks(room, a.block);
  a.stages = ring_stages(room, a.block * a.sub);
  a.tiles_m = (int)ceil_div(a.M, pair ? 256 : 128);
  a.tiles_n = (int)ceil_div(a.N, a.nt);
  a.kps = (int)ceil_div(a.kblocks, a.splits);
  const int64_t tiles = (int64_t)a.tiles_m * a.tiles_n * a.splits, workers = pair ? most / 2 : most;
  return (int)(tiles < workers ? tiles : workers) * (pair ? 2 : 1);
}
template <bool PAIR, bool A_MN, bool B_MN, int EPI, bool SMALL = false>
static cudaError_t launch_tiles(const CUtensorMap &tmA, const CUtensorMap &tmB, const CUtensorMap &tmC, VocabArgs a, int num_sms, cudaStream_t stream) {
  constexpr int smem = VocabShape<PAIR, EPI>::smem;
  auto kernel = vocab_mma_kernel<PAIR, A_MN, B_MN, EPI, SMALL>;
  static unsigned long long allowed = 0;
  const cudaError_t err = allow_smem(reinterpret_cast<const void *>(kernel), smem, allowed);
  if (err != cudaSuccess) return err;
  const int ctas = tile_ctas(PAIR, VocabShape<PAIR, EPI>::room, a, num_sms);
  return launch_after(kernel, (unsigned)ctas, V_THREADS, smem, stream, tmA, tmB, tmC, a);
}
template <bool PAIR>
static cudaError_t launch_grad(const CUtensorMap &tmX, const CUtensorMap &tmW, const CUtensorMap &tmG, VocabArgs a, const VocabRows &rows, int row_ctas,
                               int num_sms, cudaStream_t stream) {
  constexpr int smem = VocabShape<PAIR, VE_GRAD>::smem;
  static unsigned long long allowed = 0;
  const cudaError_t err = allow_smem(reinterpret_cast<const void *>(vocab_grad_kernel<PAIR>), smem, allowed);
  if (err != cudaSuccess) return err;
  const int ctas = tile_ctas(PAIR, VocabShape<PAIR, VE_GRAD>::room, a, num_sms);
  return launch_after(vocab_grad_kernel<PAIR>, (unsigned)(ctas + row_ctas), V_THREADS, smem, stream, tmX, tmW, tmG, a, (uint32_t)ctas, rows);
}
template <int EPI>
static cudaError_t launch_products(const CUtensorMap &tmGk, const CUtensorMap &tmWn, const CUtensorMap &tmX, VocabArgs ax, const CUtensorMap &tmGm,
                                   const CUtensorMap &tmXn, const CUtensorMap &tmD, VocabArgs aw, int num_sms, cudaStream_t stream) {
  constexpr int sx = VocabShape<true, EPI>::smem, sw = VocabShape<true, VE_HALF>::smem, smem = sx > sw ? sx : sw;
  static unsigned long long allowed = 0;
  const cudaError_t err = allow_smem(reinterpret_cast<const void *>(vocab_products_kernel<EPI>), smem, allowed);
  if (err != cudaSuccess) return err;
  const int wctas = tile_ctas(true, VocabShape<true, VE_HALF>::room, aw, num_sms), xctas = tile_ctas(true, VocabShape<true, EPI>::room, ax, num_sms - wctas);
  return launch_after(vocab_products_kernel<EPI>, (unsigned)(xctas + wctas), V_THREADS, smem, stream, tmGk, tmWn, tmX, ax, (uint32_t)xctas, tmGm, tmXn, tmD, aw);
}
// products whose rows are tokens
template <bool B_MN, int EPI, bool SMALL = false>
static cudaError_t launch_tokens(const CUtensorMap &tmA, const CUtensorMap &tmB, const CUtensorMap &tmC, const VocabArgs &a, int num_sms, cudaStream_t stream) {
  return small_batch(a.M) ? launch_tiles<false, false, B_MN, EPI, SMALL>(tmA, tmB, tmC, a, num_sms, stream)
                          : launch_tiles<true, false, B_MN, EPI, SMALL>(tmA, tmB, tmC, a, num_sms, stream);
}

// an operand [rows][cols] of row pitch `pitch`, in boxes of 64 columns and `box` rows: 64 where it is read across the sum
static bool operand_map(CUtensorMap *tm, const void *base, int64_t rows, int64_t cols, int64_t pitch, int box) {
  return make_tensor_map(tm, base, (uint64_t)cols, (uint64_t)rows, 1, (uint64_t)pitch, (uint64_t)pitch * rows, 64, (uint32_t)box);
}
// Rows of the tokens' operand that a CTA brings per stage.  A small batch brings no more than there are (whole groups
// of 8, as the swizzle has them): what shared memory holds below is the product of rows that no one reads.
static int token_rows(int64_t n) { return small_batch(n) ? (int)(n + 7) / 8 * 8 : 128; }
// Columns of a tile of logits that a CTA brings.
static int word_rows(int64_t n, int nt) { return small_batch(n) ? nt : nt / 2; }

static PitchJob pitch_job(const uint16_t *in, uint16_t *out, int64_t rows) {
  return {reinterpret_cast<const __half *>(in), reinterpret_cast<__half *>(out), rows};
}
static cudaError_t repitch(const PitchJob &a, const PitchJob &b, int64_t in_cols, int64_t out_cols, int num_sms, cudaStream_t stream) {
  const int64_t groups = ((a.rows + b.rows) * out_cols + 7) / 8;
  if (groups <= 0) return cudaSuccess;
  return launch_after(vocab_pitch_kernel, elementwise_grid(groups, num_sms), 256, 0, stream, a, b, in_cols, out_cols);
}
// The operands where the tensor cores can read them.
static cudaError_t operands(const VocabPlan &p, uint8_t *ws, const uint16_t *&x, const uint16_t *&w, int64_t n, int64_t v, int64_t d, int num_sms,
                            cudaStream_t stream) {
  uint16_t *xp = reinterpret_cast<uint16_t *>(ws + p.xp), *wp = reinterpret_cast<uint16_t *>(ws + p.wp);
  const cudaError_t err = repitch(pitch_job(x, xp, p.copy_x ? n : 0), pitch_job(w, wp, p.copy_w ? v : 0), d, p.dp, num_sms, stream);
  if (p.copy_x) x = xp;
  if (p.copy_w) w = wp;
  return err;
}

#define FB_TRY(e) do { const cudaError_t fb_err = (e); if (fb_err != cudaSuccess) return fb_err; } while (0)

cudaError_t launch_vocab_xent(const VocabPlan &p, void *workspace, void *ticket, const uint16_t *x, const uint16_t *w, const int32_t *targets, float *loss,
                              float *lse, int64_t n, int64_t v, int64_t d, int *failure, int num_sms, cudaStream_t stream) {
  if (n <= 0) return cudaSuccess;
  if (v <= 0) {                                   // the sum of nothing
    return launch_after(vocab_fill_kernel, elementwise_grid(n, num_sms), 256, 0, stream, loss, lse, n, -INFINITY);
  }
  uint8_t *ws = reinterpret_cast<uint8_t *>(workspace);
  FB_TRY(operands(p, ws, x, w, n, v, d, num_sms, stream));
  CUtensorMap tmX, tmW;
  VocabArgs a = {};
  a.M = (int)n; a.N = (int)v; a.kblocks = (int)ceil_div(p.dp, VK); a.splits = 1;
  a.nt = p.nt;
  a.arows = token_rows(n);
  a.halves = a.kblocks > V_ONE_SUM;
  if (!operand_map(&tmX, x, n, p.dp, p.dp, a.arows) || !operand_map(&tmW, w, v, p.dp, p.dp, word_rows(n, a.nt))) return cudaErrorInvalidValue;
  a.targets = targets; a.v = (int)v; a.v0 = 0;
  a.part = reinterpret_cast<float2 *>(ws + p.part);
  a.ztarget = reinterpret_cast<float *>(ws + p.zt);
  a.failure = failure;
  a.loss = loss; a.lse = lse; a.ticket = reinterpret_cast<uint32_t *>(ticket);
  if (last_makes_losses(n, ceil_div(v, p.nt))) return launch_tokens<false, VE_SOFTMAX, true>(tmX, tmW, tmX, a, num_sms, stream);
  FB_TRY((launch_tokens<false, VE_SOFTMAX>(tmX, tmW, tmX, a, num_sms, stream)));
  return launch_after(vocab_loss_kernel, (unsigned)ceil_div(n, 8), 256, 0, stream, a.part, (int)ceil_div(v, p.nt), a.ztarget, targets, loss, lse, n, v);
}

cudaError_t launch_vocab_xent_grad(const VocabPlan &p, void *workspace, const uint16_t *x, const uint16_t *w, const int32_t *targets,
                                   const float *loss, const float *lse, const float *dl, uint16_t *dx, uint16_t *dw, int64_t n, int64_t v,
                                   int64_t d, int *failure, int num_sms, cudaStream_t stream) {
  if (n <= 0 || v <= 0 || d <= 0) {               // what there is of the results is a sum of nothing
    if (n > 0 && d > 0) FB_TRY(cudaMemsetAsync(dx, 0, (size_t)(n * d) * 2, stream));
    if (v > 0 && d > 0) FB_TRY(cudaMemsetAsync(dw, 0, (size_t)(v * d) * 2, stream));
    return cudaSuccess;
  }
  uint8_t *ws = reinterpret_cast<uint8_t *>(workspace);
  float *rw = reinterpret_cast<float *>(ws + p.w), *slabs = reinterpret_cast<float *>(ws + p.slabs), *factor = reinterpret_cast<float *>(ws + p.scalars);
  float *cexp = p.row_ctas == 0 ? reinterpret_cast<float *>(ws + p.cexp) : nullptr;
  uint16_t *xs = reinterpret_cast<uint16_t *>(ws + p.xs), *g = reinterpret_cast<uint16_t *>(ws + p.g);
  FB_TRY(operands(p, ws, x, w, n, v, d, num_sms, stream));
  const VocabRows rows = {reinterpret_cast<const __half *>(x), n, p.dp, v, targets, loss, lse, dl, reinterpret_cast<int *>(ws + p.tops), p.top_ctas,
                          rw, factor, cexp, reinterpret_cast<__half *>(xs)};
  if (p.top_ctas > 0) FB_TRY(launch_after(vocab_tops_kernel, p.top_ctas, V_TOP_THREADS, 0, stream, rows));
  if (p.row_ctas == 0) {
    const int64_t row_ctas = ceil_div(n, V_ROW_THREADS / 32), most = (int64_t)num_sms * (2048 / V_ROW_THREADS);
    FB_TRY(launch_after(vocab_rows_kernel, (unsigned)(row_ctas < most ? row_ctas : most), V_ROW_THREADS, 0, stream, rows));
  }
  uint16_t *dxo = p.dp == d ? dx : reinterpret_cast<uint16_t *>(ws + p.dxp);
  const bool small = small_batch(n);
  const int xrows = small && !p.together ? token_rows(n) : 128;      // of dX's first operand
  for (int64_t v0 = 0; v0 < v; v0 += p.piece) {
    const int64_t vw = v - v0 < p.piece ? v - v0 : p.piece;
    CUtensorMap tmX, tmW, tmG, tmGk, tmWn, tmS, tmGm, tmXn, tmD;
    uint16_t *dwo = p.dp == d ? dw + v0 * d : reinterpret_cast<uint16_t *>(ws + p.dwp);
    VocabArgs a = {};
    const bool ok = operand_map(&tmX, x, n, p.dp, p.dp, token_rows(n)) && operand_map(&tmW, w + v0 * p.dp, vw, p.dp, p.dp, word_rows(n, p.nt)) &&
                    make_tensor_map(&tmG, g, (uint64_t)vw, (uint64_t)n, 1, (uint64_t)p.piece, (uint64_t)p.piece * n, 64, 32) &&
                    operand_map(&tmGk, g, n, vw, p.piece, xrows) && operand_map(&tmWn, w + v0 * p.dp, vw, p.dp, p.dp, 64) &&
                    (p.direct ? make_tensor_map(&tmS, dxo, (uint64_t)p.dp, (uint64_t)n, 1, (uint64_t)p.dp, (uint64_t)(p.dp * n), 64, 32)
                              : make_tensor_map(&tmS, slabs, (uint64_t)p.dp, (uint64_t)n, (uint64_t)p.splits, (uint64_t)p.dp, (uint64_t)(p.dp * n), 32, 32, true)) &&
                    operand_map(&tmGm, g, n, vw, p.piece, 64) && operand_map(&tmXn, xs, n, p.dp, p.dp, 64) &&
                    make_tensor_map(&tmD, dwo, (uint64_t)p.dp, (uint64_t)vw, 1, (uint64_t)p.dp, (uint64_t)(p.dp * vw), 64, 32);
    if (!ok) return cudaErrorInvalidValue;
    a.failure = failure;
    a.targets = targets; a.v = (int)v; a.v0 = (int)v0; a.cexp = cexp; a.losses = loss; a.lses = lse; a.factor = factor; a.w = rw;
    a.splits = 1;
    a.M = (int)n; a.N = (int)vw; a.kblocks = (int)ceil_div(p.dp, VK); a.nt = p.nt; a.arows = token_rows(n);
    if (p.row_ctas == 0) FB_TRY((launch_tokens<false, VE_GRAD>(tmX, tmW, tmG, a, num_sms, stream)));
    else if (small) FB_TRY(launch_grad<false>(tmX, tmW, tmG, a, rows, p.row_ctas, num_sms, stream));
    else FB_TRY(launch_grad<true>(tmX, tmW, tmG, a, rows, p.row_ctas, num_sms, stream));
    VocabArgs ax = a, aw = a;
    // every part has its blocks in every piece: the last one may be shorter, and then some slabs get nothing more
    ax.N = (int)p.dp; ax.kblocks = (int)ceil_div(vw, VK); ax.nt = p.ntd; ax.arows = xrows;
    ax.splits = (int)ceil_div(ax.kblocks, ceil_div(ax.kblocks, p.splits < ax.kblocks ? p.splits : ax.kblocks));
    ax.add = v0 > 0;
    aw.M = (int)vw; aw.N = (int)p.dp; aw.kblocks = (int)ceil_div(n, VK); aw.arows = 128;
    aw.nt = p.ntw;
    if (p.together) {
      if (p.direct) FB_TRY((launch_products<VE_ROWS>(tmGk, tmWn, tmS, ax, tmGm, tmXn, tmD, aw, num_sms, stream)));
      else FB_TRY((launch_products<VE_SLAB>(tmGk, tmWn, tmS, ax, tmGm, tmXn, tmD, aw, num_sms, stream)));
    } else {
      if (p.direct) FB_TRY((launch_tokens<true, VE_ROWS>(tmGk, tmWn, tmS, ax, num_sms, stream)));
      else FB_TRY((launch_tokens<true, VE_SLAB>(tmGk, tmWn, tmS, ax, num_sms, stream)));
      FB_TRY((launch_tiles<true, true, true, VE_HALF>(tmGm, tmXn, tmD, aw, num_sms, stream)));
    }
    if (p.dp != d) {                               // and with the last piece's a finished dX
      const bool both = p.direct && v0 + vw == v;
      FB_TRY(repitch(pitch_job(dwo, dw + v0 * d, vw), pitch_job(dxo, dx, both ? n : 0), p.dp, d, num_sms, stream));
    }
  }
  if (p.direct) return cudaSuccess;
  return launch_after(vocab_dx_kernel, elementwise_grid(n * p.dp / 4, num_sms), 256, 0, stream, slabs, p.splits, n, d, p.dp, targets, v, rw,
                      reinterpret_cast<__half *>(dx));
}

}  // namespace fb
