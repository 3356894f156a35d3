// Tensor-core product of two MXFP4 matrices for sm_100a: C[M,N] = A[M,K] * B[N,K]^T, fp32 accumulation,
// fp32 / fp16 / bf16 results with an optional bias and ReLU.
//
// tcgen05.mma.kind::mxf4.block_scale multiplies 64 elements of K per instruction and applies the two scale
// bytes of each operand row on the way; the scales come from tensor memory.  Persistent CTAs, one per SM,
// work by warp role:
//   warp 0      TMA producer: 128 bytes of K per row (256 elements) of A and B, 128-byte swizzle, and the two
//               512-byte scale tiles of every band of 128 rows, into a ring of shared-memory stages;
//   warp 1      moves a stage's scale tiles to tensor memory (tcgen05.cp, 32 lanes x 16 bytes broadcast to the
//               four lane quarters, which is the order the scales are stored in) and issues its four MMAs;
//   warps 2-9   epilogue: two warps per lane quarter, each on its own 32 rows: tensor memory -> registers ->
//               32 x 128-byte boxes in shared memory -> TMA stores.
//
// CG = 2: a CTA pair owns a 256 x 256 tile; each CTA stages its 128 rows of A and half the columns of B, and the
// scales of all 256 columns, since either SM's tensor memory has to hold them.
//
// Tensor memory holds 512 columns.  Two 256-column accumulators would fill it, so for 256-wide tiles they
// overlap by 64 columns, which go to the scales: accumulator 0 is columns [0, 256), accumulator 1 [192, 448),
// scale buffers from 448.  The epilogue drains the shared 64 columns first, and the MMAs of the next tile
// start as soon as those are in registers; the rest of the drain is hidden behind them.  Two scale buffers are
// used in turn: the buffer of k-block i is rewritten only after the MMAs of k-block i - 2 have completed
// (their commit is waited for), while those of k-block i - 1 keep the tensor pipe busy.
//
// Bound: what an SM takes in.  A k-block is 35 KB of operands and scales for 512 clocks of MMAs, and an SM pulls about 84 GB/s
// out of L2 whatever the clock, 0.42 us a k-block: 8192^3 to bf16 in 186 us in short bursts (5.9 PFLOP/s; without the loads of
// B 174 us, with half the MMAs 166 us), 215 to 224 us under the power cap.  Three, four and five ring stages: 239, 205, 195 us with
// the clocks read inside; rows per tile-order group 1024 / 2048 / 4096 / 8192 at 8192 x 28672 x 8192, run for seconds, 830 / 799
// / 769 / 769 us.  Scales written to tensor memory by four warps (tcgen05.st) instead of copied: 437 us.
//
// Below it in this file: the kernel for few rows (or columns), the one that splits K for few tiles, and the rules that
// choose.  Every wait is bounded; a wait that runs out raises the CTA's abort flag, all roles drain, tensor memory is
// freed and a status word tells the host that the result is invalid.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstring>
#include <type_traits>
#include <utility>

#include "internal.h"
#include "mxfp4.cuh"
#include "ptx_sm100.cuh"

namespace b200 {
namespace {

__device__ uint32_t g_mx_status = 0;  // a bounded wait ran out: 1 = gemm_mx, 2 = gemm_mx_skinny, 4 = gemm_mx_split

constexpr int kSmemBudget = 227 * 1024;
constexpr int kEpiWarps = 8;
constexpr int kThreads = 64 + 32 * kEpiWarps;
constexpr int kScaleTile = 512;  // bytes of the scales of 128 rows x 4 blocks

// tcgen05.mma.kind::mxf4 instruction descriptor: [4,6) scale id of B, [7,10) and [10,12) operand formats (1 =
// e2m1), [17,23) N >> 3, 23 scale format (1 = e8m0), [24,29) M >> 4, [29,31) scale id of A.  A scale id is the byte
// of the four-byte word (128 elements of K) at which the instruction's two scales begin: 0 or 2.
__host__ __device__ constexpr uint32_t mx_instr_desc(int mma_m, int mma_n, int scale_id) {
  return (uint32_t(scale_id) << 4) | (1u << 7) | (1u << 10) | (uint32_t(mma_n >> 3) << 17) | (1u << 23) |
         (uint32_t(mma_m >> 4) << 24) | (uint32_t(scale_id) << 29);
}

// One lane of a converged warp.  The TMA, copy and MMA loops below are run by whole warps that elect a lane around
// the asynchronous instructions themselves: the compiler then keeps descriptors and addresses in uniform registers.
// With the loops inside a branch on lane 0 every tcgen05.cp cost the issuing lane 45 clocks and every MMA 45 to 60
// (six copies and four MMAs 800 clocks against the 512 that the MMAs run); elected, six copies cost 50 together.
__device__ __forceinline__ bool elect_lane() {
  uint32_t e;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(e));
  return e != 0;
}

// A bounded wait of a whole warp, with one outcome for all its lanes.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile uint32_t* abort_flag, uint64_t budget_ns) {
  return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, abort_flag, budget_ns)) != 0;
}

// Shared-memory descriptors are handed over as their address word alone; the upper words are constants.  kOperandHi:
// rows of 128 bytes, 128-byte swizzle, 1024 bytes between groups of eight rows.  kScaleHi: lines of 16 bytes without a
// swizzle, 128 bytes between groups of eight.
constexpr uint32_t kOperandHi = (1024u >> 4) | (1u << 14) | (2u << 29);
constexpr uint32_t kScaleHi = (128u >> 4) | (1u << 14);
__device__ __forceinline__ uint32_t desc_word(uint32_t smem_addr) { return ((smem_addr & 0x3ffffu) >> 4) | (1u << 16); }

template <int CG>
__device__ __forceinline__ void mx_umma(uint32_t d_tmem, uint32_t a_desc, uint32_t b_desc, uint32_t idesc, uint32_t sa_tmem,
                                        uint32_t sb_tmem, uint32_t accumulate) {
  if constexpr (CG == 2)
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tmov.b64 a, {%1, %7};\n\tmov.b64 b, {%2, %7};\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], a, b, %3, [%4], [%5], p;\n\t}"
        :
        : "r"(d_tmem), "r"(a_desc), "r"(b_desc), "r"(idesc), "r"(sa_tmem), "r"(sb_tmem), "r"(accumulate), "n"(kOperandHi)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tmov.b64 a, {%1, %7};\n\tmov.b64 b, {%2, %7};\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], a, b, %3, [%4], [%5], p;\n\t}"
        :
        : "r"(d_tmem), "r"(a_desc), "r"(b_desc), "r"(idesc), "r"(sa_tmem), "r"(sb_tmem), "r"(accumulate), "n"(kOperandHi)
        : "memory");
}

// One scale tile, shared memory -> four columns of tensor memory (of both CTAs of a pair, each from its own).
template <int CG>
__device__ __forceinline__ void mx_copy_scales(uint32_t tmem, uint32_t desc) {
  if constexpr (CG == 2)
    asm volatile("{\n\t.reg .b64 d;\n\tmov.b64 d, {%1, %2};\n\ttcgen05.cp.cta_group::2.32x128b.warpx4 [%0], d;\n\t}" ::"r"(tmem),
                 "r"(desc), "n"(kScaleHi)
                 : "memory");
  else
    asm volatile("{\n\t.reg .b64 d;\n\tmov.b64 d, {%1, %2};\n\ttcgen05.cp.cta_group::1.32x128b.warpx4 [%0], d;\n\t}" ::"r"(tmem),
                 "r"(desc), "n"(kScaleHi)
                 : "memory");
}

// 3-D tiled load, credited to a barrier of either CTA of a pair (CG = 2) or of this CTA.
template <int CG>
__device__ __forceinline__ void mx_load_3d(void* dst, const CUtensorMap* map, uint32_t bar, int32_t x, int32_t y, int32_t z) {
  if constexpr (CG == 2)
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];"
        :
        : "r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];"
        :
        : "r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}

template <int CG_, int BN_>
struct MxTile {
  static constexpr int CG = CG_;
  static constexpr int BN = BN_;
  static constexpr int TILE_M = 128 * CG;
  static constexpr int BANDS = BN / 128;       // bands of 128 columns whose scales a CTA holds
  static constexpr int A_BYTES = 128 * 128;
  static constexpr int B_BYTES = BN / CG * 128;
  static constexpr int SA_BYTES = 2 * kScaleTile;
  static constexpr int SB_BYTES = BANDS * 2 * kScaleTile;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES + SA_BYTES + SB_BYTES;
  static constexpr int STAGING_BYTES = kEpiWarps * (32 * 128 + 128 * 4);  // a box of 32 rows x 128 bytes and 128 values of the bias
  static constexpr int STAGES_FIT = (kSmemBudget - 2048 - STAGING_BYTES) / STAGE_BYTES;
  static constexpr int STAGES = STAGES_FIT > 6 ? 6 : STAGES_FIT;
  static_assert(STAGES * STAGE_BYTES + STAGING_BYTES + 1024 + 256 <= kSmemBudget, "shared memory");
  static constexpr int SMEM_BYTES = kSmemBudget;  // all of it: who owns all of tensor memory shares the SM with nobody
  static constexpr int ACC_STEP = BN == 256 ? 192 : BN;  // columns from accumulator 0 to accumulator 1
  static constexpr int SCALE_COL = 448;                  // first column of the scale buffers
  static constexpr int SCALE_STEP = 32;                  // columns of one buffer: 8 for A, 8 x BANDS for B
  static constexpr int UNITS = BN / 64;                  // the epilogue works in units of 64 columns
  static_assert(STAGE_BYTES % 1024 == 0 && ACC_STEP + BN <= SCALE_COL && 8 + 8 * BANDS <= SCALE_STEP, "layout");
};

struct MxArgs {
  void* C;
  int64_t ldc;
  int M, N;
  int blocks;  // blocks of 32 along K
  int tiles_m, tiles_n, group_m;
  int tma_store;  // C and its rows are 16-byte aligned
  const float* bias;
  int relu;
  unsigned long long wait_budget_ns;
  int lose_kb;  // test of the give-up path: k-block of CTA 0's first tile that is never loaded; -1 = none
  int splits, kb_per_split;  // gemm_mx_split_kernel: CTAs of a cluster = ranges of K, k-blocks of a range
};

// Groups of group_m tiles of rows; inside a group m runs fastest (a wave of tiles is then a near-square patch).
__device__ __forceinline__ void mx_tile_coords(int t, const MxArgs& p, int& mb, int& nb) {
  const int per_group = p.group_m * p.tiles_n;
  const int g = t / per_group, first_m = g * p.group_m, gm = min(p.tiles_m - first_m, p.group_m), r = t - g * per_group;
  mb = first_m + r % gm;
  nb = r / gm;
}

// 32 accumulators of one row -> 32 (fp32) or 16 output words, with the tail; `bias`: the 32 columns' values.
template <int EPI>
__device__ __forceinline__ void mx_finish(const MxArgs& p, const float* bias, uint32_t (&v)[32],
                                          uint32_t (&w)[EPI == EPI_F32 ? 32 : 16]) {
  if (p.bias != nullptr) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float4 b = reinterpret_cast<const float4*>(bias)[i];
      v[4 * i] = __float_as_uint(__uint_as_float(v[4 * i]) + b.x);
      v[4 * i + 1] = __float_as_uint(__uint_as_float(v[4 * i + 1]) + b.y);
      v[4 * i + 2] = __float_as_uint(__uint_as_float(v[4 * i + 2]) + b.z);
      v[4 * i + 3] = __float_as_uint(__uint_as_float(v[4 * i + 3]) + b.w);
    }
  }
  if (p.relu) {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(fmaxf(0.0f, __uint_as_float(v[i])));
  }
#pragma unroll
  for (int i = 0; i < (EPI == EPI_F32 ? 32 : 16); ++i) {
    if constexpr (EPI == EPI_F32) {
      w[i] = v[i];
    } else if constexpr (EPI == EPI_F16) {
      const __half2 h = __floats2half2_rn(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
}

template <int CG, int BN, int EPI>
__global__ void __launch_bounds__(kThreads, 1)
gemm_mx_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
               const __grid_constant__ CUtensorMap tmap_sa, const __grid_constant__ CUtensorMap tmap_sb,
               const __grid_constant__ CUtensorMap tmap_c, const MxArgs p) {
  using T = MxTile<CG, BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* staging = smem + T::STAGES * T::STAGE_BYTES;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(staging + T::STAGING_BYTES);  // [STAGES] (pair: the leader's)
  uint64_t* empty_bar = full_bar + T::STAGES;                                    // [STAGES]
  uint64_t* acc_full = empty_bar + T::STAGES;                                    // [2]
  uint64_t* acc_go = acc_full + 2;  // the epilogue has drained the columns the next tile needs (pair: the leader's)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_go + 1);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  volatile uint32_t* epi_go_pair = tmem_slot + 2;  // "this tile's accumulator arrived", two words in turn

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t cta_rank = CG == 2 ? cluster_cta_rank() : 0u;
  const int first_tile = CG == 2 ? int(blockIdx.x >> 1) : int(blockIdx.x);
  const int tile_step = CG == 2 ? int(gridDim.x >> 1) : int(gridDim.x);
  const int num_tiles = p.tiles_m * p.tiles_n;
  const int num_kb = (p.blocks + 7) / 8;

  if (threadIdx.x == 0) {
    for (int s = 0; s < T::STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    mbar_init(&acc_full[0], 1);
    mbar_init(&acc_full[1], 1);
    mbar_init(acc_go, kEpiWarps * CG);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmap_a);
    tma_prefetch_desc(&tmap_b);
    tma_prefetch_desc(&tmap_sa);
    tma_prefetch_desc(&tmap_sb);
  }
  if (warp == 1) {
    if constexpr (CG == 2) {
      tmem_alloc_pair(tmem_slot, 512);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_slot, 512);
      tmem_relinquish();
    }
  }
  tc_fence_before_sync();
  if constexpr (CG == 2) cluster_sync_all(); else __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;

  // Nothing above touched global memory: wait for the kernel this launch was serialised behind, and let the
  // next one begin its own set-up.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    int stage = 0, it = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int t = first_tile; t < num_tiles && ok; t += tile_step, ++it) {
      int mb, nb;
      mx_tile_coords(t, p, mb, nb);
      const int m0 = mb * T::TILE_M + int(cta_rank) * 128;
      const int n0 = nb * BN + int(cta_rank) * (BN / CG);
      for (int kb = 0; kb < num_kb; ++kb) {
        if (!warp_wait(&empty_bar[stage], phase ^ 1u, abort_flag, p.wait_budget_ns)) { ok = false; break; }
        const bool lost = kb == p.lose_kb && it == 0 && blockIdx.x == 0;
        if (!lost && elect_lane()) {
          uint8_t* sa = smem + stage * T::STAGE_BYTES;
          uint8_t* sb = sa + T::A_BYTES;
          uint8_t* ssa = sb + T::B_BYTES;
          uint8_t* ssb = ssa + T::SA_BYTES;
          if constexpr (CG == 2) {
            const uint32_t bar = map_to_cta(smem_u32(&full_bar[stage]), 0);
            if (cta_rank == 0) mbar_arrive_expect_tx(&full_bar[stage], 2 * T::STAGE_BYTES);
            tma_load_2d_pair(sa, &tmap_a, bar, kb * 128, m0);
            tma_load_2d_pair(sb, &tmap_b, bar, kb * 128, n0);
            mx_load_3d<CG>(ssa, &tmap_sa, bar, 0, kb * 2, m0 >> 7);
            mx_load_3d<CG>(ssb, &tmap_sb, bar, 0, kb * 2, nb * T::BANDS);
          } else {
            mbar_arrive_expect_tx(&full_bar[stage], T::STAGE_BYTES);
            tma_load_2d(sa, &tmap_a, &full_bar[stage], kb * 128, m0);
            tma_load_2d(sb, &tmap_b, &full_bar[stage], kb * 128, n0);
            mx_load_3d<CG>(ssa, &tmap_sa, smem_u32(&full_bar[stage]), 0, kb * 2, m0 >> 7);
            mx_load_3d<CG>(ssb, &tmap_sb, smem_u32(&full_bar[stage]), 0, kb * 2, nb * T::BANDS);
          }
        }
        __syncwarp();
        if (++stage == T::STAGES) { stage = 0; phase ^= 1u; }
      }
    }
    if constexpr (CG == 2) {
      // Stay until every stage has been released: the releases are arrivals of the leader's commits in this
      // CTA's shared memory, which must still exist.
      for (int i = 0; i < T::STAGES && ok; ++i) {
        ok = warp_wait(&empty_bar[stage], phase ^ 1u, abort_flag, p.wait_budget_ns);
        if (++stage == T::STAGES) { stage = 0; phase ^= 1u; }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ scale copies and MMAs
    if (cta_rank == 0) {
      constexpr uint32_t idesc0 = mx_instr_desc(T::TILE_M, BN, 0), idesc2 = mx_instr_desc(T::TILE_M, BN, 2);
      const uint32_t ring = smem_u32(smem);
      const uint32_t a_desc0 = desc_word(ring);
      const uint32_t b_desc0 = desc_word(ring + T::A_BYTES);
      const uint32_t s_desc0 = desc_word(ring + T::A_BYTES + T::B_BYTES);
      constexpr uint32_t kStageStep = T::STAGE_BYTES >> 4;
      int stage = 0, behind = 0;  // `behind`: the stage of the k-block before the last
      uint32_t phase = 0, behind_phase = 0, count = 0;
      bool ok = true;
      int it = 0;
      for (int t = first_tile; t < num_tiles && ok; t += tile_step, ++it) {
        const int ab = it & 1;
        // the epilogue is done with the tile before the last, and with what the last one shares with this one
        if (!warp_wait(acc_go, uint32_t(it + 1) & 1u, abort_flag, p.wait_budget_ns)) break;
        const uint32_t d_tmem = tmem_base + uint32_t(ab * T::ACC_STEP);
        for (int kb = 0; kb < num_kb; ++kb, ++count) {
          if (!warp_wait(&full_bar[stage], phase, abort_flag, p.wait_budget_ns)) { ok = false; break; }
          if (count >= 2) {
            if (!warp_wait(&empty_bar[behind], behind_phase, abort_flag, p.wait_budget_ns)) { ok = false; break; }
            if (++behind == T::STAGES) { behind = 0; behind_phase ^= 1u; }
          }
          tc_fence_after_sync();
          const uint32_t sa_tmem = tmem_base + uint32_t(T::SCALE_COL) + (count & 1u) * uint32_t(T::SCALE_STEP);
          const uint32_t sb_tmem = sa_tmem + 8;
          const uint32_t s_desc = s_desc0 + uint32_t(stage) * kStageStep;
          const uint32_t a_desc = a_desc0 + uint32_t(stage) * kStageStep;
          const uint32_t b_desc = b_desc0 + uint32_t(stage) * kStageStep;
          const int left = p.blocks - kb * 8;  // blocks of 32 this stage really holds
          if (elect_lane()) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              mx_copy_scales<CG>(sa_tmem + uint32_t(4 * h), s_desc + uint32_t((h * kScaleTile) >> 4));
#pragma unroll
              for (int b = 0; b < T::BANDS; ++b)
                mx_copy_scales<CG>(sb_tmem + uint32_t(h * 4 * T::BANDS + 4 * b),
                                   s_desc + uint32_t((T::SA_BYTES + (2 * b + h) * kScaleTile) >> 4));
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if (2 * j < left)
                mx_umma<CG>(d_tmem, a_desc + uint32_t(2 * j), b_desc + uint32_t(2 * j), (j & 1) ? idesc2 : idesc0,
                            sa_tmem + uint32_t(4 * (j >> 1)), sb_tmem + uint32_t(4 * T::BANDS * (j >> 1)),
                            (kb | j) != 0 ? 1u : 0u);
            }
            if constexpr (CG == 2) umma_commit_pair(&empty_bar[stage], 3); else umma_commit(&empty_bar[stage]);
            if (kb + 1 == num_kb) {
              if constexpr (CG == 2) umma_commit_pair(&acc_full[ab], 3); else umma_commit(&acc_full[ab]);
            }
          }
          __syncwarp();
          if (++stage == T::STAGES) { stage = 0; phase ^= 1u; }
        }
      }
    }
  } else {
    // ------------------------------------------------------------------ epilogue
    constexpr int OUT_BYTES = EPI == EPI_F32 ? 4 : 2;
    constexpr int HALF_CHUNKS = 32 * OUT_BYTES / 16;  // 16-byte chunks of 32 outputs of a row
    constexpr int BOX_COLS = 128 / OUT_BYTES;         // a box: 32 rows of 128 bytes
    constexpr int MINE = T::UNITS / 2;
    const int group = (warp - 2) >> 2;  // two warps per quarter share a tile's units of 64 columns
    const int quarter = warp & 3;       // tensor-memory lanes this warp may read
    uint8_t* box = staging + (warp - 2) * (32 * 128);
    float* bias_buf = reinterpret_cast<float*>(staging + kEpiWarps * 32 * 128) + (warp - 2) * 128;
    auto box_at = [&](int row, int byte) { return box + row * 128 + (((byte >> 4) ^ (row & 7)) << 4) + (byte & 15); };
    int it = 0;
    for (int t = first_tile; t < num_tiles; t += tile_step, ++it) {
      int mb, nb;
      mx_tile_coords(t, p, mb, nb);
      const int ab = it & 1;
      // Group 0 begins with the unit that the other accumulator overlaps (the last one of accumulator 0, the first one
      // of accumulator 1); group 1 has the units between.
      auto unit_of = [&](int i) { return T::UNITS == 2 ? group : (group == 0 ? ((i ^ ab) ? 0 : 3) : 1 + i); };
      if (p.bias != nullptr) {  // on its way while the tile is computed
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 2 * MINE; ++i)
          bias_buf[32 * i + lane] = p.bias[min(nb * BN + unit_of(i >> 1) * 64 + (i & 1) * 32 + lane, p.N - 1)];
        __syncwarp();
      }
      volatile uint32_t* epi_go = epi_go_pair + (it & 1);
      // One warp polls the barrier; all eight agree on the outcome.
      if (warp == 2) {
        const bool ok = mbar_wait_bounded(&acc_full[ab], (it >> 1) & 1, abort_flag, p.wait_budget_ns);
        if (lane == 0) *epi_go = ok ? 1u : 0u;
      }
      named_barrier_sync(2, 32 * kEpiWarps);
      if (*epi_go == 0u) break;
      tc_fence_after_sync();
      const int row0 = mb * T::TILE_M + int(cta_rank) * 128 + quarter * 32;
      const int rows = min(32, p.M - row0);  // may be negative
      const uint32_t taddr = tmem_base + (uint32_t(quarter * 32) << 16) + uint32_t(ab * T::ACC_STEP);
      uint32_t v[2][32];
      tmem_ld_32x32(taddr + uint32_t(unit_of(0) * 64), v[0]);
      tmem_ld_32x32(taddr + uint32_t(unit_of(0) * 64 + 32), v[1]);
#pragma unroll
      for (int i = 0; i < MINE; ++i) {
        tmem_ld_wait();
        if (i == 0) {
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) {
            if constexpr (CG == 2) mbar_arrive_cluster(map_to_cta(smem_u32(acc_go), 0)); else mbar_arrive(acc_go);
          }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int n0 = nb * BN + unit_of(i) * 64 + 32 * h;
          const int c0 = EPI == EPI_F32 ? n0 : n0 - 32 * h, cols = min(BOX_COLS, p.N - c0);  // the box's columns
          uint32_t w[EPI == EPI_F32 ? 32 : 16];
          mx_finish<EPI>(p, bias_buf + 64 * i + 32 * h, v[h], w);
          // the registers are free: the next unit's values may come
          if (i + 1 < MINE) tmem_ld_32x32(taddr + uint32_t(unit_of(i + 1) * 64 + 32 * h), v[h]);
          if (EPI == EPI_F32 || h == 0) {
            if (p.tma_store && lane == 0) tma_store_wait_read<0>();  // this warp's previous store has read the box
            __syncwarp();
          }
          const int chunk0 = EPI == EPI_F32 ? 0 : h * HALF_CHUNKS;
#pragma unroll
          for (int u = 0; u < HALF_CHUNKS; ++u)
            *reinterpret_cast<uint4*>(box_at(lane, 16 * (chunk0 + u))) = make_uint4(w[4 * u], w[4 * u + 1], w[4 * u + 2], w[4 * u + 3]);
          if (EPI != EPI_F32 && h == 0) continue;
          if (p.tma_store) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0 && rows > 0 && cols > 0) {
              tma_store_2d(&tmap_c, box, c0, row0);
              tma_store_commit();
            }
          } else {
            // C or its rows are not 16-byte aligned.  fp32: a row of the box at a time, consecutive lanes consecutive
            // words.  16 bits: four rows at a time, eight lanes a row.  Where a row begins s elements after a 16-byte
            // boundary, lanes 1..7 write the seven whole chunks of 16 bytes that it covers, put together from five words of
            // the box, and the eight elements before and after those go one to a lane.  (Each lane storing its own row,
            // element by element: 230 us for 951 x 23085 with K = 68; a row at a time in words: 54; this 30.)
            __syncwarp();
            char* corner = static_cast<char*>(p.C) + (int64_t(row0) * p.ldc + c0) * OUT_BYTES;
            if constexpr (EPI == EPI_F32) {
#pragma unroll 8
              for (int r = 0; r < 32; ++r)
                if (r < rows && lane < cols)
                  reinterpret_cast<uint32_t*>(corner + int64_t(r) * p.ldc * 4)[lane] = *reinterpret_cast<const uint32_t*>(box_at(r, 4 * lane));
            } else {
#pragma unroll 2
              for (int j = 0; j < 8; ++j) {
                const int r = 4 * j + (lane >> 3), u = lane & 7;
                uint16_t* c16 = reinterpret_cast<uint16_t*>(corner + int64_t(r) * p.ldc * 2);
                const int s = int(reinterpret_cast<uintptr_t>(c16) & 15) >> 1;
                const int e = 8 * u - s;  // lanes 1..7: first element of the chunk
                uint32_t words[5];
#pragma unroll
                for (int k = 0; k < 5; ++k)
                  words[k] = *reinterpret_cast<const uint32_t*>(box_at(r, min(max(2 * (e & ~1), 0) + 4 * k, 124)));
                if (r < rows) {
                  if (u > 0) {
                    uint32_t out[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) out[k] = s & 1 ? __funnelshift_r(words[k], words[k + 1], 16) : words[k];
                    if (e + 8 <= cols) {
                      *reinterpret_cast<uint4*>(c16 + e) = make_uint4(out[0], out[1], out[2], out[3]);
                    } else {
#pragma unroll
                      for (int k = 0; k < 8; ++k)
                        if (e + k < cols) c16[e + k] = uint16_t(out[k >> 1] >> ((k & 1) * 16));
                    }
                  }
                  const int single = u < 8 - s ? u : 56 + u;
                  if (single < cols) c16[single] = *reinterpret_cast<const uint16_t*>(box_at(r, 2 * single));
                }
              }
            }
          }
        }
      }
    }
    if (lane == 0 && p.tma_store) tma_store_wait_all<0>();
  }

  // Every role gets here: either its loop ended or its wait was abandoned.
  __syncwarp();
  __syncthreads();
  if (*abort_flag) {
    if (threadIdx.x == 0) atomicOr(&g_mx_status, 1u);
    // Give copies and MMAs still in flight time to land before shared and tensor memory go away.
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 2000000ull) __nanosleep(1000);
  }
  tc_fence_before_sync();
  if constexpr (CG == 2) cluster_sync_all(); else __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    if constexpr (CG == 2) tmem_dealloc_pair(tmem_base, 512); else tmem_dealloc(tmem_base, 512);
  }
}

// ------------------------------------------------------------------------------ few rows of A
//
// A product of at most 32 rows of A streams B (the weights) and computes little.  Here the weights are the 128-row
// operand of the MMA and the rows of A ("tokens", padded to 16) its N dimension, so no instruction is spent on rows
// that do not exist, and an accumulator lane is one output feature.  A tile of 128 features is shared by a cluster of
// S CTAs, one range of K each, so that every SM streams; the partial sums meet through distributed shared
// memory: each CTA of the cluster finishes 128 / S features, adding the ranges in K order.
//
// SRC = 1, 2, 3: the tokens arrive as fp32, fp16 or bf16 rows and fourteen warps quantise this CTA's range of them into
// shared memory, in the order the MMA reads, while the weights are on their way: one launch for a layer.
// SRC = 0: they arrive packed and travel through the ring with the weights.
//
// A product of few COLUMNS of C (few rows of B) is the same with the operands in each other's place.
//
// Warp 0 issues the loads, warp 1 the scale copies and MMAs, the others quantise, all take part in the tail.  The scale
// buffers in tensor memory are those of the ring's stages, so a buffer is rewritten only after the stage's MMAs.

enum { SRC_PACKED = 0, SRC_F32 = 1, SRC_F16 = 2, SRC_BF16 = 3 };
constexpr int kSkQuantWarps = 14;
__host__ __device__ constexpr int sk_threads(int src) { return src == SRC_PACKED ? 256 : 64 + 32 * kSkQuantWarps; }
constexpr int kSkMaxStages = 12;
constexpr int kSkMaxPieces = 16;  // pieces of 512 elements in a CTA's range of a token
// (Figures of the few-row and split kernels in this file: bf16, calls in a row in a CUDA graph, weights from HBM.)
// Rows of A the kernel takes.  Against the kernels for 128 x 128 tiles, us: [11008, 4096] weights, 1 row 7.8 / 12.3, 16 rows 10.1 /
// 12.2, 32 rows 11.3 / 11.3, 64 rows 16.0 / 10.0; [4096, 4096], 32 rows 7.6 / 7.5; [4096, 11008], 64 rows 14.3 / 10.1.
constexpr int kSkRows = 32;
// Rows that the kernel quantises itself, which every tile of features does again, against a quantiser's launch before it.
// One launch / two, us: 1 row [11008, 4096] 8.0 / 11.2, 16 rows 12.2 / 14.4; 16 rows [4096, 11008] 10.6 / 12.3; 32 rows
// [4096, 4096] 9.3 / 10.6, [1024, 1024] 7.5 / 9.2; 64 rows [1024, 1024] 10.5 / 7.4; 1 row [28672, 8192], more tiles than SMs,
// 41.2 / 24.5.  So: up to 16 rows, up to 32 of a limited number of elements, where every tile has an SM.
constexpr int kSkFusedRows = 16;
constexpr int64_t kSkFusedElements = 131072, kSkFusedN = 148 * 128;
constexpr int64_t kSkFusedK = 65536;      // ... and their length: an eighth of it fits in shared memory
constexpr int kWeightBytes = 128 * 128;     // 128 features x 256 elements
constexpr int kWeightScales = 2 * kScaleTile;

struct MxSkinnyArgs {
  void* C;
  const void* X;  // rows of A as they are (SRC != 0)
  int64_t ldc;
  int M, N, K;
  int blocks;          // blocks of 32 along K
  int tokens;          // M rounded up to 16
  int splits;          // CTAs of a cluster = ranges of K
  int kb_per_split;    // k-blocks (256 elements) per range; the last range may be shorter, never empty
  int stages;
  int tmem_cols;
  int scale_col;       // first column of the scale buffers (16 columns each)
  int x_vec;           // rows of X are 16-byte aligned
  const float* bias;
  int relu;
  int swapped;         // the two operands have changed places: lanes are rows of C, columns its columns
  unsigned long long wait_budget_ns;
  int lose_kb;
};

template <int SRC> struct SkSource { using type = float; };
template <> struct SkSource<SRC_F16> { using type = __half; };
template <> struct SkSource<SRC_BF16> { using type = __nv_bfloat16; };

__device__ __forceinline__ void st_cluster_v4(uint32_t cluster_addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(cluster_addr), "r"(a), "r"(b), "r"(c), "r"(d)
               : "memory");
}
__device__ __forceinline__ void st_cluster_u32(uint32_t cluster_addr, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr), "r"(v) : "memory");
}

// Output of token `m`, feature `n`.
template <int EPI>
__device__ __forceinline__ void sk_store(const MxSkinnyArgs& p, int m, int n, float y) {
  if (p.swapped) {
    const int t = m;
    m = n;
    n = t;
  }
  if (p.bias != nullptr) y += p.bias[n];
  if (p.relu) y = fmaxf(0.0f, y);
  const int64_t at = int64_t(m) * p.ldc + n;
  if constexpr (EPI == EPI_F32) static_cast<float*>(p.C)[at] = y;
  else if constexpr (EPI == EPI_F16) static_cast<__half*>(p.C)[at] = __float2half_rn(y);
  else static_cast<__nv_bfloat16*>(p.C)[at] = __float2bfloat16_rn(y);
}

template <int SRC, int EPI>
__global__ void __launch_bounds__(sk_threads(SRC), 2)
gemm_mx_skinny_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_sw,
                      const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_sx,
                      const MxSkinnyArgs p) {
  using X = typename SkSource<SRC>::type;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int tokens = p.tokens, S = p.splits;
  const int token_bytes = tokens * 128;  // one k-block of the tokens
  // ring: weights | tokens (packed source only) | weight scales | token scales (packed source only)
  const int stage_bytes = kWeightBytes + kWeightScales + (SRC == SRC_PACKED ? token_bytes + 2 * kScaleTile : 0);
  const int scale_ofs = kWeightBytes + (SRC == SRC_PACKED ? token_bytes : 0);
  uint8_t* xq = smem + p.stages * stage_bytes;  // quantised tokens: [k-block][tokens][128 bytes], then their scales
  uint8_t* xs = xq + (SRC == SRC_PACKED ? 0 : p.kb_per_split * token_bytes);
  float* exch = reinterpret_cast<float*>(xs + (SRC == SRC_PACKED ? 0 : p.kb_per_split * 2 * kScaleTile));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(exch) + (S > 1 ? 128 * tokens * 4 : 0));
  uint64_t* empty_bar = full_bar + kSkMaxStages;
  uint64_t* acc_full = empty_bar + kSkMaxStages;
  uint64_t* x_ready = acc_full + 1;  // [kSkMaxPieces]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(x_ready + kSkMaxPieces);
  volatile uint32_t* abort_flag = tmem_slot + 1;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = S > 1 ? cluster_cta_rank() : 0u;
  const int tile = int(blockIdx.x) / S;
  const int n0 = tile * 128;
  const int num_kb = (p.blocks + 7) / 8;
  const int kb0 = int(rank) * p.kb_per_split;
  const int kb_count = min(p.kb_per_split, num_kb - kb0);

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    mbar_init(acc_full, 1);
    if constexpr (SRC != SRC_PACKED)
      for (int i = 0; i < kSkMaxPieces; ++i) mbar_init(&x_ready[i], uint32_t(p.M));
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmap_w);
    tma_prefetch_desc(&tmap_sw);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, uint32_t(p.tmem_cols));
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncwarp();
  if (S > 1) cluster_sync_all(); else __syncthreads();  // every CTA of the cluster runs from here on
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;

  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  if (warp == 0) {
    // ------------------------------------------------------------------ loads
    int stage = 0;
    uint32_t phase = 0;
    for (int i = 0; i < kb_count; ++i) {
      if (!warp_wait(&empty_bar[stage], phase ^ 1u, abort_flag, p.wait_budget_ns)) break;
      const int kb = kb0 + i;
      const bool lost = kb == p.lose_kb && blockIdx.x == 0;
      if (!lost && elect_lane()) {
        uint8_t* sw = smem + stage * stage_bytes;
        uint8_t* ss = sw + scale_ofs;
        mbar_arrive_expect_tx(&full_bar[stage], uint32_t(stage_bytes));
        tma_load_2d(sw, &tmap_w, &full_bar[stage], kb * 128, n0);
        mx_load_3d<1>(ss, &tmap_sw, smem_u32(&full_bar[stage]), 0, kb * 2, tile);
        if constexpr (SRC == SRC_PACKED) {
          tma_load_2d(sw + kWeightBytes, &tmap_x, &full_bar[stage], kb * 128, 0);
          mx_load_3d<1>(ss + kWeightScales, &tmap_sx, smem_u32(&full_bar[stage]), 0, kb * 2, 0);
        }
      }
      __syncwarp();
      if (++stage == p.stages) { stage = 0; phase ^= 1u; }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ scale copies and MMAs
    const uint32_t idesc0 = mx_instr_desc(128, tokens, 0), idesc2 = mx_instr_desc(128, tokens, 2);
    const uint32_t ring = smem_u32(smem);
    const uint32_t w_desc0 = desc_word(ring);
    const uint32_t x_desc0 = desc_word(SRC == SRC_PACKED ? ring + kWeightBytes : smem_u32(xq));
    const uint32_t sw_desc0 = desc_word(ring + uint32_t(scale_ofs));
    const uint32_t sx_desc0 = desc_word(SRC == SRC_PACKED ? ring + uint32_t(scale_ofs + kWeightScales) : smem_u32(xs));
    const uint32_t w_step = uint32_t(stage_bytes >> 4);
    const uint32_t x_step = SRC == SRC_PACKED ? w_step : uint32_t(token_bytes >> 4);
    const uint32_t sx_step = SRC == SRC_PACKED ? w_step : uint32_t((2 * kScaleTile) >> 4);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int i = 0; i < kb_count && ok; ++i) {
      if constexpr (SRC != SRC_PACKED) {
        if ((i & 1) == 0 && !warp_wait(&x_ready[i >> 1], 0, abort_flag, p.wait_budget_ns)) { ok = false; break; }
      }
      if (!warp_wait(&full_bar[stage], phase, abort_flag, p.wait_budget_ns)) { ok = false; break; }
      tc_fence_after_sync();
      const int at = SRC == SRC_PACKED ? stage : i;
      const uint32_t sa_tmem = tmem_base + uint32_t(p.scale_col + stage * 16);
      const uint32_t sb_tmem = sa_tmem + 8;
      const uint32_t w_desc = w_desc0 + uint32_t(stage) * w_step, sw_desc = sw_desc0 + uint32_t(stage) * w_step;
      const uint32_t x_desc = x_desc0 + uint32_t(at) * x_step, sx_desc = sx_desc0 + uint32_t(at) * sx_step;
      const int left = p.blocks - (kb0 + i) * 8;
      if (elect_lane()) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          mx_copy_scales<1>(sa_tmem + uint32_t(4 * h), sw_desc + uint32_t((h * kScaleTile) >> 4));
          mx_copy_scales<1>(sb_tmem + uint32_t(4 * h), sx_desc + uint32_t((h * kScaleTile) >> 4));
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (2 * j < left)
            mx_umma<1>(tmem_base, w_desc + uint32_t(2 * j), x_desc + uint32_t(2 * j), (j & 1) ? idesc2 : idesc0,
                       sa_tmem + uint32_t(4 * (j >> 1)), sb_tmem + uint32_t(4 * (j >> 1)), (i | j) != 0 ? 1u : 0u);
        }
        umma_commit(&empty_bar[stage]);
        if (i + 1 == kb_count) umma_commit(acc_full);
      }
      __syncwarp();
      if (++stage == p.stages) { stage = 0; phase ^= 1u; }
    }
  } else if constexpr (SRC != SRC_PACKED) {
    // ------------------------------------------------------------------ tokens -> shared memory
    // A warp takes 512 elements (a piece, two k-blocks) of a token at a time, sixteen a lane, two lanes a block.  The first
    // piece of all tokens comes first, so that its MMAs can start.  (10 / 14 / 18 warps, us: 1 row [11008, 4096] 7.8 / 7.9 /
    // 8.7, 16 rows [4096, 11008] 11.8 / 10.6 / 12.1, 32 rows [4096, 4096] 10.2 / 9.4 / 10.3.)
    const X* x = static_cast<const X*>(p.X);
    const int pieces = (kb_count + 1) / 2;
    const int piece_step = kSkQuantWarps / p.M, m_step = kSkQuantWarps - piece_step * p.M;
    int piece_next = (warp - 2) / p.M, m_next = (warp - 2) - piece_next * p.M;
    while (piece_next < pieces) {
      const int piece = piece_next, m = m_next, e = piece * 512 + lane * 16;
      piece_next += piece_step;
      m_next += m_step;
      if (m_next >= p.M) {
        m_next -= p.M;
        ++piece_next;
      }
      Sixteen<X> raw;
      const int64_t k = int64_t(kb0) * 256 + e;
      load16(x + int64_t(m) * p.K + k, p.K - k, raw, p.x_vec != 0);
      uint32_t top = top_of<X, Sixteen<X>::WORDS>(raw.w);
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      const uint32_t byte = mx_scale_byte(top);
      const uint2 codes = encode16(raw, byte);
      uint32_t four = byte << (4 * (lane & 6));
      four |= __shfl_xor_sync(0xffffffffu, four, 2);
      four |= __shfl_xor_sync(0xffffffffu, four, 4);
      const int kb = e >> 8;  // k-block within this CTA's range
      if (kb < kb_count) {
        // 128-byte swizzle: 16-byte chunk c of row m lies at chunk c ^ (m % 8)
        const int in_row = (e & 255) >> 1, chunk = (in_row >> 4) ^ (m & 7);
        *reinterpret_cast<uint2*>(xq + kb * token_bytes + m * 128 + (chunk << 4) + (in_row & 15)) = codes;
        if ((lane & 7) == 0)
          *reinterpret_cast<uint32_t*>(xs + kb * 2 * kScaleTile + ((e >> 7) & 1) * kScaleTile + (m & 31) * 16 + (m >> 5) * 4) = four;
      }
      fence_proxy_async_smem();  // the MMAs and scale copies read what was written here
      __syncwarp();
      if (lane == 0) mbar_arrive(&x_ready[piece]);
    }
  }
  __syncwarp();

  // Tail: an accumulator lane is a feature, a column a token.  The warps that share a quarter of the lanes take sixteen
  // tokens each in turn.
  const int quarter = warp & 3, feature = quarter * 32 + lane;
  const int own = 128 / S;  // features a CTA of the cluster finishes
  const bool acc_ready = warp_wait(acc_full, 0, abort_flag, p.wait_budget_ns);
  tc_fence_after_sync();
  if (acc_ready) {
    const uint32_t dst_cta = S > 1 ? map_to_cta(smem_u32(exch), uint32_t(feature / own)) : 0u;
    for (int m0 = (warp >> 2) * 16; m0 < p.M; m0 += sk_threads(SRC) / 8) {
      uint32_t v[16];
      tmem_ld_32x16(tmem_base + (uint32_t(quarter * 32) << 16) + uint32_t(m0), v);
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        if (m0 + i < p.M) {
          if (S > 1) st_cluster_u32(dst_cta + uint32_t(((int(rank) * tokens + m0 + i) * own + feature % own) * 4), v[i]);
          else if (n0 + feature < p.N) sk_store<EPI>(p, m0 + i, n0 + feature, __uint_as_float(v[i]));
        }
      }
    }
  }
  __syncwarp();
  if (S > 1) {
    cluster_sync_all();  // every range's sums have arrived, and nobody writes into another CTA after this
    if (*abort_flag == 0u) {
      const int first = n0 + int(rank) * own;
      for (int i = threadIdx.x; i < own * p.M; i += sk_threads(SRC)) {
        const int m = i / own, f = i - m * own;
        if (first + f < p.N) {
          float y = exch[m * own + f];
          for (int r = 1; r < S; ++r) y += exch[(r * tokens + m) * own + f];
          sk_store<EPI>(p, m, first + f, y);
        }
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (*abort_flag) {
    if (threadIdx.x == 0) atomicOr(&g_mx_status, 2u);
    // Give copies and MMAs still in flight time to land before shared and tensor memory go away.
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 2000000ull) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, uint32_t(p.tmem_cols));
  }
}

// ------------------------------------------------------------------------------ few tiles, long K
//
// A product with too few 128 x 128 tiles to occupy the GPU runs at the pace of one CTA per tile (a k-block, 34 KB, takes
// an SM about 0.4 us to pull in).  Here a tile belongs to a cluster of S CTAs, one range of K each.  The partial sums
// meet through distributed shared memory: the tile's columns are dealt out, 128 / S to a CTA; every epilogue warp sends
// its 32 rows to the owners, 16 bytes (four columns) a lane, into the slot of its range; after a cluster barrier every
// CTA adds the slots of its columns in K order and finishes them.
// Slots: [range][four columns][row][4 floats], so that consecutive lanes (rows) are neighbours on both sides.

struct MxSplit {
  static constexpr int STAGE_BYTES = MxTile<1, 128>::STAGE_BYTES;
  static constexpr int EXCHANGE_BYTES = 128 * 128 * 4;
  static constexpr int STAGES = (kSmemBudget - 2048 - EXCHANGE_BYTES) / STAGE_BYTES;
  static constexpr int SMEM_BYTES = kSmemBudget;
  static constexpr int TMEM_COLS = 256;  // 128 of sums, 16 of scales for each stage
  static_assert(128 + 16 * STAGES <= TMEM_COLS, "tensor memory");
};

template <int EPI>
__global__ void __launch_bounds__(kThreads, 1)
gemm_mx_split_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                     const __grid_constant__ CUtensorMap tmap_sa, const __grid_constant__ CUtensorMap tmap_sb, const MxArgs p) {
  using T = MxTile<1, 128>;
  constexpr int STAGES = MxSplit::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* exch = smem + STAGES * T::STAGE_BYTES;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(exch + MxSplit::EXCHANGE_BYTES);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* acc_full = empty_bar + STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_full + 1);
  volatile uint32_t* abort_flag = tmem_slot + 1;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int S = p.splits;
  const uint32_t rank = cluster_cta_rank();
  const int tile = int(blockIdx.x) / S;
  const int mb = tile % p.tiles_m, nb = tile / p.tiles_m;
  const int num_kb = (p.blocks + 7) / 8;
  const int kb0 = int(rank) * p.kb_per_split;
  const int kb_count = min(p.kb_per_split, num_kb - kb0);  // never empty

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    mbar_init(acc_full, 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmap_a);
    tma_prefetch_desc(&tmap_b);
    tma_prefetch_desc(&tmap_sa);
    tma_prefetch_desc(&tmap_sb);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, MxSplit::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncwarp();
  cluster_sync_all();  // every CTA of the cluster runs from here on
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;

  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  if (warp == 0) {
    // ------------------------------------------------------------------ loads
    int stage = 0;
    uint32_t phase = 0;
    for (int i = 0; i < kb_count; ++i) {
      if (!warp_wait(&empty_bar[stage], phase ^ 1u, abort_flag, p.wait_budget_ns)) break;
      const int kb = kb0 + i;
      const bool lost = kb == p.lose_kb && blockIdx.x == 0;
      if (!lost && elect_lane()) {
        uint8_t* sa = smem + stage * T::STAGE_BYTES;
        uint8_t* sb = sa + T::A_BYTES;
        uint8_t* ssa = sb + T::B_BYTES;
        uint8_t* ssb = ssa + T::SA_BYTES;
        mbar_arrive_expect_tx(&full_bar[stage], T::STAGE_BYTES);
        tma_load_2d(sa, &tmap_a, &full_bar[stage], kb * 128, mb * 128);
        tma_load_2d(sb, &tmap_b, &full_bar[stage], kb * 128, nb * 128);
        mx_load_3d<1>(ssa, &tmap_sa, smem_u32(&full_bar[stage]), 0, kb * 2, mb);
        mx_load_3d<1>(ssb, &tmap_sb, smem_u32(&full_bar[stage]), 0, kb * 2, nb);
      }
      __syncwarp();
      if (++stage == STAGES) { stage = 0; phase ^= 1u; }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ scale copies and MMAs
    constexpr uint32_t idesc0 = mx_instr_desc(128, 128, 0), idesc2 = mx_instr_desc(128, 128, 2);
    const uint32_t ring = smem_u32(smem);
    const uint32_t a_desc0 = desc_word(ring), b_desc0 = desc_word(ring + T::A_BYTES);
    const uint32_t s_desc0 = desc_word(ring + T::A_BYTES + T::B_BYTES);
    constexpr uint32_t kStageStep = T::STAGE_BYTES >> 4;
    int stage = 0;
    uint32_t phase = 0;
    for (int i = 0; i < kb_count; ++i) {
      if (!warp_wait(&full_bar[stage], phase, abort_flag, p.wait_budget_ns)) break;
      tc_fence_after_sync();
      // the scale buffers are the stages' own: one is rewritten only after its stage's MMAs
      const uint32_t sa_tmem = tmem_base + uint32_t(128 + stage * 16), sb_tmem = sa_tmem + 8;
      const uint32_t a_desc = a_desc0 + uint32_t(stage) * kStageStep, b_desc = b_desc0 + uint32_t(stage) * kStageStep;
      const uint32_t s_desc = s_desc0 + uint32_t(stage) * kStageStep;
      const int left = p.blocks - (kb0 + i) * 8;
      if (elect_lane()) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          mx_copy_scales<1>(sa_tmem + uint32_t(4 * h), s_desc + uint32_t((h * kScaleTile) >> 4));
          mx_copy_scales<1>(sb_tmem + uint32_t(4 * h), s_desc + uint32_t((T::SA_BYTES + h * kScaleTile) >> 4));
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (2 * j < left)
            mx_umma<1>(tmem_base, a_desc + uint32_t(2 * j), b_desc + uint32_t(2 * j), (j & 1) ? idesc2 : idesc0,
                       sa_tmem + uint32_t(4 * (j >> 1)), sb_tmem + uint32_t(4 * (j >> 1)), (i | j) != 0 ? 1u : 0u);
        }
        umma_commit(&empty_bar[stage]);
        if (i + 1 == kb_count) umma_commit(acc_full);
      }
      __syncwarp();
      if (++stage == STAGES) { stage = 0; phase ^= 1u; }
    }
  }
  __syncwarp();

  const int own = 128 / S, own_units = own / 4;  // columns a CTA finishes, and those in fours
  if (warp >= 2) {
    const int group = (warp - 2) >> 2, quarter = warp & 3;
    const bool ready = warp_wait(acc_full, 0, abort_flag, p.wait_budget_ns);
    tc_fence_after_sync();
    if (ready) {
      const uint32_t taddr = tmem_base + (uint32_t(quarter * 32) << 16) + uint32_t(group * 64);
      uint32_t v[2][32];
      tmem_ld_32x32(taddr, v[0]);
      tmem_ld_32x32(taddr + 32, v[1]);
      tmem_ld_wait();
      const uint32_t slot = smem_u32(exch) + uint32_t((int(rank) * own_units * 128 + quarter * 32 + lane) * 16);
#pragma unroll
      for (int u = 0; u < 16; ++u) {
        const int c = group * 16 + u, owner = c / own_units;  // the c-th four columns of the tile
        st_cluster_v4(map_to_cta(slot, uint32_t(owner)) + uint32_t((c - owner * own_units) * 128 * 16), v[u >> 3][4 * (u & 7)],
                      v[u >> 3][4 * (u & 7) + 1], v[u >> 3][4 * (u & 7) + 2], v[u >> 3][4 * (u & 7) + 3]);
      }
    }
  }
  __syncwarp();
  cluster_sync_all();  // every range's sums have arrived, and nobody writes into another CTA after this

  if (*abort_flag == 0u) {
    // eight columns of a row at a time
    const int units = own / 8 * 128;
    for (int i = threadIdx.x; i < units; i += kThreads) {
      const int row = i & 127, g = i >> 7, m = mb * 128 + row, n = nb * 128 + int(rank) * own + g * 8;
      if (m >= p.M || n >= p.N) continue;
      float y[8] = {};
      for (int r = 0; r < S; ++r) {
        const float4* slot = reinterpret_cast<const float4*>(exch) + (r * own_units + 2 * g) * 128 + row;
        const float4 lo = slot[0], hi = slot[128];
        y[0] += lo.x; y[1] += lo.y; y[2] += lo.z; y[3] += lo.w;
        y[4] += hi.x; y[5] += hi.y; y[6] += hi.z; y[7] += hi.w;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (p.bias != nullptr) y[e] += p.bias[min(n + e, p.N - 1)];
        if (p.relu) y[e] = fmaxf(0.0f, y[e]);
      }
      using Out = typename std::conditional<EPI == EPI_F32, float, typename std::conditional<EPI == EPI_F16, __half, __nv_bfloat16>::type>::type;
      alignas(16) Out out[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if constexpr (EPI == EPI_F32) out[e] = y[e];
        else if constexpr (EPI == EPI_F16) out[e] = __float2half_rn(y[e]);
        else out[e] = __float2bfloat16_rn(y[e]);
      }
      Out* dst = static_cast<Out*>(p.C) + int64_t(m) * p.ldc + n;
      if (p.tma_store && n + 8 <= p.N) {  // 16-byte aligned
#pragma unroll
        for (int k = 0; k < int(sizeof(out) / 16); ++k) reinterpret_cast<uint4*>(dst)[k] = reinterpret_cast<const uint4*>(out)[k];
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (n + e < p.N) dst[e] = out[e];
      }
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (*abort_flag) {
    if (threadIdx.x == 0) atomicOr(&g_mx_status, 4u);
    // Give copies and MMAs still in flight time to land before shared and tensor memory go away.
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 2000000ull) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, MxSplit::TMEM_COLS);
  }
}

// ------------------------------------------------------------------------------ host side

// Packed elements as bytes: 128-byte swizzle, zeros outside the matrix.
int map_elements(CUtensorMap* map, const void* q, int64_t rows, int64_t row_bytes, int box_rows) {
  return encode_operand_map(map, KIND_I8, q, rows, row_bytes, row_bytes, 128, box_rows, false);
}
// Scale tiles: [bands][tiles along K][128 words]; a box is two tiles along K of `box_bands` bands.
int map_scales(CUtensorMap* map, const void* s, int64_t rows, int64_t tiles, int box_bands) {
  const uint64_t dims[3] = {kScaleTile / 4, uint64_t(tiles), uint64_t((rows + 127) / 128)};
  const uint64_t strides[2] = {kScaleTile, uint64_t(tiles) * kScaleTile};
  const uint32_t box[3] = {kScaleTile / 4, 2, uint32_t(box_bands)};
  return encode_tiled_map(map, CU_TENSOR_MAP_DATA_TYPE_INT32, 3, s, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
}
int map_output(CUtensorMap* map, int epi, const void* c, int64_t rows, int64_t cols, int64_t ldc) {
  const int elem = epi == EPI_F32 ? 4 : 2;
  const uint64_t dims[2] = {uint64_t(cols), uint64_t(rows)};
  const uint64_t strides[1] = {uint64_t(ldc) * elem};
  const uint32_t box[2] = {uint32_t(128 / elem), 32};
  return encode_tiled_map(map, epi == EPI_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, c, dims,
                          strides, box, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE);
}

template <int CG, int BN, int EPI>
int launch_tile(const MxGemm& g, int sms, cudaStream_t stream) {
  using T = MxTile<CG, BN>;
  auto kernel = gemm_mx_kernel<CG, BN, EPI>;
  static thread_local int last_dev = -1;  // the shared-memory attribute is per device
  int dev = 0;
  B200_CUDA_TRY(cudaGetDevice(&dev));
  if (dev != last_dev) {
    B200_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, T::SMEM_BYTES));
    last_dev = dev;
  }
  MxArgs p;
  memset(&p, 0, sizeof(p));
  p.C = g.C;
  p.ldc = g.ldc;
  p.M = int(g.M);
  p.N = int(g.N);
  p.blocks = int((g.K + 31) / 32);
  p.tiles_m = int((g.M + T::TILE_M - 1) / T::TILE_M);
  p.tiles_n = int((g.N + BN - 1) / BN);
  p.group_m = 4096 / T::TILE_M;
  p.bias = g.tail.bias;
  p.relu = g.tail.flags & B200_LINEAR_RELU;
  wait_test_settings(&p.lose_kb, &p.wait_budget_ns);
  const int elem = EPI == EPI_F32 ? 4 : 2;
  p.tma_store = (g.ldc * elem) % 16 == 0 && reinterpret_cast<uintptr_t>(g.C) % 16 == 0;

  const int64_t row_bytes = mx_row_bytes(g.K), tiles_k = (g.K + 127) / 128;
  CUtensorMap ma, mb, msa, msb, mc;
  memset(&mc, 0, sizeof(mc));
  int rc = map_elements(&ma, g.A, g.M, row_bytes, 128);
  if (!rc) rc = map_elements(&mb, g.B, g.N, row_bytes, BN / CG);
  if (!rc) rc = map_scales(&msa, g.a_scale, g.M, tiles_k, 1);
  if (!rc) rc = map_scales(&msb, g.b_scale, g.N, tiles_k, T::BANDS);
  if (!rc && p.tma_store) rc = map_output(&mc, EPI, g.C, g.M, g.N, g.ldc);
  if (rc) return rc;

  const int64_t tiles = int64_t(p.tiles_m) * p.tiles_n;
  if (tiles > (int64_t(1) << 30)) return fail(B200_ERR_TOO_LARGE, "MXFP4 product: too many tiles");
  cudaLaunchConfig_t cfg = {};
  const int64_t slots = sms / CG;
  cfg.gridDim = dim3(unsigned((tiles < slots ? tiles : slots) * CG));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = T::SMEM_BYTES;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int nattr = 0;
  if (dependent_launch_enabled()) {
    attr[nattr].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[nattr].val.programmaticStreamSerializationAllowed = 1;
    ++nattr;
  }
  if (CG == 2) {
    attr[nattr].id = cudaLaunchAttributeClusterDimension;
    attr[nattr].val.clusterDim.x = 2;
    attr[nattr].val.clusterDim.y = 1;
    attr[nattr].val.clusterDim.z = 1;
    ++nattr;
  }
  cfg.attrs = attr;
  cfg.numAttrs = unsigned(nattr);
  B200_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, ma, mb, msa, msb, mc, p));
  return B200_OK;
}

struct SkinnyPlan {
  int splits = 0, per = 0, stages = 0, smem = 0, tokens = 0, tmem_cols = 0;
};

// Several of these CTAs share an SM, and a CTA that finds no room in tensor memory waits in tcgen05.alloc without a
// limit while its cluster waits for it.  So a CTA's share of an SM's shared memory (1 KB of which the system takes)
// is never below its share of the 512 columns: CTAs that fit together in the one fit in the other, whatever
// launches they come from.
constexpr int kSmSharedBytes = 228 * 1024;
int skinny_tmem_cols(int tokens, int stages) {
  int cols = 32;
  while (cols < tokens + 16 * stages) cols *= 2;
  return cols;
}
int skinny_smem(bool packed, int tokens, int per, int splits, int stages) {
  const int stage = kWeightBytes + kWeightScales + (packed ? tokens * 128 + 2 * kScaleTile : 0);
  const int need = stages * stage + (packed ? 0 : per * (tokens * 128 + 2 * kScaleTile)) +
                   (splits > 1 ? 128 * tokens * 4 : 0) + 1024 + 512;
  const int share = skinny_tmem_cols(tokens, stages) * (kSmSharedBytes / 512) - 1024;
  return need > share ? need : share;
}

// Cluster size: the largest that asks for at most a quarter more CTAs than there are SMs.  Measured, 1 / 2 / 4 / 8 ranges, us:
// one row, [11008, 4096] (86 tiles) 9.3 / 8.0 / 12.1 / 17.3; 8 rows, [4096, 4096] (32 tiles) 9.3 / 7.3 / 6.3 / 7.2; 16 rows,
// [4096, 11008] packed 15.1 / 11.6 / 9.2 / 10.2.  The shares are uneven: 86 tiles in two ranges are 172 CTAs, so that 24 of 148
// SMs stream 16 k-blocks where the mean is 9.3; 32 tiles in four are 128 CTAs, and 20 SMs stream nothing.
SkinnyPlan plan_skinny(const MxGemm& g, bool packed, int sms) {
  SkinnyPlan best;
  const int num_kb = int((g.K + 255) / 256), tokens = int((g.M + 15) / 16) * 16;
  const int64_t tiles = (g.N + 127) / 128;
  for (int s = 1; s <= 8; s *= 2) {
    if (best.splits && tiles * s * 4 > int64_t(sms) * 5) break;
    const int per = (num_kb + s - 1) / s;
    if ((num_kb + per - 1) / per != s) continue;  // a range would be empty
    // a ring that leaves room for a second CTA on the SM, another cluster's or the next launch's (with all of the SM's
    // memory one row of the 86-tile layer takes 13.4 us instead of 8.0)
    int stages = per < kSkMaxStages ? per : kSkMaxStages;
    while (stages > 2 && skinny_smem(packed, tokens, per, s, stages) > kSmSharedBytes / 2 - 1024) --stages;
    const int smem = skinny_smem(packed, tokens, per, s, stages);
    if (smem > kSmemBudget || (!packed && (per + 1) / 2 > kSkMaxPieces)) continue;
    best.splits = s;
    best.per = per;
    best.stages = stages;
    best.smem = smem;
    best.tokens = tokens;
    best.tmem_cols = skinny_tmem_cols(tokens, stages);
  }
  return best;
}

template <int SRC, int EPI>
int launch_skinny(const MxGemm& g, const SkinnyPlan& plan, cudaStream_t stream, bool swapped = false) {
  auto kernel = gemm_mx_skinny_kernel<SRC, EPI>;
  static thread_local int last_dev = -1;
  int dev = 0;
  B200_CUDA_TRY(cudaGetDevice(&dev));
  if (dev != last_dev) {
    B200_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBudget));
    last_dev = dev;
  }
  MxSkinnyArgs p;
  memset(&p, 0, sizeof(p));
  p.C = g.C;
  p.X = g.X;
  p.ldc = g.ldc;
  p.M = int(g.M);
  p.N = int(g.N);
  p.K = int(g.K);
  p.blocks = int((g.K + 31) / 32);
  p.tokens = plan.tokens;
  p.splits = plan.splits;
  p.kb_per_split = plan.per;
  p.stages = plan.stages;
  p.scale_col = plan.tokens;
  p.tmem_cols = plan.tmem_cols;
  p.swapped = swapped;
  p.bias = g.tail.bias;
  p.relu = g.tail.flags & B200_LINEAR_RELU;
  wait_test_settings(&p.lose_kb, &p.wait_budget_ns);
  const int64_t row_bytes = mx_row_bytes(g.K), tiles_k = (g.K + 127) / 128;
  CUtensorMap mw, msw, mx, msx;
  int rc = map_elements(&mw, g.B, g.N, row_bytes, 128);
  if (!rc) rc = map_scales(&msw, g.b_scale, g.N, tiles_k, 1);
  if (rc) return rc;
  if (SRC == SRC_PACKED) {
    rc = map_elements(&mx, g.A, g.M, row_bytes, plan.tokens);
    if (!rc) rc = map_scales(&msx, g.a_scale, g.M, tiles_k, 1);
    if (rc) return rc;
  } else {
    const int64_t pitch = g.K * (SRC == SRC_F32 ? 4 : 2);
    p.x_vec = pitch % 16 == 0 && reinterpret_cast<uintptr_t>(g.X) % 16 == 0;
    memset(&mx, 0, sizeof(mx));
    memset(&msx, 0, sizeof(msx));
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned((g.N + 127) / 128 * plan.splits));
  cfg.blockDim = dim3(unsigned(sk_threads(SRC)));
  cfg.dynamicSmemBytes = size_t(plan.smem);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int nattr = 0;
  if (dependent_launch_enabled()) {
    attr[nattr].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[nattr].val.programmaticStreamSerializationAllowed = 1;
    ++nattr;
  }
  if (plan.splits > 1) {
    attr[nattr].id = cudaLaunchAttributeClusterDimension;
    attr[nattr].val.clusterDim.x = unsigned(plan.splits);
    attr[nattr].val.clusterDim.y = 1;
    attr[nattr].val.clusterDim.z = 1;
    ++nattr;
  }
  cfg.attrs = attr;
  cfg.numAttrs = unsigned(nattr);
  B200_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, mw, msw, mx, msx, p));
  return B200_OK;
}

int device_sms(int* sms) {
  int dev = 0;
  B200_CUDA_TRY(cudaGetDevice(&dev));
  B200_CUDA_TRY(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev));
  return B200_OK;
}

// Ranges of K for a product of `tiles` 128 x 128 tiles (1 = do not split).  1 / 2 / 4 / 8 ranges, us: K = 2048, 16 tiles 6.4 /
// 6.2 / 5.7 / 11.4; K = 4096, 14 tiles 9.5 / 7.7 / 6.6 / 7.0, 32 tiles 9.5 / 7.5 / 7.3 / 18.8, 36 tiles 9.4 / 7.4 / 12.8 / 19.3, 74
// tiles 9.8 / 8.6 / 21.0; K = 11008, 14 tiles 19.6 / 12.1 / 8.9 / 8.3, 16 tiles 19.5 / 11.7 / 8.4 / 14.3, 32 tiles 19.7 / 11.9 / 9.6 /
// 22.4, 74 tiles 19.9 / 13.1 / 27.6.  A cluster has to find its CTAs' SMs inside one group of SMs, so not every SM can be used
// by clusters of four (seven eighths of them) or eight (three quarters) at once; where a cluster has to wait the time doubles.
int split_ranges(int64_t tiles, int num_kb, int sms) {
  auto whole = [&](int s) { return ((num_kb + s - 1) / s) * (s - 1) < num_kb; };  // no range is empty
  if (num_kb >= 32 && tiles * 8 * 4 <= int64_t(sms) * 3 && whole(8)) return 8;
  if (num_kb >= 8 && tiles * 4 * 8 <= int64_t(sms) * 7 && whole(4)) return 4;
  if (num_kb >= 12 && tiles * 2 <= sms && whole(2)) return 2;
  return 1;
}

template <int EPI>
int launch_split(const MxGemm& g, int splits, cudaStream_t stream) {
  auto kernel = gemm_mx_split_kernel<EPI>;
  static thread_local int last_dev = -1;  // the shared-memory attribute is per device
  int dev = 0;
  B200_CUDA_TRY(cudaGetDevice(&dev));
  if (dev != last_dev) {
    B200_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MxSplit::SMEM_BYTES));
    last_dev = dev;
  }
  MxArgs p;
  memset(&p, 0, sizeof(p));
  p.C = g.C;
  p.ldc = g.ldc;
  p.M = int(g.M);
  p.N = int(g.N);
  p.blocks = int((g.K + 31) / 32);
  p.tiles_m = int((g.M + 127) / 128);
  p.tiles_n = int((g.N + 127) / 128);
  p.bias = g.tail.bias;
  p.relu = g.tail.flags & B200_LINEAR_RELU;
  p.splits = splits;
  p.kb_per_split = ((p.blocks + 7) / 8 + splits - 1) / splits;
  wait_test_settings(&p.lose_kb, &p.wait_budget_ns);
  const int elem = EPI == EPI_F32 ? 4 : 2;
  p.tma_store = (g.ldc * elem) % 16 == 0 && reinterpret_cast<uintptr_t>(g.C) % 16 == 0;
  const int64_t row_bytes = mx_row_bytes(g.K), tiles_k = (g.K + 127) / 128;
  CUtensorMap ma, mb, msa, msb;
  int rc = map_elements(&ma, g.A, g.M, row_bytes, 128);
  if (!rc) rc = map_elements(&mb, g.B, g.N, row_bytes, 128);
  if (!rc) rc = map_scales(&msa, g.a_scale, g.M, tiles_k, 1);
  if (!rc) rc = map_scales(&msb, g.b_scale, g.N, tiles_k, 1);
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(p.tiles_m * p.tiles_n * splits));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = MxSplit::SMEM_BYTES;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(splits);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = dependent_launch_enabled() ? 2 : 1;
  B200_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, ma, mb, msa, msb, p));
  return B200_OK;
}

template <int EPI>
int launch_epi(const MxGemm& g, cudaStream_t stream) {
  int sms = 0;
  int rc = device_sms(&sms);
  if (rc) return rc;
  if (g.M <= kSkRows) {
    const SkinnyPlan plan = plan_skinny(g, true, sms);
    if (plan.splits) return launch_skinny<SRC_PACKED, EPI>(g, plan, stream);
  }
  if (g.N <= kSkRows && g.M > g.N) {
    MxGemm t = g;
    std::swap(t.A, t.B);
    std::swap(t.a_scale, t.b_scale);
    std::swap(t.M, t.N);
    const SkinnyPlan plan = plan_skinny(t, true, sms);
    if (plan.splits) return launch_skinny<SRC_PACKED, EPI>(t, plan, stream, true);
  }
  const int64_t tiles = ((g.M + 127) / 128) * ((g.N + 127) / 128);
  const int splits = split_ranges(tiles, int((g.K + 255) / 256), sms);
  if (splits > 1) return launch_split<EPI>(g, splits, stream);
  // CTA pairs once they give every pair of SMs a tile.  A k-block takes an SM about as long in either kernel, so what counts is
  // the rounds of tiles.  Single CTAs / pairs, us, K = 4096 where nothing else is said: 2304 x 2304 22.6 / 16.5, 2048 x 4096 30.0 /
  // 17.2, 32768 x 128 17.1 / 16.3, 32768 x 64 16.4 / 15.8.  Where fewer pairs have a tile but single CTAs need two rounds, pairs
  // would be the faster ones too: 1024 x 4096 16.6 / 10.9 (K = 2048: 10.2 / 8.3, K = 11008: 37.1 / 19.2), 256 x 11008 16.4 / 11.5,
  // 2048 x 2048 with K = 2048 10.3 / 8.2.
  const int64_t pair_tiles = ((g.M + 255) / 256) * ((g.N + 255) / 256);
  if (g.M > 128 && pair_tiles >= sms / 2) return launch_tile<2, 256, EPI>(g, sms, stream);
  return launch_tile<1, 128, EPI>(g, sms, stream);
}

}  // namespace

int launch_mx_gemm(int out_dtype, const MxGemm& g, cudaStream_t stream) {
  switch (out_dtype) {
    case B200_F32: return launch_epi<EPI_F32>(g, stream);
    case B200_F16: return launch_epi<EPI_F16>(g, stream);
    default: return launch_epi<EPI_BF16>(g, stream);
  }
}

bool mx_layer_in_one_launch(int64_t rows, int64_t K, int64_t N) {
  return K <= kSkFusedK && N <= kSkFusedN && (rows <= kSkFusedRows || (rows <= kSkRows && rows * K <= kSkFusedElements));
}

int launch_mx_layer(int dtype, const MxGemm& g, cudaStream_t stream) {
  int sms = 0;
  int rc = device_sms(&sms);
  if (rc) return rc;
  const SkinnyPlan plan = plan_skinny(g, false, sms);
  if (!plan.splits) return fail(B200_ERR_TOO_LARGE, "linear_mxfp4: in_features %lld", (long long)g.K);
  switch (dtype) {
    case B200_F32: return launch_skinny<SRC_F32, EPI_F32>(g, plan, stream);
    case B200_F16: return launch_skinny<SRC_F16, EPI_F16>(g, plan, stream);
    default: return launch_skinny<SRC_BF16, EPI_BF16>(g, plan, stream);
  }
}

int read_and_clear_mx_status(uint32_t* out) {
  uint32_t zero = 0;
  B200_CUDA_TRY(cudaMemcpyFromSymbol(out, g_mx_status, sizeof(uint32_t)));
  if (*out) B200_CUDA_TRY(cudaMemcpyToSymbol(g_mx_status, &zero, sizeof(uint32_t)));
  return B200_OK;
}

}  // namespace b200
