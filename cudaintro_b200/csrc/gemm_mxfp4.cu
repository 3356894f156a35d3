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
// Every wait is bounded; a wait that runs out raises the CTA's abort flag, all roles drain, tensor memory is freed
// and a status word tells the host that the result is invalid.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstring>

#include "internal.h"
#include "mxfp4.cuh"
#include "ptx_sm100.cuh"

namespace b200 {
namespace {

__device__ uint32_t g_mx_status = 0;  // bit 0: a bounded wait ran out somewhere

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

template <int CG>
__device__ __forceinline__ void mx_umma(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t sa_tmem,
                                        uint32_t sb_tmem, uint32_t accumulate) {
  if constexpr (CG == 2)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        :
        : "r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sa_tmem), "r"(sb_tmem), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        :
        : "r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sa_tmem), "r"(sb_tmem), "r"(accumulate)
        : "memory");
}

// One scale tile, shared memory -> four columns of tensor memory (of both CTAs of a pair, each from its own).
template <int CG>
__device__ __forceinline__ void mx_copy_scales(uint32_t tmem, uint64_t desc) {
  if constexpr (CG == 2)
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
  else
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
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
  static constexpr int STAGING_BYTES = kEpiWarps * 32 * 128;
  static constexpr int STAGES_FIT = (kSmemBudget - 2048 - STAGING_BYTES) / STAGE_BYTES;
  static constexpr int STAGES = STAGES_FIT > 6 ? 6 : STAGES_FIT;
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + STAGING_BYTES + 1024 + 256;
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
  int tma_store;
  const float* bias;
  int relu;
  unsigned long long wait_budget_ns;
  int lose_kb;  // test of the give-up path: k-block of CTA 0's first tile that is never loaded; -1 = none
};

// Groups of group_m tiles of rows; inside a group m runs fastest (a wave of tiles is then a near-square patch).
__device__ __forceinline__ void mx_tile_coords(int t, const MxArgs& p, int& mb, int& nb) {
  const int per_group = p.group_m * p.tiles_n;
  const int g = t / per_group, first_m = g * p.group_m, gm = min(p.tiles_m - first_m, p.group_m), r = t - g * per_group;
  mb = first_m + r % gm;
  nb = r / gm;
}

// 32 accumulators of one row -> 32 (fp32) or 16 output words, with the tail.
template <int EPI>
__device__ __forceinline__ void mx_finish(const MxArgs& p, int n0, uint32_t (&v)[32], uint32_t* w) {
  if (p.bias != nullptr) {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      v[i] = __float_as_uint(__uint_as_float(v[i]) + p.bias[min(n0 + i, p.N - 1)]);
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
      const uint64_t a_desc0 = make_smem_desc_sw128(ring, 16, 1024);
      const uint64_t b_desc0 = make_smem_desc_sw128(ring + T::A_BYTES, 16, 1024);
      // scale tiles: 8 x 16-byte core matrices, 128 bytes apart, no swizzle
      const uint64_t s_desc0 = make_smem_desc(ring + T::A_BYTES + T::B_BYTES, 16, 128, 0);
      constexpr uint64_t kStageStep = uint64_t(T::STAGE_BYTES >> 4);
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
          const uint64_t s_desc = s_desc0 + uint64_t(stage) * kStageStep;
          const uint64_t a_desc = a_desc0 + uint64_t(stage) * kStageStep;
          const uint64_t b_desc = b_desc0 + uint64_t(stage) * kStageStep;
          const int left = p.blocks - kb * 8;  // blocks of 32 this stage really holds
          if (elect_lane()) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              mx_copy_scales<CG>(sa_tmem + uint32_t(4 * h), s_desc + uint64_t((h * kScaleTile) >> 4));
#pragma unroll
              for (int b = 0; b < T::BANDS; ++b)
                mx_copy_scales<CG>(sb_tmem + uint32_t(h * 4 * T::BANDS + 4 * b),
                                   s_desc + uint64_t((T::SA_BYTES + (2 * b + h) * kScaleTile) >> 4));
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if (2 * j < left)
                mx_umma<CG>(d_tmem, a_desc + uint64_t(2 * j), b_desc + uint64_t(2 * j), (j & 1) ? idesc2 : idesc0,
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
    constexpr int BOX_COLS = 128 / OUT_BYTES;
    const int group = (warp - 2) >> 2;  // two warps per quarter share a tile's units of 64 columns
    const int quarter = warp & 3;       // tensor-memory lanes this warp may read
    uint8_t* buf = staging + (warp - 2) * (32 * 128);
    int it = 0;
    for (int t = first_tile; t < num_tiles; t += tile_step, ++it) {
      int mb, nb;
      mx_tile_coords(t, p, mb, nb);
      const int ab = it & 1;
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
      const uint32_t taddr = tmem_base + (uint32_t(quarter * 32) << 16) + uint32_t(ab * T::ACC_STEP);
#pragma unroll 1
      for (int i = 0; i < T::UNITS / 2; ++i) {
        // Group 0 begins with the unit that the other accumulator overlaps (the last one of accumulator 0, the
        // first one of accumulator 1); group 1 has the units between.
        const int unit = T::UNITS == 2 ? group : (group == 0 ? ((i ^ ab) ? 0 : 3) : 1 + i);
        const int n0 = nb * BN + unit * 64;
        uint32_t v[2][32];
        tmem_ld_32x32(taddr + uint32_t(unit * 64), v[0]);
        tmem_ld_32x32(taddr + uint32_t(unit * 64 + 32), v[1]);
        tmem_ld_wait();
        if (i == 0) {
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) {
            if constexpr (CG == 2) mbar_arrive_cluster(map_to_cta(smem_u32(acc_go), 0)); else mbar_arrive(acc_go);
          }
        }
        if (n0 >= p.N) continue;
        if (p.tma_store) {
#pragma unroll
          for (int box = 0; box < 64 / BOX_COLS; ++box) {
            uint32_t w[32];
            mx_finish<EPI>(p, n0 + box * BOX_COLS, v[box], w);
            if constexpr (EPI != EPI_F32) mx_finish<EPI>(p, n0 + 32, v[1], w + 16);
            if (lane == 0) tma_store_wait_read<0>();  // this warp's previous store has read the buffer
            __syncwarp();
#pragma unroll
            for (int u = 0; u < 8; ++u)
              *reinterpret_cast<uint4*>(buf + lane * 128 + ((u ^ (lane & 7)) << 4)) =
                  make_uint4(w[4 * u], w[4 * u + 1], w[4 * u + 2], w[4 * u + 3]);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0 && row0 < p.M && n0 + box * BOX_COLS < p.N) {
              tma_store_2d(&tmap_c, buf, n0 + box * BOX_COLS, row0);
              tma_store_commit();
            }
          }
        } else if (row0 + lane < p.M) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t w[32];
            mx_finish<EPI>(p, n0 + 32 * h, v[h], w);
            char* crow = static_cast<char*>(p.C) + (int64_t(row0 + lane) * p.ldc + n0 + 32 * h) * OUT_BYTES;
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (n0 + 32 * h + e < p.N) {
                if constexpr (EPI == EPI_F32) reinterpret_cast<uint32_t*>(crow)[e] = w[e];
                else reinterpret_cast<uint16_t*>(crow)[e] = uint16_t(w[e >> 1] >> ((e & 1) * 16));
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

template <int EPI>
int launch_epi(const MxGemm& g, cudaStream_t stream) {
  int dev = 0, sms = 0;
  B200_CUDA_TRY(cudaGetDevice(&dev));
  B200_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  // CTA pairs once they give every pair of SMs a tile.
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

int read_and_clear_mx_status(uint32_t* out) {
  uint32_t zero = 0;
  B200_CUDA_TRY(cudaMemcpyFromSymbol(out, g_mx_status, sizeof(uint32_t)));
  if (*out) B200_CUDA_TRY(cudaMemcpyToSymbol(g_mx_status, &zero, sizeof(uint32_t)));
  return B200_OK;
}

}  // namespace b200
