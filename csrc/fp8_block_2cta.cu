// Products in 8-bit floating point with fp32 scales per block of 128 on CTA pairs (same contract as fp8_block_gemm.cu): tiles of
// 256 rows x 256 columns, tcgen05.mma.cta_group::2 kind::f8f6f4.
//
// Each CTA loads its own 128 rows of `a` and half of the weight rows, 32 KB per block of K where one CTA on its own would load
// 48 KB for 128 x 256: an SM takes in about 64 bytes per clock from L2, and a block is 512 clocks of the tensor core.
// Every block of K has an accumulator of its own, 256 columns, two of them; eight warps (two warpgroups, a quarter of the rows and
// half of the columns each) add scale * accumulator to 128 fp32 sums per thread.  Those sums and the 64 registers in flight need
// more than the 168 registers that 384 threads can have, so the load and MMA warpgroup hands its registers over (setmaxnreg:
// 40 + 232 + 232 = 3 x 168); with 168, the sums spilled, which doubled the traffic to L2.
//
// Barriers as in gemm_2cta_sm100.cu, with an accumulator per block instead of per tile.
#include <cuda.h>
#include <cuda_runtime.h>

#include "expert_ops.h"
#include "fp8_block.cuh"
#include "gemm_sm100.cuh"
#include "gemm_sm100.h"
#include "grouped_common.cuh"
#include "umma_2cta.cuh"

namespace msccl {
namespace sm100 {

namespace {

constexpr int kFPThreads = 384;                  // 0 producer, 1 MMA, 2 and 3 idle, 4..11 scaling and epilogue
constexpr int kFPEpilogueWarps = 8;
constexpr int kFPTile = 256;
constexpr int kFPOperand = 128 * kFBlock;        // 16 KB
constexpr int kFPStageBytes = 2 * kFPOperand;
constexpr int kFPStages = 6;
constexpr int kFPTmemCols = 2 * kFPTile;
constexpr size_t kFPSmem = 1024 + static_cast<size_t>(kFPStages) * kFPStageBytes + 256;
constexpr int kLaunchRegs = 168, kLoadRegs = 40, kSumRegs = 232;
static_assert(kLoadRegs + 2 * kSumRegs <= 3 * kLaunchRegs, "the warpgroups share the registers that the CTA was launched with");

__device__ __forceinline__ void umma_f8_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(static_cast<uint32_t>(accumulate))
      : "memory");
}

__global__ void __launch_bounds__(kFPThreads, 1)
fp8_block_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w, const FArgs g) {
  constexpr int S = kFPStages, COLS = kFPTile / 2;
  extern __shared__ uint8_t smem_raw[];
  __shared__ GroupTable table;
  __shared__ int s_skip;
  uint8_t* stage_base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(stage_base + static_cast<size_t>(S) * kFPStageBytes);
  uint64_t *full_bar = bars, *empty_bar = bars + S, *acc_full = bars + 2 * S, *acc_empty = bars + 2 * S + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * S + 4);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int n_tiles = (g.n + kFPTile - 1) / kFPTile;
  const int k_blocks = (g.k + kFBlock - 1) / kFBlock;
  const int first = static_cast<int>(cluster_id_x()), step = static_cast<int>(num_clusters_x());

  if (threadIdx.x == 0) {
    // an earlier launch gave up: skip the work; the leader's reading decides for the pair
    s_skip = g.error_words != nullptr && *reinterpret_cast<volatile int*>(g.error_words) != 0 ? 1 : 0;
    for (int s = 0; s < S; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], 2 * kFPEpilogueWarps);
    }
    *abort_flag = 0;
    mbar_fence_init();
    prefetch_tensormap(&map_a);
    prefetch_tensormap(&map_w);
  }
  if (warp == 1) tmem_alloc_pair(tmem_slot, kFPTmemCols);
  if (warp == 2) build_table(table, g, [&](int rows) { return (rows + kFPTile - 1) / kFPTile * n_tiles; });
  tc_fence_before_sync();
  cluster_sync_all();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  const bool skip = ld_shared_cluster_u32(map_to_cta(smem_u32(&s_skip), 0)) != 0;
  const int num_tiles = skip ? 0 : table.tile_start[g.groups];

  auto locate = [&](int tile, int& e, int& row, int& column) {
    while (tile >= table.tile_start[e + 1]) ++e;
    const int rows = table.row_start[e + 1] - table.row_start[e];
    int tm, tn;
    tile_coords(tile - table.tile_start[e], (rows + kFPTile - 1) / kFPTile, n_tiles, kFGroupTileRows / kFPTile, tm, tn);
    row = table.row_start[e] + tm * kFPTile + static_cast<int>(rank) * BM;
    column = tn * kFPTile;
  };

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kLoadRegs));
    if (warp == 0 && elect_one()) {
      int stage = 0, e = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = first; tile < num_tiles && ok; tile += step) {
        int row, column;
        locate(tile, e, row, column);
        column += static_cast<int>(rank) * (kFPTile / 2);
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1, abort_flag)) {
            gemm_fail(g.error_words, abort_flag, GEMM_TIMEOUT_EMPTY, 0, stage);
            ok = false;
            break;
          }
          uint8_t* a_dst = stage_base + static_cast<size_t>(stage) * kFPStageBytes;
          if (leader) mbar_expect_tx(&full_bar[stage], 2 * kFPStageBytes);
          const uint32_t bar = map_to_cta(smem_u32(&full_bar[stage]), 0);
          tma_pair_2d(a_dst, &map_a, bar, kb * kFBlock, row);
          tma_pair_3d(a_dst + kFPOperand, &map_w, bar, kb * kFBlock, column, e);
          if (++stage == S) { stage = 0; phase ^= 1; }
        }
      }
      if (!ok) drain_wait();
    } else if (warp == 1 && leader && elect_one()) {
      constexpr uint32_t idesc = (1u << 4) | (static_cast<uint32_t>(kFPTile >> 3) << 17) | (static_cast<uint32_t>(kFPTile >> 4) << 24);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int tile = first; tile < num_tiles && ok; tile += step) {
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!mbar_wait(&acc_empty[acc], acc_phase ^ 1, abort_flag)) {
            gemm_fail(g.error_words, abort_flag, GEMM_TIMEOUT_ACC, 1, acc);
            ok = false;
            break;
          }
          if (!mbar_wait(&full_bar[stage], phase, abort_flag)) {
            gemm_fail(g.error_words, abort_flag, GEMM_TIMEOUT_FULL, 1, stage);
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t a_addr = smem_u32(stage_base + static_cast<size_t>(stage) * kFPStageBytes);
          const uint64_t adesc = smem_desc_sw128(a_addr), bdesc = smem_desc_sw128(a_addr + kFPOperand);
          const uint32_t tmem_d = tmem_base + static_cast<uint32_t>(acc * kFPTile);
#pragma unroll
          for (int k = 0; k < kFBlock / 32; ++k)
            umma_f8_pair(tmem_d, adesc + static_cast<uint64_t>(k * 2), bdesc + static_cast<uint64_t>(k * 2), idesc, k != 0);
          tc_commit_pair(&empty_bar[stage], 3);
          tc_commit_pair(&acc_full[acc], 3);
          if (++stage == S) { stage = 0; phase ^= 1; }
          if (++acc == 2) { acc = 0; acc_phase ^= 1; }
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSumRegs));
    const int quarter = warp % 4, half = (warp - 4) / 4;
    const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(half * COLS);
    int acc = 0, e = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    for (int tile = first; tile < num_tiles && ok; tile += step) {
      int row, column;
      locate(tile, e, row, column);
      const int left = table.row_start[e + 1] - row - quarter * 32;       // rows of this warp that are the group's
      row += quarter * 32 + lane;
      column += half * COLS;
      float2 sum[COLS / 2];
#pragma unroll
      for (int i = 0; i < COLS / 2; ++i) sum[i] = make_float2(0.0f, 0.0f);
      ScaleStream<4> scales(g.sa + min(row, g.rows - 1) * g.sa_row, g.sa_block, weight_scales(g, e, column, k_blocks), k_blocks, left > 0);
      for (int kb0 = 0; kb0 < k_blocks && ok; kb0 += 4) {
       scales.advance();
#pragma unroll
       for (int j = 0; j < 4; ++j) {
        if (kb0 + j >= k_blocks) break;
        const float scale = scales.now[j];
        ok = mbar_wait(&acc_full[acc], acc_phase, abort_flag);
        ok = __all_sync(kFullMask, ok);
        if (!ok) {
          if (lane == 0) gemm_fail(g.error_words, abort_flag, GEMM_TIMEOUT_ACC, 2, acc);
          break;
        }
        tc_fence_after_sync();
        const float2 s2 = make_float2(scale, scale);
        const uint32_t taddr = lane_base + static_cast<uint32_t>(acc * kFPTile);
        uint32_t r0[32], r1[32];                 // the next 32 columns are on their way while these are added
        if (left > 0) {
          tmem_ld32(taddr, r0);
          wait_loaded(r0);
          tmem_ld32(taddr + 32, r1);
#pragma unroll
          for (int i = 0; i < 16; ++i) fma2(sum[i], s2, r0[2 * i], r0[2 * i + 1]);
          wait_loaded(r1);
          tmem_ld32(taddr + 64, r0);
#pragma unroll
          for (int i = 0; i < 16; ++i) fma2(sum[16 + i], s2, r1[2 * i], r1[2 * i + 1]);
          wait_loaded(r0);
          tmem_ld32(taddr + 96, r1);
#pragma unroll
          for (int i = 0; i < 16; ++i) fma2(sum[32 + i], s2, r0[2 * i], r0[2 * i + 1]);
          wait_loaded(r1);
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster_relaxed(map_to_cta(smem_u32(&acc_empty[acc]), 0));
        if (left > 0) {
#pragma unroll
          for (int i = 0; i < 16; ++i) fma2(sum[48 + i], s2, r1[2 * i], r1[2 * i + 1]);
        }
        if (++acc == 2) { acc = 0; acc_phase ^= 1; }
       }
      }
      if (ok && lane < left) store_row(g, row, column, sum);
    }
    if (g.zero_rest && !skip) zero_rest_rows(table, g, blockIdx.x * kFPEpilogueWarps + warp - 4, gridDim.x * kFPEpilogueWarps);
  }

  tc_fence_before_sync();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem_base, kFPTmemCols);
  }
}

}  // namespace

cudaError_t launch_fp8_block_pairs(const CUtensorMap& map_a, const CUtensorMap& map_w, const FArgs& g, int most_tiles, cudaStream_t stream) {
  static int cached[64] = {};
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (cached[dev] == 0) {
    // the warpgroups can only trade registers that the launch gives them
    cudaFuncAttributes attr;
    err = cudaFuncGetAttributes(&attr, fp8_block_pair_kernel);
    if (err != cudaSuccess) return err;
    if (attr.numRegs != kLaunchRegs) return cudaErrorInvalidConfiguration;
    int clusters = 0;
    err = pair_clusters(fp8_block_pair_kernel, kFPSmem, &clusters, kFPThreads);
    if (err != cudaSuccess) return err;
    if (clusters <= 0) return cudaErrorLaunchOutOfResources;
    cached[dev] = clusters;
  }
  return launch_pairs_threads(fp8_block_pair_kernel, kFPSmem, most_tiles < cached[dev] ? most_tiles : cached[dev], kFPThreads, stream, map_a,
                              map_w, g);
}

}  // namespace sm100
}  // namespace msccl
