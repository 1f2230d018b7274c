// Gradient of the matrices of grouped products, for sm_100a:  dw[e, n, k] = sum over the rows t of group e of dy[t, n] x[t, k].
//
// Both operands are read as they lie in memory: the reduction runs over rows, so both are MN-major (64 features x 64 rows slabs of
// 8 KB).  CTA pairs (cta_group::2) compute 256 x 256 tiles; a group without rows writes zeros.  x is the M operand, so that
// the lanes of an accumulator run along k, the contiguous dimension of the result (dy as the M operand gave every lane a row of
// its own to store to, 16 bytes at a time: 8 groups of 1024 rows, n = k = 4096, 432 us).
//
// The reduction is ragged: the last 64-row block of a group also holds rows of the next group (or memory behind the last one,
// which may hold anything).  Those rows have to be zero in both operands, since 0 times infinity is not 0.  Loading that block
// completes on a barrier of the CTA's own instead of the leader's; a fix-up warp then clears the rows, orders its writes before
// the tensor core's reads and tells the MMA thread.  All other blocks never pass through it.
//
//   tail_full[s]    one per CTA: this CTA's loads of a last block (full[s] then completes without bytes).
//   tail_ready[s]   leader only, two arrivals: the fix-up warps of the pair.  The MMA thread waits for it before a last block.
// The other barriers are those of gemm_2cta_sm100.cu.  An arrival of each producer on the leader's barrier with every block (in place
// of tail_ready) releases memory at cluster scope and took 0.55 us of the 0.83 us per block.
#include <cuda.h>
#include <cuda_runtime.h>

#include <type_traits>

#include "expert_ops.h"
#include "gemm_sm100.cuh"
#include "gemm_sm100.h"
#include "grouped_common.cuh"
#include "umma_2cta.cuh"

namespace msccl {
namespace sm100 {

namespace {

constexpr int kWEpilogueWarps = 4;
constexpr int kWThreads = 96 + 32 * kWEpilogueWarps;      // 0 producer, 1 MMA, 2..5 epilogue, 6 fix-up
constexpr int kWTile = 256;
constexpr int kWOperand = 2 * kSlabBytes;        // 128 features x 64 rows
constexpr int kWStageBytes = 2 * kWOperand;
constexpr int kWStages = 6;
constexpr int kWTmemCols = 2 * kWTile;
constexpr size_t kWSmem = 1024 + static_cast<size_t>(kWStages) * kWStageBytes + 256;

struct WgradArgs {
  const int* offsets;
  void* out;
  long long ldo, lde;
  int rows, groups, n, k;
  int* error_words;
};

template <bool BF16, bool F32OUT>
__global__ void __launch_bounds__(kWThreads, 1)
grouped_wgrad_kernel(const __grid_constant__ CUtensorMap map_dy, const __grid_constant__ CUtensorMap map_x, const WgradArgs g) {
  constexpr int S = kWStages;
  extern __shared__ uint8_t smem_raw[];
  __shared__ GroupTable table;
  __shared__ int s_skip;
  uint8_t* stage_base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(stage_base + static_cast<size_t>(S) * kWStageBytes);
  uint64_t *full_bar = bars, *empty_bar = bars + S, *tail_full = bars + 2 * S, *tail_ready = bars + 3 * S;
  uint64_t *acc_full = bars + 4 * S, *acc_empty = bars + 4 * S + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 4 * S + 4);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int n_tiles = (g.n + kWTile - 1) / kWTile, k_tiles = (g.k + kWTile - 1) / kWTile;
  const int first = static_cast<int>(cluster_id_x()), step = static_cast<int>(num_clusters_x());
  const int per_group = n_tiles * k_tiles, num_tiles = per_group * g.groups;

  if (threadIdx.x == 0) {
    s_skip = g.error_words != nullptr && *reinterpret_cast<volatile int*>(g.error_words) != 0 ? 1 : 0;
    for (int s = 0; s < S; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
      mbar_init(&tail_full[s], 1);
      mbar_init(&tail_ready[s], 2);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], 2 * kWEpilogueWarps);
    }
    *abort_flag = 0;
    mbar_fence_init();
    prefetch_tensormap(&map_dy);
    prefetch_tensormap(&map_x);
  }
  if (warp == 1) tmem_alloc_pair(tmem_slot, kWTmemCols);
  if (warp == 2) build_groups(table, g.offsets, g.groups, g.rows, [](int) { return 0; });
  tc_fence_before_sync();
  cluster_sync_all();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  const bool skip = ld_shared_cluster_u32(map_to_cta(smem_u32(&s_skip), 0)) != 0;

  auto locate = [&](int tile, int& e, int& n0, int& k0) {
    e = tile / per_group;
    int tm, tn;
    tile_coords(tile - e * per_group, n_tiles, k_tiles, 8, tm, tn);
    n0 = tm * kWTile;
    k0 = tn * kWTile;
  };

  if (skip) {
    // fall through to the common exit
  } else if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = first; tile < num_tiles && ok; tile += step) {
        int e, n0, k0;
        locate(tile, e, n0, k0);
        n0 += static_cast<int>(rank) * BM;
        k0 += static_cast<int>(rank) * BM;
        const int lo = table.row_start[e], rows = table.row_start[e + 1] - lo;
        for (int r = 0; r < rows; r += BK) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1, abort_flag)) {
            gemm_fail(g.error_words, abort_flag, GEMM_TIMEOUT_EMPTY, 0, stage);
            ok = false;
            break;
          }
          uint8_t* dst = stage_base + static_cast<size_t>(stage) * kWStageBytes;
          const uint32_t bar = map_to_cta(smem_u32(&full_bar[stage]), 0);
          if (rows - r >= BK) {
            if (leader) mbar_expect_tx(&full_bar[stage], 2 * kWStageBytes);
            tma_pair_2d(dst, &map_x, bar, k0, lo + r);
            tma_pair_2d(dst + kSlabBytes, &map_x, bar, k0 + 64, lo + r);
            tma_pair_2d(dst + kWOperand, &map_dy, bar, n0, lo + r);
            tma_pair_2d(dst + kWOperand + kSlabBytes, &map_dy, bar, n0 + 64, lo + r);
          } else {
            if (leader) mbar_arrive(&full_bar[stage]);
            mbar_expect_tx(&tail_full[stage], kWStageBytes);
            tma_load_2d(dst, &map_x, &tail_full[stage], k0, lo + r);
            tma_load_2d(dst + kSlabBytes, &map_x, &tail_full[stage], k0 + 64, lo + r);
            tma_load_2d(dst + kWOperand, &map_dy, &tail_full[stage], n0, lo + r);
            tma_load_2d(dst + kWOperand + kSlabBytes, &map_dy, &tail_full[stage], n0 + 64, lo + r);
          }
          if (++stage == S) { stage = 0; phase ^= 1; }
        }
      }
      if (!ok) drain_wait();
    }
  } else if (warp == 1) {
    if (lane == 0 && leader) {
      constexpr uint32_t idesc = idesc_16bit(BF16, kWTile, kWTile) | kIdescTransA | kIdescTransB;
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0, tail_phase = 0;      // tail_phase: one bit per stage
      bool ok = true;
      for (int tile = first; tile < num_tiles && ok; tile += step) {
        const int e = tile / per_group, rows = table.row_start[e + 1] - table.row_start[e];
        if (rows == 0) continue;
        if (!mbar_wait(&acc_empty[acc], acc_phase ^ 1, abort_flag)) {
          gemm_fail(g.error_words, abort_flag, GEMM_TIMEOUT_ACC, 1, acc);
          break;
        }
        tc_fence_after_sync();
        const uint32_t tmem_d = tmem_base + static_cast<uint32_t>(acc * kWTile);
        for (int r = 0; r < rows; r += BK) {
          if (!mbar_wait(&full_bar[stage], phase, abort_flag)) {
            gemm_fail(g.error_words, abort_flag, GEMM_TIMEOUT_FULL, 1, stage);
            ok = false;
            break;
          }
          if (rows - r < BK) {
            if (!mbar_wait(&tail_ready[stage], (tail_phase >> stage) & 1u, abort_flag)) {
              gemm_fail(g.error_words, abort_flag, GEMM_TIMEOUT_FULL, 3, stage);
              ok = false;
              break;
            }
            tail_phase ^= 1u << stage;
          }
          tc_fence_after_sync();
          const uint32_t addr = smem_u32(stage_base + static_cast<size_t>(stage) * kWStageBytes);
          const uint64_t adesc = smem_desc_mn_sw128(addr), bdesc = smem_desc_mn_sw128(addr + kWOperand);
#pragma unroll
          for (int k = 0; k < BK / UMMA_K; ++k)
            umma_bf16_pair(tmem_d, adesc + static_cast<uint64_t>(k * 128), bdesc + static_cast<uint64_t>(k * 128), idesc, (r | k) != 0);
          tc_commit_pair(&empty_bar[stage], 3);
          if (++stage == S) { stage = 0; phase ^= 1; }
        }
        if (ok) tc_commit_pair(&acc_full[acc], 3);
        if (++acc == 2) { acc = 0; acc_phase ^= 1; }
      }
    }
  } else if (warp == 2 + kWEpilogueWarps) {
    int stage = 0;
    uint32_t tail_phase = 0;                     // one bit per stage
    for (int tile = first; tile < num_tiles; tile += step) {
      const int e = tile / per_group, rows = table.row_start[e + 1] - table.row_start[e];
      const int blocks = (rows + BK - 1) / BK, left = rows % BK;
      if (left != 0) {
        const int s = (stage + blocks - 1) % S;
        bool ok = mbar_wait(&tail_full[s], (tail_phase >> s) & 1u, abort_flag);
        ok = __all_sync(kFullMask, ok);
        if (!ok) {
          if (lane == 0) gemm_fail(g.error_words, abort_flag, GEMM_TIMEOUT_FULL, 3, s);
          break;
        }
        tail_phase ^= 1u << s;
        // four slabs of 64 rows x 128 bytes: 8 lanes clear a row of each
        uint8_t* base = stage_base + static_cast<size_t>(s) * kWStageBytes + (lane % 8) * 16;
        for (int r = left + lane / 8; r < BK; r += 4)
#pragma unroll
          for (int slab = 0; slab < 4; ++slab) *reinterpret_cast<uint4*>(base + slab * kSlabBytes + r * 128) = make_uint4(0, 0, 0, 0);
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(map_to_cta(smem_u32(&tail_ready[s]), 0));
      }
      stage = (stage + blocks) % S;
    }
  } else {
    const int quarter = warp % 4;
    int acc = 0;
    uint32_t acc_phase = 0;
    for (int tile = first; tile < num_tiles; tile += step) {
      int e, n0, k0;
      locate(tile, e, n0, k0);
      const bool empty = table.row_start[e + 1] == table.row_start[e];
      if (!empty) {
        bool ok = mbar_wait(&acc_full[acc], acc_phase, abort_flag);
        ok = __all_sync(kFullMask, ok);
        if (!ok) {
          if (lane == 0) gemm_fail(g.error_words, abort_flag, GEMM_TIMEOUT_ACC, 2, acc);
          break;
        }
        tc_fence_after_sync();
      }
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(acc * kWTile);
      const int columns = min(kWTile, g.n - n0);
      // fp32: a lane stores value k of row n0 + c + i; 16 bits: values k .. k + 7 of row n0 + c + 8 m + lane % 8
      const int k = k0 + static_cast<int>(rank) * BM + quarter * 32 + (F32OUT ? lane : lane & ~7), lane_row = F32OUT ? 0 : lane & 7;
      const bool in = k < g.k;
      using Out = std::conditional_t<F32OUT, float, uint16_t>;
      Out* dst = static_cast<Out*>(g.out) + e * g.lde + (n0 + lane_row) * g.ldo + k;
      const long long row8 = 8 * g.ldo;
      for (int c = 0; c < columns; c += 32) {
        uint32_t r[32];
        if (empty) {
#pragma unroll
          for (int i = 0; i < 32; ++i) r[i] = 0u;
        } else {
          tmem_ld32(taddr + c, r);
          wait_loaded(r);
        }
        const int left = in ? columns - c - lane_row : 0;      // rows from this lane's first on
        if constexpr (F32OUT) {
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            if (i < left) *dst = __uint_as_float(r[i]);
            dst += g.ldo;
          }
        } else {
          uint4 v[4];
          transpose_chunk<BF16>(r, lane, v);
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            if (8 * m < left) *reinterpret_cast<uint4*>(dst) = v[m];
            dst += row8;
          }
        }
      }
      if (!empty) {
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster_relaxed(map_to_cta(smem_u32(&acc_empty[acc]), 0));
        if (++acc == 2) { acc = 0; acc_phase ^= 1; }
      }
    }
  }

  tc_fence_before_sync();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem_base, kWTmemCols);
  }
}

template <bool BF16, bool F32OUT>
cudaError_t launch(const CUtensorMap& map_dy, const CUtensorMap& map_x, const WgradArgs& g, int tiles, cudaStream_t stream) {
  static int cached[64] = {};
  auto kernel = grouped_wgrad_kernel<BF16, F32OUT>;
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (cached[dev] == 0) {
    int clusters = 0;
    err = pair_clusters(kernel, kWSmem, &clusters, kWThreads);
    if (err != cudaSuccess) return err;
    if (clusters <= 0) return cudaErrorLaunchOutOfResources;
    cached[dev] = clusters;
  }
  return launch_pairs_threads(kernel, kWSmem, tiles < cached[dev] ? tiles : cached[dev], kWThreads, stream, map_dy, map_x, g);
}

}  // namespace

// dy: [rows, n], x: [rows, k], out: [groups, n, k] (pitch ldo, matrix stride lde), of the operands' type or fp32.
cudaError_t launch_grouped_wgrad(const void* dy, long long lddy, const void* x, long long ldx, const int* offsets, void* out, long long ldo,
                                 long long lde, int rows, int groups, int n, int k, int elem, bool f32_out, int* error_words,
                                 cudaStream_t stream) {
  if (rows < 1 || groups < 1 || groups > kMaxGroups || n < 8 || k < 8 || n % 8 != 0 || k % 8 != 0 || lddy % 8 != 0 || ldx % 8 != 0 ||
      ldo % (f32_out ? 4 : 8) != 0 || lde % (f32_out ? 4 : 8) != 0 || (elem != kElemBF16 && elem != kElemF16))
    return cudaErrorInvalidValue;
  WgradArgs g;
  g.offsets = offsets;
  g.out = out;
  g.ldo = ldo;
  g.lde = lde;
  g.rows = rows;
  g.groups = groups;
  g.n = n;
  g.k = k;
  g.error_words = error_words;
  const uint32_t box[2] = {64, 64};
  const uint64_t dy_dims[2] = {static_cast<uint64_t>(n), static_cast<uint64_t>(rows)}, dy_strides[1] = {static_cast<uint64_t>(lddy) * 2};
  const uint64_t x_dims[2] = {static_cast<uint64_t>(k), static_cast<uint64_t>(rows)}, x_strides[1] = {static_cast<uint64_t>(ldx) * 2};
  const CUtensorMap map_dy = make_swizzled_map(dy, 2, 2, dy_dims, dy_strides, box);
  const CUtensorMap map_x = make_swizzled_map(x, 2, 2, x_dims, x_strides, box);
  const long long tiles = static_cast<long long>(groups) * ((n + kWTile - 1) / kWTile) * ((k + kWTile - 1) / kWTile);
  if (tiles > (1ll << 30)) return cudaErrorInvalidValue;
  const bool bf16 = elem == kElemBF16;
  if (f32_out) return bf16 ? launch<true, true>(map_dy, map_x, g, static_cast<int>(tiles), stream) : launch<false, true>(map_dy, map_x, g, static_cast<int>(tiles), stream);
  return bf16 ? launch<true, false>(map_dy, map_x, g, static_cast<int>(tiles), stream) : launch<false, false>(map_dy, map_x, g, static_cast<int>(tiles), stream);
}

}  // namespace sm100
}  // namespace msccl
