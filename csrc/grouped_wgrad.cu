// Gradient of the matrices of grouped products, for sm_100a:  dw[e, n, k] = sum over the rows t of group e of dy[t, n] x[t, k].
//
// Both operands are read as they lie in memory: the reduction runs over rows, so both are MN-major (64 features x 64 rows slabs of
// 8 KB).  CTA pairs (cta_group::2) compute 256 x 256 tiles; a group without rows writes zeros.  8 groups of 1024 rows, n = k = 4096:
// 168 us, 1.64 PFLOP/s; of few rows the writes of the result are the bound (64 groups of 64 rows, n = k = 2048: 139 us, 3.9 TB/s).
//
// Stores of whole lines: in 16 bits dy is the M operand, a lane of the accumulator is a row n, and eight lanes exchange pieces so that
// they store 128 consecutive bytes of k.  (With the lanes along k a warp has 64 bytes of a row, and the same 64 groups took 215 us.)
// For fp32 x is the M operand: 32 lanes along k are 128 bytes without an exchange (the exchange: 8 x 1024 rows 2 % more).
//
// The reduction is ragged: the last 64-row block of a group also covers rows of the next group (or memory behind the last one, which
// may hold anything).  Those rows have to be zero in both operands, since 0 times infinity is not 0.  So that block goes a way of
// its own: a fix-up warp in each CTA loads it into a buffer beside the pipeline, clears the rows, orders its writes before the tensor
// core's reads and tells the MMA thread, which takes the block last.  The buffer is free again when the tile is done, so the block
// of the next tile is ready long before its turn.  (Through the pipeline, every such block held up the tensor core for
// 1.5 us.  A second buffer in place of the sixth stage: 8 x 1000 rows, n = k = 4096, 169 instead of 178 us, but 2 x 4096 rows 217 instead of
// 173.)
//
//   tail_full    one per CTA: this CTA's loads of the block.      tail_empty   one per CTA: its MMAs are done (commit).
//   tail_ready   leader only, two arrivals: the fix-up warps of the pair.
// The other barriers are those of gemm_2cta_sm100.cu.  An arrival of each producer on the leader's barrier with every block releases
// memory at cluster scope and took 0.55 us of 0.83 us per block; nothing of that kind is in the loop.
#include <cuda.h>
#include <cuda_runtime.h>

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
// the pipeline, the block on its own, row_start of the groups, the barriers: 226 KB, so the base has to be aligned as it is
constexpr int kWTableBytes = (kMaxGroups + 1) * 4 + 12;
constexpr size_t kWSmem = static_cast<size_t>(kWStages + 1) * kWStageBytes + kWTableBytes + 256;
// All CTAs finish a tile of equal groups at about the same time.  Stored at once, their results hold up the loads of the next tiles for longer
// than the pipeline lasts, so from kWPacedRows rows on, where the products leave time, the stores are spread out by a pause (in ns)
// after every 64 values of a row, or half of it after every 32 rows of fp32.  n = k = 4096, without / with pauses: 8 x 1024 rows
// 174 / 168 us, in fp32 213 / 205; 8 x 768 rows 139 / 139, in fp32 176 / 165; 2 x 4096 rows the same.
constexpr int kWPacedRows = 768, kWPause = 500;
static_assert(kWSmem <= 227 * 1024 && kWTableBytes % 16 == 0, "");

struct WgradArgs {
  const int* offsets;
  void* out;
  long long ldo, lde;
  int rows, groups, n, k;
  int* error_words;
};

// 64 columns of this lane's row of the accumulator as 16-bit values, in eight pieces of eight.
template <bool BF16>
__device__ __forceinline__ void load_row(uint32_t taddr, uint4 (&v)[8]) {
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    uint32_t r[32];
    tmem_ld32(taddr + 32 * half, r);
    wait_loaded(r);
    auto pack = [&](int i) { return pack_16bit(BF16, __uint_as_float(r[i]), __uint_as_float(r[i + 1])); };
#pragma unroll
    for (int i = 0; i < 4; ++i) v[4 * half + i] = make_uint4(pack(8 * i), pack(8 * i + 2), pack(8 * i + 4), pack(8 * i + 6));
  }
}

// From piece i of the lane's own row to piece lane % 8 of row i of its eight lanes, which then store 128 consecutive bytes together.
// An exchange for each bit that lane and piece swap, 48 shuffles.
__device__ __forceinline__ void transpose_lines(uint4 (&v)[8], int lane) {
#pragma unroll
  for (int bit = 1; bit < 8; bit *= 2) {
    const bool up = (lane & bit) != 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i & bit) continue;
      uint4 &low = v[i], &high = v[i | bit];
      const uint4 give = up ? low : high;
      uint4 got;
      got.x = __shfl_xor_sync(kFullMask, give.x, bit);
      got.y = __shfl_xor_sync(kFullMask, give.y, bit);
      got.z = __shfl_xor_sync(kFullMask, give.z, bit);
      got.w = __shfl_xor_sync(kFullMask, give.w, bit);
      if (up) low = got;
      else high = got;
    }
  }
}

template <bool BF16, bool F32OUT>
__global__ void __launch_bounds__(kWThreads, 1)
grouped_wgrad_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const WgradArgs g) {
  constexpr int S = kWStages;
  extern __shared__ __align__(1024) uint8_t stage_base[];
  uint8_t* tail_base = stage_base + static_cast<size_t>(S) * kWStageBytes;
  int* row_start = reinterpret_cast<int*>(tail_base + kWStageBytes);
  uint64_t* bars = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(row_start) + kWTableBytes);
  uint64_t *full_bar = bars, *empty_bar = bars + S, *acc_full = bars + 2 * S, *acc_empty = bars + 2 * S + 2;
  uint64_t *tail_full = bars + 2 * S + 4, *tail_ready = tail_full + 1, *tail_empty = tail_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * S + 8);
  int* s_skip = reinterpret_cast<int*>(tmem_slot + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 2);

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int n_tiles = (g.n + kWTile - 1) / kWTile, k_tiles = (g.k + kWTile - 1) / kWTile;
  const int first = static_cast<int>(cluster_id_x()), step = static_cast<int>(num_clusters_x());
  const int per_group = n_tiles * k_tiles, num_tiles = per_group * g.groups;

  if (threadIdx.x == 0) {
    // an earlier launch gave up: skip the work; the leader's reading decides for the pair
    *s_skip = g.error_words != nullptr && *reinterpret_cast<volatile int*>(g.error_words) != 0 ? 1 : 0;
    for (int s = 0; s < S; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    mbar_init(tail_full, 1);
    mbar_init(tail_ready, 2);
    mbar_init(tail_empty, 1);
    for (int a = 0; a < 2; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], 2 * kWEpilogueWarps);
    }
    *abort_flag = 0;
    if (smem_u32(stage_base) % 1024 != 0) {        // the swizzle pattern starts on such a boundary: nothing would be right
      *s_skip = 1;
      gemm_fail(g.error_words, abort_flag, GEMM_TIMEOUT_EMPTY, 9, 0);
    }
    mbar_fence_init();
    prefetch_tensormap(&map_a);
    prefetch_tensormap(&map_b);
  }
  if (warp == 1) tmem_alloc_pair(tmem_slot, kWTmemCols);
  if (warp == 2) build_row_starts(row_start, g.offsets, g.groups, g.rows);
  tc_fence_before_sync();
  cluster_sync_all();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  const bool skip = ld_shared_cluster_u32(map_to_cta(smem_u32(s_skip), 0)) != 0;

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
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = first; tile < num_tiles && ok; tile += step) {
        int e, n0, k0;
        locate(tile, e, n0, k0);
        const int a0 = (F32OUT ? k0 : n0) + static_cast<int>(rank) * BM, b0 = (F32OUT ? n0 : k0) + static_cast<int>(rank) * BM;
        const int lo = row_start[e], end = row_start[e + 1];
        for (int r = lo; r + BK <= end; r += BK) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1, abort_flag)) {
            gemm_fail(g.error_words, abort_flag, GEMM_TIMEOUT_EMPTY, 0, stage);
            ok = false;
            break;
          }
          uint8_t* dst = stage_base + static_cast<size_t>(stage) * kWStageBytes;
          const uint32_t bar = map_to_cta(smem_u32(&full_bar[stage]), 0);
          if (leader) mbar_expect_tx(&full_bar[stage], 2 * kWStageBytes);
          tma_pair_2d(dst, &map_a, bar, a0, r);
          tma_pair_2d(dst + kSlabBytes, &map_a, bar, a0 + 64, r);
          tma_pair_2d(dst + kWOperand, &map_b, bar, b0, r);
          tma_pair_2d(dst + kWOperand + kSlabBytes, &map_b, bar, b0 + 64, r);
          if (++stage == S) { stage = 0; phase ^= 1; }
        }
      }
      if (!ok) drain_wait();
    }
  } else if (warp == 1) {
    if (leader && elect_one()) {
      constexpr uint32_t idesc = idesc_16bit(BF16, kWTile, kWTile) | kIdescTransA | kIdescTransB;
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0, tail_phase = 0;
      auto block = [&](uint32_t addr, uint32_t tmem_d, bool accumulate) {
        const uint64_t adesc = smem_desc_mn_sw128(addr), bdesc = smem_desc_mn_sw128(addr + kWOperand);
#pragma unroll
        for (int k = 0; k < BK / UMMA_K; ++k)
          umma_bf16_pair(tmem_d, adesc + static_cast<uint64_t>(k * 128), bdesc + static_cast<uint64_t>(k * 128), idesc, accumulate || k != 0);
      };
      bool ok = true;
      for (int tile = first; tile < num_tiles && ok; tile += step) {
        const int e = tile / per_group, rows = row_start[e + 1] - row_start[e];
        if (rows == 0) continue;
        if (!mbar_wait(&acc_empty[acc], acc_phase ^ 1, abort_flag)) {
          gemm_fail(g.error_words, abort_flag, GEMM_TIMEOUT_ACC, 1, acc);
          break;
        }
        tc_fence_after_sync();
        const uint32_t tmem_d = tmem_base + static_cast<uint32_t>(acc * kWTile);
        for (int r = 0; r + BK <= rows; r += BK) {
          if (!mbar_wait(&full_bar[stage], phase, abort_flag)) {
            gemm_fail(g.error_words, abort_flag, GEMM_TIMEOUT_FULL, 1, stage);
            ok = false;
            break;
          }
          tc_fence_after_sync();
          block(smem_u32(stage_base + static_cast<size_t>(stage) * kWStageBytes), tmem_d, r != 0);
          tc_commit_pair(&empty_bar[stage], 3);
          if (++stage == S) { stage = 0; phase ^= 1; }
        }
        if (ok && rows % BK != 0) {
          if (!mbar_wait(tail_ready, tail_phase, abort_flag)) {
            gemm_fail(g.error_words, abort_flag, GEMM_TIMEOUT_FULL, 1, S);
            break;
          }
          tail_phase ^= 1;
          tc_fence_after_sync();
          block(smem_u32(tail_base), tmem_d, rows > BK);
          tc_commit_pair(tail_empty, 3);
        }
        if (ok) tc_commit_pair(&acc_full[acc], 3);
        if (++acc == 2) { acc = 0; acc_phase ^= 1; }
      }
    }
  } else if (warp == 2 + kWEpilogueWarps) {
    uint32_t phase = 0;
    for (int tile = first; tile < num_tiles; tile += step) {
      int e, n0, k0;
      locate(tile, e, n0, k0);
      const int a0 = (F32OUT ? k0 : n0) + static_cast<int>(rank) * BM, b0 = (F32OUT ? n0 : k0) + static_cast<int>(rank) * BM;
      const int left = (row_start[e + 1] - row_start[e]) % BK, r0 = row_start[e + 1] - left;
      if (left == 0) continue;
      bool ok = mbar_wait_warp(tail_empty, phase ^ 1, abort_flag);
      if (ok) {
        if (elect_one()) {
          mbar_expect_tx(tail_full, kWStageBytes);
          tma_load_2d(tail_base, &map_a, tail_full, a0, r0);
          tma_load_2d(tail_base + kSlabBytes, &map_a, tail_full, a0 + 64, r0);
          tma_load_2d(tail_base + kWOperand, &map_b, tail_full, b0, r0);
          tma_load_2d(tail_base + kWOperand + kSlabBytes, &map_b, tail_full, b0 + 64, r0);
        }
        __syncwarp();
        ok = mbar_wait_warp(tail_full, phase, abort_flag);
        if (!ok) drain_wait();
      }
      if (!ok) {
        if (lane == 0) gemm_fail(g.error_words, abort_flag, GEMM_TIMEOUT_FULL, 3, 0);
        break;
      }
      phase ^= 1;
      // four slabs of 64 rows x 128 bytes: 8 lanes clear a row of each
      for (int r = left + lane / 8; r < BK; r += 4)
#pragma unroll
        for (int slab = 0; slab < 4; ++slab)
          *reinterpret_cast<uint4*>(tail_base + slab * kSlabBytes + r * 128 + (lane % 8) * 16) = make_uint4(0, 0, 0, 0);
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(map_to_cta(smem_u32(tail_ready), 0));
    }
  } else {
    const int quarter = warp % 4;
    int acc = 0;
    uint32_t acc_phase = 0;
    for (int tile = first; tile < num_tiles; tile += step) {
      int e, n0, k0;
      locate(tile, e, n0, k0);
      const bool empty = row_start[e + 1] == row_start[e];
      if (!empty) {
        bool ok = mbar_wait_warp(&acc_full[acc], acc_phase, abort_flag);
        if (!ok) {
          if (lane == 0) gemm_fail(g.error_words, abort_flag, GEMM_TIMEOUT_ACC, 2, acc);
          break;
        }
        tc_fence_after_sync();
      }
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(acc * kWTile);
      const int lanes_at = static_cast<int>(rank) * BM + quarter * 32;
      const bool paced = row_start[e + 1] - row_start[e] >= kWPacedRows && tile + step < num_tiles;
      if constexpr (F32OUT) {
        // a lane stores value k of the rows n0, n0 + 1, ...
        const int columns = min(kWTile, g.n - n0), k = k0 + lanes_at + lane;
        float* dst = static_cast<float*>(g.out) + e * g.lde + n0 * g.ldo + k;
        for (int c = 0; c < columns; c += 32) {
          uint32_t r[32];
          if (empty) {
#pragma unroll
            for (int i = 0; i < 32; ++i) r[i] = 0u;
          } else {
            tmem_ld32(taddr + c, r);
            wait_loaded(r);
          }
          const int left = k < g.k ? columns - c : 0;
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            if (i < left) *dst = __uint_as_float(r[i]);
            dst += g.ldo;
          }
          if (paced) __nanosleep(kWPause / 2);
        }
      } else {
        // after the exchange a lane has values k .. k + 7 of the rows n, n + 1, ... n + 7
        const int columns = min(kWTile, g.k - k0), n = n0 + lanes_at + (lane & ~7), k = 8 * (lane & 7), left = g.n - n;
        uint16_t* dst = static_cast<uint16_t*>(g.out) + e * g.lde + n * g.ldo + k0 + k;
        for (int c = 0; c < columns; c += 64) {
          uint4 v[8];
          if (empty) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = make_uint4(0u, 0u, 0u, 0u);
          } else {
            load_row<BF16>(taddr + c, v);
            transpose_lines(v, lane);
          }
          if (c + k < columns) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (i < left) *reinterpret_cast<uint4*>(dst + i * g.ldo) = v[i];
          }
          dst += 64;
          if (paced) __nanosleep(kWPause);
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
  return launch_pairs_threads(kernel, kWSmem, tiles < cached[dev] ? tiles : cached[dev], kWThreads, stream, F32OUT ? map_x : map_dy, F32OUT ? map_dy : map_x, g);
}

}  // namespace

// dy: [rows, n], x: [rows, k], out: [groups, n, k] (pitch ldo, matrix stride lde), of the operands' type or fp32.
cudaError_t launch_grouped_wgrad(const void* dy, long long lddy, const void* x, long long ldx, const int* offsets, void* out, long long ldo,
                                 long long lde, int rows, int groups, int n, int k, int elem, bool f32_out, int* error_words,
                                 cudaStream_t stream) {
  if (rows < 1 || rows > kMaxRows || groups < 1 || groups > kMaxGroups || n < 8 || n > kMaxRows || k < 8 || k > kMaxRows || n % 8 != 0 || k % 8 != 0 || lddy % 8 != 0 || ldx % 8 != 0 ||
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
  auto run = f32_out ? (bf16 ? launch<true, true> : launch<false, true>) : (bf16 ? launch<true, false> : launch<false, false>);
  return run(map_dy, map_x, g, static_cast<int>(tiles), stream);
}

}  // namespace sm100
}  // namespace msccl
