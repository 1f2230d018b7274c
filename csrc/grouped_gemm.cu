// Products of the rows of every group with the group's matrix, for sm_100a:
//
//   forward    y[t, n]  = sum_k x[t, k]  w[e, n, k]        (w K-major: the reduction dimension is the contiguous one)
//   backward   dx[t, k] = sum_n dy[t, n] w[e, n, k]        (w MN-major: read through descriptors, no transposed copy)
//
// for the rows t of group e, [offsets[e], offsets[e + 1]).  bf16 or fp16 in and out, fp32 accumulators.  Group sizes are known on
// the device only: every CTA derives the same list of tiles from the offsets, so nothing is copied to the host.
//
// The weights are the M operand and the rows of the group the N operand of the MMA: 256 features (of a CTA pair, cta_group::2)
// by up to BN = 64 or 256 rows; N is a field of the instruction, so a group of 700 rows is cut into 256 + 256 + 188 or, better, into
// three about equal tiles, in steps of 32 rows.  8192 rows in 8 unequal groups of 14336 x 4096: 611 us, 1.58 PFLOP/s, with equal tiles,
// 693 with full ones and a narrow last one (the pair that gets one full tile more sets the time), 825 run without a pause with full
// ones only, 784 with equal ones (the power cap).  Rows of a tile that belong to the next group only reach columns of the accumulator
// that are not stored, whatever they hold.  What is left of both operands behind the reduction dimension reads as zero.
//
// The accumulator holds a feature per lane and a row per column; the epilogue transposes it (transpose_chunk).
//
// Synchronisation is that of gemm_2cta_sm100.cu.
#include <cuda.h>
#include <cuda_runtime.h>

#include <stdexcept>

#include "expert_ops.h"
#include "gemm_sm100.cuh"
#include "gemm_sm100.h"
#include "grouped_common.cuh"
#include "umma_2cta.cuh"

namespace msccl {
namespace sm100 {

namespace {

constexpr int kGroupTileRows = 2048;             // rows that a group of tiles walks together (L2, see tile_coords)
constexpr int kGEpilogueWarps = 8;               // two on each quarter of the lanes
constexpr int kGThreads = 64 + 32 * kGEpilogueWarps;
constexpr int kGABytes = BM * BK * 2;            // this CTA's 128 features: 16 KB
constexpr int kGSmemLimit = 220 * 1024;

template <int BN> struct Geometry {
  static constexpr int kPiece = 32 * BK * 2;                 // rows of the last tile of a group come in pieces of 32 per CTA
  static constexpr int kBBytes = BN / 2 * BK * 2;
  static constexpr int kStageBytes = kGABytes + kBBytes;
  static constexpr int kFit = (kGSmemLimit - 2048) / kStageBytes;
  static constexpr int kStages = kFit < 10 ? kFit : 10;
  static constexpr size_t kSmem = 1024 + static_cast<size_t>(kStages) * kStageBytes + 256;
  static constexpr int kTmemCols = 2 * BN;
};

struct GroupedArgs {
  const int* offsets;
  uint16_t* out;
  long long ldo;
  int rows, groups, features, reduction;
  int zero_rest;                                 // rows of no group become zero
  int* error_words;
};

template <int BN, bool MN_MAJOR, bool BF16>
__global__ void __launch_bounds__(kGThreads, 1)
grouped_gemm_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                    const __grid_constant__ CUtensorMap map_piece, const GroupedArgs g) {
  using Geo = Geometry<BN>;
  constexpr int S = Geo::kStages;
  extern __shared__ uint8_t smem_raw[];
  __shared__ GroupTable table;
  __shared__ int s_skip;
  uint8_t* stage_base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(stage_base + static_cast<size_t>(S) * Geo::kStageBytes);
  uint64_t *full_bar = bars, *empty_bar = bars + S, *acc_full = bars + 2 * S, *acc_empty = bars + 2 * S + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * S + 4);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int f_tiles = (g.features + 2 * BM - 1) / (2 * BM);
  const int k_blocks = (g.reduction + BK - 1) / BK;
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
      mbar_init(&acc_empty[a], 2 * kGEpilogueWarps);
    }
    *abort_flag = 0;
    mbar_fence_init();
    prefetch_tensormap(&map_w);
    prefetch_tensormap(&map_x);
    prefetch_tensormap(&map_piece);
  }
  if (warp == 1) tmem_alloc_pair(tmem_slot, Geo::kTmemCols);
  if (warp == 2) build_groups(table, g.offsets, g.groups, g.rows, [&](int rows) { return (rows + BN - 1) / BN * f_tiles; });
  tc_fence_before_sync();
  cluster_sync_all();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  const bool skip = ld_shared_cluster_u32(map_to_cta(smem_u32(&s_skip), 0)) != 0;
  const int num_tiles = table.tile_start[g.groups];

  // tile -> group e, first row, width (rows, a multiple of 32) and first feature; e only moves forward.  A group of r rows has
  // ceil(r / BN) tiles; since all but one of them at full width would not hold it, none of them is empty at any width that holds it.
  auto locate = [&](int tile, int& e, int& row, int& width, int& feature) {
    while (tile >= table.tile_start[e + 1]) ++e;
    const int rows = table.row_start[e + 1] - table.row_start[e];
    int tm, tn;
    const int tiles = (rows + BN - 1) / BN, each = ((rows + tiles - 1) / tiles + 31) / 32 * 32;
    tile_coords(tile - table.tile_start[e], tiles, f_tiles, kGroupTileRows / BN, tm, tn);
    row = table.row_start[e] + tm * each;
    width = min(each, (table.row_start[e + 1] - row + 31) / 32 * 32);
    feature = tn * 2 * BM;
  };

  if (skip) {
    // fall through to the common exit
  } else if (warp == 0) {
    if (elect_one()) {
      int stage = 0, e = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = first; tile < num_tiles && ok; tile += step) {
        int row, width, feature;
        locate(tile, e, row, width, feature);
        const int pieces = (width / 2 + 31) / 32;      // of this CTA's width / 2 rows
        const bool whole = pieces * Geo::kPiece == Geo::kBBytes;
        const uint32_t bytes = kGABytes + pieces * Geo::kPiece;
        row += static_cast<int>(rank) * (width / 2);
        feature += static_cast<int>(rank) * BM;
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1, abort_flag)) {
            gemm_fail(g.error_words, abort_flag, GEMM_TIMEOUT_EMPTY, 0, stage);
            ok = false;
            break;
          }
          uint8_t* a_dst = stage_base + static_cast<size_t>(stage) * Geo::kStageBytes;
          if (leader) mbar_expect_tx(&full_bar[stage], 2 * bytes);
          const uint32_t bar = map_to_cta(smem_u32(&full_bar[stage]), 0);
          if (MN_MAJOR) {
            tma_pair_3d(a_dst, &map_w, bar, feature, kb * BK, e);
            tma_pair_3d(a_dst + kSlabBytes, &map_w, bar, feature + 64, kb * BK, e);
          } else {
            tma_pair_3d(a_dst, &map_w, bar, kb * BK, feature, e);
          }
          if (whole) {
            tma_pair_2d(a_dst + kGABytes, &map_x, bar, kb * BK, row);
          } else {
            for (int p = 0; p < pieces; ++p) tma_pair_2d(a_dst + kGABytes + p * Geo::kPiece, &map_piece, bar, kb * BK, row + 32 * p);
          }
          if (++stage == S) { stage = 0; phase ^= 1; }
        }
      }
      if (!ok) drain_wait();
    }
  } else if (warp == 1) {
    if (leader && elect_one()) {
      constexpr uint32_t idesc_rest = idesc_16bit(BF16, 2 * BM, 0) | (MN_MAJOR ? kIdescTransA : 0u);
      int stage = 0, acc = 0, e = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int tile = first; tile < num_tiles && ok; tile += step) {
        int row, width, feature;
        locate(tile, e, row, width, feature);
        const uint32_t idesc = idesc_rest | static_cast<uint32_t>(width >> 3) << 17;
        if (!mbar_wait(&acc_empty[acc], acc_phase ^ 1, abort_flag)) {
          gemm_fail(g.error_words, abort_flag, GEMM_TIMEOUT_ACC, 1, acc);
          break;
        }
        tc_fence_after_sync();
        const uint32_t tmem_d = tmem_base + static_cast<uint32_t>(acc * BN);
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!mbar_wait(&full_bar[stage], phase, abort_flag)) {
            gemm_fail(g.error_words, abort_flag, GEMM_TIMEOUT_FULL, 1, stage);
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t a_addr = smem_u32(stage_base + static_cast<size_t>(stage) * Geo::kStageBytes);
          const uint64_t adesc = MN_MAJOR ? smem_desc_mn_sw128(a_addr) : smem_desc_sw128(a_addr);
          const uint64_t bdesc = smem_desc_sw128(a_addr + kGABytes);
          constexpr uint64_t a_step = MN_MAJOR ? 16 * 128 / 16 : 2;      // 16 reduction elements, in units of 16 bytes
#pragma unroll
          for (int k = 0; k < BK / UMMA_K; ++k)
            umma_bf16_pair(tmem_d, adesc + k * a_step, bdesc + static_cast<uint64_t>(k * 2), idesc, (kb | k) != 0);
          tc_commit_pair(&empty_bar[stage], 3);
          if (++stage == S) { stage = 0; phase ^= 1; }
        }
        if (ok) tc_commit_pair(&acc_full[acc], 3);
        if (++acc == 2) { acc = 0; acc_phase ^= 1; }
      }
    }
  } else {
    const int quarter = warp % 4, half = (warp - 2) / 4;      // the halves take every other chunk of 32 columns
    int acc = 0, e = 0;
    uint32_t acc_phase = 0;
    for (int tile = first; tile < num_tiles; tile += step) {
      int row, width, feature;
      locate(tile, e, row, width, feature);
      const int row_end = table.row_start[e + 1];
      bool ok = mbar_wait_warp(&acc_full[acc], acc_phase, abort_flag);
      if (!ok) {
        if (lane == 0) gemm_fail(g.error_words, abort_flag, GEMM_TIMEOUT_ACC, 2, acc);
        break;
      }
      tc_fence_after_sync();
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(acc * BN);
      const int f = feature + static_cast<int>(rank) * BM + quarter * 32 + (lane & ~7);       // this lane stores features f .. f + 7
      const bool in = f < g.features;
      const int columns = min(width, row_end - row);
      for (int c = half * 32; c < columns; c += 64) {
        uint32_t r[32];
        tmem_ld32(taddr + c, r);
        wait_loaded(r);
        uint4 v[4];
        transpose_chunk<BF16>(r, lane, v);
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          const int t = c + 8 * m + (lane & 7);
          if (in && t < columns) *reinterpret_cast<uint4*>(g.out + (row + t) * g.ldo + f) = v[m];
        }
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster_relaxed(map_to_cta(smem_u32(&acc_empty[acc]), 0));
      if (++acc == 2) { acc = 0; acc_phase ^= 1; }
    }
    if (g.zero_rest) {                           // rows before the first group and behind the last one
      const int head = table.row_start[0], tail = table.row_start[g.groups];
      const int rest = head + g.rows - tail;
      for (int i = blockIdx.x * kGEpilogueWarps + warp - 2; i < rest; i += gridDim.x * kGEpilogueWarps) {
        uint4* dst = reinterpret_cast<uint4*>(g.out + static_cast<long long>(i < head ? i : tail + i - head) * g.ldo);
        for (int v = lane; v < g.features / 8; v += 32) dst[v] = make_uint4(0, 0, 0, 0);
      }
    }
  }

  tc_fence_before_sync();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem_base, Geo::kTmemCols);
  }
}

template <int BN, bool MN_MAJOR, bool BF16>
cudaError_t launch(const CUtensorMap& map_w, const CUtensorMap& map_x, const CUtensorMap& map_piece, const GroupedArgs& g, int most_tiles,
                   cudaStream_t stream) {
  static int cached[64] = {};
  auto kernel = grouped_gemm_kernel<BN, MN_MAJOR, BF16>;
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (cached[dev] == 0) {
    int clusters = 0;
    err = pair_clusters(kernel, Geometry<BN>::kSmem, &clusters, kGThreads);
    if (err != cudaSuccess) return err;
    if (clusters <= 0) return cudaErrorLaunchOutOfResources;
    cached[dev] = clusters;
  }
  return launch_pairs_threads(kernel, Geometry<BN>::kSmem, most_tiles < cached[dev] ? most_tiles : cached[dev], kGThreads, stream, map_w, map_x,
                              map_piece, g);
}

template <int BN>
cudaError_t launch_by_type(bool mn_major, bool bf16, const CUtensorMap& map_w, const CUtensorMap& map_x, const CUtensorMap& map_piece,
                           const GroupedArgs& g, int most_tiles, cudaStream_t stream) {
  auto run = mn_major ? (bf16 ? launch<BN, true, true> : launch<BN, true, false>) : (bf16 ? launch<BN, false, true> : launch<BN, false, false>);
  return run(map_w, map_x, map_piece, g, most_tiles, stream);
}

}  // namespace

// w: [groups, n, k] (pitch ldw, matrix stride lde, elements); x: [rows, k] and out: [rows, n], or with `backward` x: [rows, n]
// (dy) and out: [rows, k].  n % 8 == 0, k % 8 == 0, everything 16-byte aligned.  bn: 64 or 256 rows per tile.
cudaError_t launch_grouped_gemm(const void* x, long long ldx, const void* w, long long ldw, long long lde, const int* offsets, void* out,
                                long long ldo, int rows, int groups, int n, int k, bool backward, int elem, int bn, bool zero_rest,
                                int* error_words, cudaStream_t stream) {
  if (rows < 1 || rows > kMaxRows || groups < 1 || groups > kMaxGroups || n < 8 || n > kMaxRows || k < 8 || k > kMaxRows || n % 8 != 0 || k % 8 != 0 || ldx % 8 != 0 || ldw % 8 != 0 ||
      lde % 8 != 0 || ldo % 8 != 0 || (elem != kElemBF16 && elem != kElemF16))
    return cudaErrorInvalidValue;
  GroupedArgs g;
  g.offsets = offsets;
  g.out = static_cast<uint16_t*>(out);
  g.ldo = ldo;
  g.rows = rows;
  g.groups = groups;
  g.features = backward ? k : n;
  g.reduction = backward ? n : k;
  g.zero_rest = zero_rest ? 1 : 0;
  g.error_words = error_words;
  const uint64_t w_dims[3] = {static_cast<uint64_t>(k), static_cast<uint64_t>(n), static_cast<uint64_t>(groups)};
  const uint64_t w_strides[2] = {static_cast<uint64_t>(ldw) * 2, static_cast<uint64_t>(lde) * 2};
  const uint32_t w_box[3] = {64, backward ? 64u : 128u, 1};
  const CUtensorMap map_w = make_swizzled_map(w, 2, 3, w_dims, w_strides, w_box);
  const uint64_t x_dims[2] = {static_cast<uint64_t>(g.reduction), static_cast<uint64_t>(rows)};
  const uint64_t x_strides[1] = {static_cast<uint64_t>(ldx) * 2};
  const uint32_t x_box[2] = {64, static_cast<uint32_t>(bn / 2)};
  const uint32_t piece_box[2] = {64, 32};
  const CUtensorMap map_x = make_swizzled_map(x, 2, 2, x_dims, x_strides, x_box);
  const CUtensorMap map_piece = make_swizzled_map(x, 2, 2, x_dims, x_strides, piece_box);
  // as many tiles as there can be: every group may end inside one
  const long long f_tiles = (g.features + 2 * BM - 1) / (2 * BM), active = groups < rows ? groups : rows;
  const long long most = f_tiles * (rows / bn + active);
  if (most > (1ll << 30)) return cudaErrorInvalidValue;
  const int most_tiles = most < 1 ? 1 : static_cast<int>(most);
  const bool bf16 = elem == kElemBF16;
  switch (bn) {
    case 64: return launch_by_type<64>(backward, bf16, map_w, map_x, map_piece, g, most_tiles, stream);
    case 256: return launch_by_type<256>(backward, bf16, map_w, map_x, map_piece, g, most_tiles, stream);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace sm100
}  // namespace msccl
