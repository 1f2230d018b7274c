// Products in 8-bit floating point with fp32 scales per block of 128, for sm_100a, dense or by group:
//
//   d[t, n] = sum over blocks b of K:  sa[t, b] * sb[e, n / 128, b] * (sum over k in b of a[t, k] w[e, n, k])
//
// a, w: e4m3; sa: one scale per row and 128 values; sb: one per 128 x 128 values; d: bf16.
//
// The scales are arbitrary fp32 numbers, so the tensor core cannot apply them (its block scales are powers of two): every block of
// K gets columns of its own in tensor memory (tcgen05.mma kind::f8f6f4, four instructions of K = 32), and eight warps add scale *
// accumulator to fp32 sums in registers while the tensor core goes on.  The lane of an accumulator is a row, so that one number per
// thread and block scales all of its columns.  Tiles are 128 rows x BN columns of one CTA: warps 2 .. 9 take a quarter of the rows
// and half of the columns each.
//
// What bounds it: an exchange between the roles (commit, wait, arrival) costs some hundred clocks whatever it hands over, so two or
// four blocks of K share one (8192 x 4096 x 14336: 625 us with one, 438 with two); the operands of a 128 x 128 tile come from L2 at 19
// TB/s, which alone takes 405 us there.  Tried: 128 x 256 tiles (128 sums a thread spill, and a spilled value comes back from L2:
// 614 us), CTA pairs with 256 x 256 (481: one block per accumulator) and 256 x 128 tiles (438, and 549 against 519 us at 8192 x 14336 x
// 4096).
//
// With at most 32 rows in all only 32 rows of `a` are loaded; the tensor core then reads what follows in the same stage as the
// other rows, and their results are not read.
//
// The two scales of a block are multiplied with each other in fp32, so that product has to be a normal number (as those of
// quantize_block.cu's scales are, unless both operands are near an end of fp32's range).
//
// Every wait is bounded (gemm_sm100.cuh).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "expert_ops.h"
#include "gemm_sm100.cuh"
#include "gemm_sm100.h"
#include "grouped_common.cuh"

namespace msccl {
namespace sm100 {

namespace {

constexpr int kFBlock = 128;                     // K values per scale = bytes per shared-memory row
constexpr int kFGroupTileRows = 2048;            // rows that a group of tiles walks together (L2, see tile_coords)

struct FArgs {
  const int* offsets;                            // nullptr: one group of all rows
  const float *sa, *sb;
  long long sa_row, sa_block;                    // strides of sa
  __nv_bfloat16* out;
  long long ldo;
  int rows, groups, n, k;
  int zero_rest;
  int* error_words;
};

// Two fp32 sums at once: acc += scale * v.
__device__ __forceinline__ void fma2(float2& acc, float2 scale, uint32_t lo, uint32_t hi) {
  unsigned long long a, s, v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(a) : "f"(acc.x), "f"(acc.y));
  asm("mov.b64 %0, {%1, %2};" : "=l"(s) : "f"(scale.x), "f"(scale.y));
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(lo), "r"(hi));
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(a) : "l"(s), "l"(v));
  asm("mov.b64 {%0, %1}, %2;" : "=f"(acc.x), "=f"(acc.y) : "l"(a));
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
// Wait for this thread's tensor-memory loads; the registers pass through (as in wait_loaded).
__device__ __forceinline__ void wait_loaded16(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                 "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :: "memory");
}

// The scales of one row and one 128-column block of the result, U blocks of K at a time: while U are used, the next U are on their way
// from L2, and they are multiplied when their turn comes.  The kernel takes two exchanges' worth at a time: one block ahead, every
// block took as long as a load; one exchange ahead, 128 x 4096 x 14336 took 39 us instead of 31.
template <int U>
struct ScaleStream {
  const float *sa, *sb;
  long long step;
  int left;
  float now[U], a[U], b[U];
  __device__ __forceinline__ ScaleStream(const float* sa_, long long step_, const float* sb_, int blocks, bool active)
      : sa(sa_), sb(sb_), step(step_), left(active ? blocks : 0) {
    fetch();
  }
  __device__ __forceinline__ void fetch() {
    if (left >= U) {
#pragma unroll
      for (int i = 0; i < U; ++i) {
        a[i] = *sa;
        b[i] = sb[i];
        sa += step;
      }
      sb += U;
    } else {
#pragma unroll
      for (int i = 0; i < U; ++i) {
        a[i] = i < left ? *sa : 0.0f;
        b[i] = i < left ? sb[i] : 0.0f;
        if (i + 1 < left) sa += step;
      }
    }
    left -= U;
  }
  __device__ __forceinline__ void advance() {      // before blocks 0, U, 2 U ..: now[0 .. U - 1] are theirs
#pragma unroll
    for (int i = 0; i < U; ++i) now[i] = a[i] * b[i];
    fetch();
  }
};

// Where the scales of column block `column / 128` of group e start.
__device__ __forceinline__ const float* weight_scales(const FArgs& g, int e, int column, int k_blocks) {
  const int n_blocks = (g.n + kFBlock - 1) / kFBlock;
  return g.sb + (static_cast<long long>(e) * n_blocks + min(column / kFBlock, n_blocks - 1)) * k_blocks;
}

template <typename TilesOf>
__device__ __forceinline__ void build_table(GroupTable& table, const FArgs& g, TilesOf tiles_of) {       // whole warp
  if (g.offsets != nullptr) {
    build_groups(table, g.offsets, g.groups, g.rows, tiles_of);
  } else if (threadIdx.x % 32 == 0) {
    table.row_start[0] = table.tile_start[0] = 0;
    table.row_start[1] = g.rows;
    table.tile_start[1] = tiles_of(g.rows);
  }
}

// Rows before the first group and behind the last one become zero; `warp` of `warps` all over the grid.
__device__ __forceinline__ void zero_rest_rows(const GroupTable& table, const FArgs& g, int warp, int warps) {
  const int head = table.row_start[0], tail = table.row_start[g.groups], rest = head + g.rows - tail, lane = threadIdx.x % 32;
  for (int i = warp; i < rest; i += warps) {
    uint4* dst = reinterpret_cast<uint4*>(g.out + static_cast<long long>(i < head ? i : tail + i - head) * g.ldo);
    for (int v = lane; v < g.n / 8; v += 32) dst[v] = make_uint4(0, 0, 0, 0);
  }
}

// The columns [column, column + 2 * PAIRS) of 32 rows, one per lane, as bf16, as far as the result has them (multiples of 8 columns).
// PAIRS / 4 lanes exchange their 16-byte pieces first, so that they store one stretch of a row instead of a piece of one row each.
template <int PAIRS>
__device__ __forceinline__ void store_rows(const FArgs& g, long long row0, int rows, int column, const float2 (&sum)[PAIRS]) {
  constexpr int P = PAIRS / 4;                   // pieces of a row: 2, 4 or 8
  const int lane = threadIdx.x % 32;
  uint4 v[P];
#pragma unroll
  for (int i = 0; i < P; ++i)
    v[i] = make_uint4(pack_bf16(sum[4 * i].x, sum[4 * i].y), pack_bf16(sum[4 * i + 1].x, sum[4 * i + 1].y),
                      pack_bf16(sum[4 * i + 2].x, sum[4 * i + 2].y), pack_bf16(sum[4 * i + 3].x, sum[4 * i + 3].y));
  // transpose P x P pieces among P lanes: afterwards v[i] is piece lane % P of row (lane / P) * P + i
#pragma unroll
  for (int bit = 1; bit < P; bit <<= 1) {
    const bool up = (lane & bit) != 0;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      if (i & bit) continue;
      const uint4 give = up ? v[i] : v[i | bit];
      const uint4 got = make_uint4(__shfl_xor_sync(kFullMask, give.x, bit), __shfl_xor_sync(kFullMask, give.y, bit),
                                   __shfl_xor_sync(kFullMask, give.z, bit), __shfl_xor_sync(kFullMask, give.w, bit));
      if (up) v[i] = got; else v[i | bit] = got;
    }
  }
  const int c = column + lane % P * 8, first = lane / P * P;
  if (c >= g.n) return;
  __nv_bfloat16* out = g.out + (row0 + first) * g.ldo + c;
#pragma unroll
  for (int i = 0; i < P; ++i) {
    if (first + i < rows) *reinterpret_cast<uint4*>(out) = v[i];
    out += g.ldo;
  }
}

constexpr int kFThreads = 320;                   // 0 producer, 1 MMA, 2..9 scaling and epilogue
constexpr int kFEpilogueWarps = 8;
constexpr int kFSmemLimit = 216 * 1024;

// U blocks of K share a stage, an accumulator and every wait: an exchange between the roles costs some hundred clocks whatever it
// hands over, a block of 32 columns is 64 clocks of the tensor core.
template <int BN, int AR> struct FGeometry {
  static constexpr int kU = AR == 32 && BN <= 64 ? 4 : 2;
  static constexpr int kABytes = AR * kFBlock;
  static constexpr int kBBytes = BN * kFBlock;
  static constexpr int kStageBytes = kU * (kABytes + kBBytes);        // kU blocks of a, then kU blocks of w
  static_assert((kU - 1) * kABytes + BM * kFBlock <= kStageBytes, "the MMA reads BM rows of every block of a");
  static constexpr int kFit = kFSmemLimit / kStageBytes;
  static constexpr int kStages = kFit < 8 ? kFit : 8;
  static constexpr int kAccs = 512 / (kU * BN) < 4 ? 512 / (kU * BN) : 4;
  static constexpr int kTmemCols = kAccs * kU * BN;
  static constexpr size_t kSmem = 1024 + static_cast<size_t>(kStages) * kStageBytes + 512;
};

__device__ __forceinline__ void umma_f8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(static_cast<uint32_t>(accumulate))
      : "memory");
}

template <int BN, int AR>
__global__ void __launch_bounds__(kFThreads, 1)
fp8_block_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w, const FArgs g) {
  using Geo = FGeometry<BN, AR>;
  constexpr int S = Geo::kStages, ACCS = Geo::kAccs, U = Geo::kU;
  constexpr int COLS = BN / 2;                   // columns of one epilogue thread
  constexpr int CHUNK = 16;
  extern __shared__ uint8_t smem_raw[];
  __shared__ GroupTable table;
  uint8_t* stage_base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(stage_base + static_cast<size_t>(S) * Geo::kStageBytes);
  uint64_t *full_bar = bars, *empty_bar = bars + S, *acc_full = bars + 2 * S, *acc_empty = bars + 2 * S + ACCS;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * S + 2 * ACCS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int n_tiles = (g.n + BN - 1) / BN;
  const int k_blocks = (g.k + kFBlock - 1) / kFBlock;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < ACCS; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], kFEpilogueWarps);
    }
    // an earlier launch gave up: every role leaves at its first wait
    *abort_flag = g.error_words != nullptr && *reinterpret_cast<volatile int*>(g.error_words) != 0 ? 1 : 0;
    mbar_fence_init();
    prefetch_tensormap(&map_a);
    prefetch_tensormap(&map_w);
  }
  if (warp == 1) tmem_alloc(tmem_slot, Geo::kTmemCols);
  if (warp == 2) build_table(table, g, [&](int rows) { return (rows + BM - 1) / BM * n_tiles; });
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  const bool skip = *abort_flag != 0;
  const int num_tiles = skip ? 0 : table.tile_start[g.groups];
  __syncthreads();                               // nobody raises the flag before everybody has read it

  auto locate = [&](int tile, int& e, int& row, int& column) {
    while (tile >= table.tile_start[e + 1]) ++e;
    const int rows = table.row_start[e + 1] - table.row_start[e];
    int tm, tn;
    tile_coords(tile - table.tile_start[e], (rows + BM - 1) / BM, n_tiles, kFGroupTileRows / BM, tm, tn);
    row = table.row_start[e] + tm * BM;
    column = tn * BN;
  };

  if (warp == 0) {
    if (elect_one()) {
      int stage = 0, e = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = blockIdx.x; tile < num_tiles && ok; tile += gridDim.x) {
        int row, column;
        locate(tile, e, row, column);
        for (int kb = 0; kb < k_blocks; kb += U) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1, abort_flag)) {
            gemm_fail(g.error_words, abort_flag, GEMM_TIMEOUT_EMPTY, 0, stage);
            ok = false;
            break;
          }
          uint8_t* dst = stage_base + static_cast<size_t>(stage) * Geo::kStageBytes;
          const int here = min(U, k_blocks - kb);
          mbar_expect_tx(&full_bar[stage], here * (Geo::kABytes + Geo::kBBytes));
#pragma unroll
          for (int u = 0; u < U; ++u) {
            if (u >= here) break;
            tma_load_2d(dst + u * Geo::kABytes, &map_a, &full_bar[stage], (kb + u) * kFBlock, row);
            tma_load_3d(dst + U * Geo::kABytes + u * Geo::kBBytes, &map_w, &full_bar[stage], (kb + u) * kFBlock, column, e);
          }
          if (++stage == S) { stage = 0; phase ^= 1; }
        }
      }
      if (!ok) drain_wait();
    }
  } else if (warp == 1) {
    if (elect_one()) {
      constexpr uint32_t idesc = (1u << 4) | (static_cast<uint32_t>(BN >> 3) << 17) | (static_cast<uint32_t>(BM >> 4) << 24);   // e4m3 x e4m3 -> fp32
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int tile = blockIdx.x; tile < num_tiles && ok; tile += gridDim.x) {
        for (int kb = 0; kb < k_blocks; kb += U) {
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
          const uint32_t a_addr = smem_u32(stage_base + static_cast<size_t>(stage) * Geo::kStageBytes);
          const uint64_t adesc = smem_desc_sw128(a_addr), bdesc = smem_desc_sw128(a_addr + U * Geo::kABytes);
          const uint32_t tmem_d = tmem_base + static_cast<uint32_t>(acc * U * BN);
          const int here = min(U, k_blocks - kb);
#pragma unroll
          for (int u = 0; u < U; ++u) {
            if (u >= here) break;
#pragma unroll
            for (int k = 0; k < kFBlock / 32; ++k)
              umma_f8(tmem_d + u * BN, adesc + static_cast<uint64_t>(u * (Geo::kABytes / 16) + k * 2),
                      bdesc + static_cast<uint64_t>(u * (Geo::kBBytes / 16) + k * 2), idesc, k != 0);
          }
          tc_commit(&empty_bar[stage]);
          tc_commit(&acc_full[acc]);
          if (++stage == S) { stage = 0; phase ^= 1; }
          if (++acc == ACCS) { acc = 0; acc_phase ^= 1; }
        }
      }
    }
  } else {
    const int quarter = warp % 4, half = (warp - 2) / 4;
    int acc = 0, e = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    for (int tile = blockIdx.x; tile < num_tiles && ok; tile += gridDim.x) {
      int row, column;
      locate(tile, e, row, column);
      const int left = table.row_start[e + 1] - row - quarter * 32;       // rows of this warp that are the group's
      row += quarter * 32 + lane;
      column += half * COLS;
      float2 sum[COLS / 2];
#pragma unroll
      for (int i = 0; i < COLS / 2; ++i) sum[i] = make_float2(0.0f, 0.0f);
      ScaleStream<2 * U> scales(g.sa + min(row, g.rows - 1) * g.sa_row, g.sa_block, weight_scales(g, e, column, k_blocks), k_blocks, left > 0);
      for (int kb0 = 0; kb0 < k_blocks && ok; kb0 += 2 * U) {
        scales.advance();
#pragma unroll
        for (int turn = 0; turn < 2; ++turn) {
          const int kb = kb0 + turn * U;
          if (kb >= k_blocks) break;
          ok = mbar_wait_warp(&acc_full[acc], acc_phase, abort_flag);
          if (!ok) {
            if (lane == 0) gemm_fail(g.error_words, abort_flag, GEMM_TIMEOUT_ACC, 2, acc);
            break;
          }
          tc_fence_after_sync();
          const int here = min(U, k_blocks - kb);
          const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(acc * U * BN + half * COLS);
          auto release = [&] {
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[acc]);
          };
          if (left > 0) {
            // CHUNK columns of a block at a time; the next ones are on their way while these are added, and the accumulator is free
            // again before the last ones are
            constexpr int PER = COLS / CHUNK;
            uint32_t r[2][CHUNK];
            tmem_ld16(taddr, r[0]);
#pragma unroll
            for (int q = 0; q < U * PER; ++q) {
              if (q / PER >= here) break;
              wait_loaded16(r[q % 2]);
              if ((q + 1) % PER != 0 || (q + 1) / PER < here)
                tmem_ld16(taddr + (q + 1) / PER * BN + (q + 1) % PER * CHUNK, r[(q + 1) % 2]);
              else
                release();
              const float2 s2 = make_float2(scales.now[turn * U + q / PER], scales.now[turn * U + q / PER]);
#pragma unroll
              for (int i = 0; i < CHUNK / 2; ++i) fma2(sum[q % PER * (CHUNK / 2) + i], s2, r[q % 2][2 * i], r[q % 2][2 * i + 1]);
            }
          } else {
            release();
          }
          if (++acc == ACCS) { acc = 0; acc_phase ^= 1; }
        }
      }
      if (ok && left > 0) store_rows(g, row - lane, left, column, sum);
    }
    if (g.zero_rest && !skip) zero_rest_rows(table, g, blockIdx.x * kFEpilogueWarps + warp - 2, gridDim.x * kFEpilogueWarps);
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, Geo::kTmemCols);
  }
}

template <int BN, int AR>
cudaError_t launch(const CUtensorMap& map_a, const CUtensorMap& map_w, const FArgs& g, int most_tiles, cudaStream_t stream) {
  auto kernel = fp8_block_kernel<BN, AR>;
  static bool ready[64] = {};
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!ready[dev]) {
    err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(FGeometry<BN, AR>::kSmem));
    if (err != cudaSuccess) return err;
    ready[dev] = true;
  }
  kernel<<<most_tiles < sm_count() ? most_tiles : sm_count(), kFThreads, FGeometry<BN, AR>::kSmem, stream>>>(map_a, map_w, g);
  return cudaGetLastError();
}

}  // namespace

// a: [rows, k] e4m3 (pitch lda bytes), sa: [rows, ceil(k / 128)] with the strides given; w: [groups, n, k] e4m3 (pitch ldw, matrix
// stride lde), sb: [groups, ceil(n / 128), ceil(k / 128)] contiguous; out: [rows, n] bf16.  k % 16 == 0, n % 8 == 0.
// bn: 32, 64 or 128 columns per tile; few_rows: there are at most 32 rows.
cudaError_t launch_fp8_block_gemm(const void* a, long long lda, const float* sa, long long sa_row, long long sa_block, const void* w,
                                  long long ldw, long long lde, const float* sb, const int* offsets, void* out, long long ldo, int rows,
                                  int groups, int n, int k, int bn, bool few_rows, bool zero_rest, int* error_words, cudaStream_t stream) {
  if (rows < 1 || rows > kMaxRows || groups < 1 || groups > kMaxGroups || n < 8 || n > kMaxRows || k < 16 || k > kMaxRows || n % 8 != 0 || k % 16 != 0 || lda % 16 != 0 || ldw % 16 != 0 ||
      lde % 16 != 0 || ldo % 8 != 0 || (offsets == nullptr && groups != 1) || (few_rows && rows > 32))
    return cudaErrorInvalidValue;
  FArgs g;
  g.offsets = offsets;
  g.sa = sa;
  g.sb = sb;
  g.sa_row = sa_row;
  g.sa_block = sa_block;
  g.out = static_cast<__nv_bfloat16*>(out);
  g.ldo = ldo;
  g.rows = rows;
  g.groups = groups;
  g.n = n;
  g.k = k;
  g.zero_rest = zero_rest ? 1 : 0;
  g.error_words = error_words;
  const uint64_t a_dims[2] = {static_cast<uint64_t>(k), static_cast<uint64_t>(rows)}, a_strides[1] = {static_cast<uint64_t>(lda)};
  const uint32_t a_box[2] = {kFBlock, few_rows ? 32u : static_cast<uint32_t>(BM)};
  const CUtensorMap map_a = make_swizzled_map(a, 1, 2, a_dims, a_strides, a_box);
  const uint64_t w_dims[3] = {static_cast<uint64_t>(k), static_cast<uint64_t>(n), static_cast<uint64_t>(groups)};
  const uint64_t w_strides[2] = {static_cast<uint64_t>(ldw), static_cast<uint64_t>(lde)};
  const uint32_t w_box[3] = {kFBlock, static_cast<uint32_t>(bn), 1};
  const CUtensorMap map_w = make_swizzled_map(w, 1, 3, w_dims, w_strides, w_box);
  const long long active = groups < rows ? groups : rows, most = static_cast<long long>((n + bn - 1) / bn) * (rows / BM + active);
  if (most > (1ll << 30)) return cudaErrorInvalidValue;
  const int tiles = static_cast<int>(most);
  switch (bn) {
    case 32: return few_rows ? launch<32, 32>(map_a, map_w, g, tiles, stream) : launch<32, BM>(map_a, map_w, g, tiles, stream);
    case 64: return few_rows ? launch<64, 32>(map_a, map_w, g, tiles, stream) : launch<64, BM>(map_a, map_w, g, tiles, stream);
    case 128: return few_rows ? launch<128, 32>(map_a, map_w, g, tiles, stream) : launch<128, BM>(map_a, map_w, g, tiles, stream);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace sm100
}  // namespace msccl
