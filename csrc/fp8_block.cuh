// Pieces shared by the kernels of block-scaled fp8 products with fp32 scales (fp8_block_gemm.cu, fp8_block_2cta.cu).
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "gemm_sm100.cuh"
#include "grouped_common.cuh"

namespace msccl {
namespace sm100 {

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

// The scales of one row and one 128-column block of the result, U blocks of K at a time: while U are used, the next U are on their way
// from L2, and they are multiplied when their turn comes.  (One block ahead, every block took as long as a load.)
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
#pragma unroll
    for (int i = 0; i < U; ++i) {
      a[i] = i < left ? sa[i * step] : 0.0f;
      b[i] = i < left ? sb[i] : 0.0f;
    }
    sa += U * step;
    sb += U;
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

// One row's columns [column, column + 2 * PAIRS) as bf16, as far as the result has them (multiples of 8).
template <int PAIRS>
__device__ __forceinline__ void store_row(const FArgs& g, long long row, int column, const float2 (&sum)[PAIRS]) {
  __nv_bfloat16* out = g.out + row * g.ldo + column;
#pragma unroll
  for (int c = 0; c < PAIRS; c += 4)
    if (column + 2 * c < g.n)
      *reinterpret_cast<uint4*>(out + 2 * c) = make_uint4(pack_bf16(sum[c].x, sum[c].y), pack_bf16(sum[c + 1].x, sum[c + 1].y),
                                                          pack_bf16(sum[c + 2].x, sum[c + 2].y), pack_bf16(sum[c + 3].x, sum[c + 3].y));
}

cudaError_t launch_fp8_block_pairs(const CUtensorMap& map_a, const CUtensorMap& map_w, const FArgs& g, int most_tiles, cudaStream_t stream);

}  // namespace sm100
}  // namespace msccl
