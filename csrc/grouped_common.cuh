// Pieces shared by the grouped products (grouped_gemm.cu, grouped_wgrad.cu, fp8_block_gemm.cu): the table of groups, tensor maps of
// two and three dimensions, descriptors of operands whose reduction dimension is not the contiguous one.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "gemm_sm100.cuh"
#include "umma_2cta.cuh"

namespace msccl {
namespace sm100 {

constexpr int kMaxGroups = 512;
constexpr int kMaxRows = 1 << 30;                // also of n and k: index arithmetic of tiles stays in 32 bits
constexpr unsigned int kFullMask = 0xffffffffu;

// Rows of every group and the number of tiles before it.  Offsets come from the device and may be anything: they are clamped to
// [0, rows] and to their running maximum, so that groups never overlap and no index leaves the tensors.
struct GroupTable {
  int row_start[kMaxGroups + 1];
  int tile_start[kMaxGroups + 1];
};

// Whole warp.
__device__ __forceinline__ void build_row_starts(int* row_start, const int* __restrict__ offsets, int groups, int rows) {
  const int lane = threadIdx.x % 32;
  int high = 0;                                  // running maximum
  for (int b = 0; b <= groups; b += 32) {
    int v = b + lane <= groups ? min(max(offsets[b + lane], 0), rows) : 0;
    v = max(v, high);
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int up = __shfl_up_sync(kFullMask, v, off);
      if (lane >= off) v = max(v, up);
    }
    if (b + lane <= groups) row_start[b + lane] = v;
    high = __shfl_sync(kFullMask, v, 31);
  }
  __syncwarp();
}

// Whole warp.  tiles_of(rows) = tiles of a group of that many rows.
template <typename TilesOf>
__device__ __forceinline__ void build_groups(GroupTable& g, const int* __restrict__ offsets, int groups, int rows, TilesOf tiles_of) {
  const int lane = threadIdx.x % 32;
  build_row_starts(g.row_start, offsets, groups, rows);
  int before = 0;
  if (lane == 0) g.tile_start[0] = 0;
  for (int b = 0; b < groups; b += 32) {
    int t = b + lane < groups ? tiles_of(g.row_start[b + lane + 1] - g.row_start[b + lane]) : 0;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int up = __shfl_up_sync(kFullMask, t, off);
      if (lane >= off) t += up;
    }
    if (b + lane < groups) g.tile_start[b + lane + 1] = before + t;
    before += __shfl_sync(kFullMask, t, 31);
  }
  __syncwarp();
}

// Loads of one CTA of a pair whose bytes are counted on the mbarrier at `bar`, which may belong to the partner (no multicast).
__device__ __forceinline__ void tma_pair_2d(void* dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void tma_pair_3d(void* dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
}
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z) : "memory");
}

// Arrival on a barrier of the pair that orders no memory of this thread: an accumulator is free once its loads have returned
// (tcgen05.wait::ld).  The releasing form waits until the thread's stores are visible to the cluster, half a microsecond and more.
__device__ __forceinline__ void mbar_arrive_cluster_relaxed(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// One lane of a converged warp.  Code behind `if (elect_one())` is known to run in one thread: tcgen05.mma then costs 39 clocks to
// issue and a commit about 5, against 54 and 44 behind `if (lane == 0)`.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\tselp.u32 %0, 1, 0, e;\n\t}" : "=r"(p));
  return p != 0;
}

// Wait of a whole warp.  (All lanes poll: one lane that tells the others is later by a shuffle and a branch, which an fp8 block notices.)
__device__ __forceinline__ bool mbar_wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  const bool ok = mbar_wait(bar, parity, abort_flag);
  return __all_sync(kFullMask, ok);
}

// Operand whose M (or N) dimension is the contiguous one, 128-byte swizzle: slabs of 64 elements x 64 reduction rows (8 KB, 128
// bytes per reduction row).  Leading byte offset: from one slab to the next; stride byte offset: 8 reduction rows.
constexpr int kSlabBytes = 64 * 128;
__device__ __forceinline__ uint64_t smem_desc_mn_sw128(uint32_t smem_addr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_addr >> 4) & 0x3FFF);
  d |= static_cast<uint64_t>(kSlabBytes >> 4) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}
// Bits of the instruction descriptor (kind::f16): fp32 accumulator, both operands f16 or both bf16.
constexpr uint32_t kIdescTransA = 1u << 15, kIdescTransB = 1u << 16;
__host__ __device__ constexpr uint32_t idesc_16bit(bool bf16, int m, int n) {
  return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

__device__ __forceinline__ uint32_t pack_16bit(bool bf16, float lo, float hi) {
  uint32_t r;
  if (bf16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Wait for this thread's tensor-memory loads; the registers pass through, so that nothing that uses them moves ahead of the wait.
__device__ __forceinline__ void wait_loaded(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                 "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :: "memory");
  asm volatile("" : "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                 "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :: "memory");
}

// An accumulator chunk with a feature per lane and 32 rows in the registers, as 16-bit values with eight features of one row per
// lane: v[m] = features (lane & ~7) .. + 7 of row 8 m + lane % 8.  Three exchanges among eight lanes, 32 shuffles.  Four lanes then
// store 64 consecutive bytes of a row; storing a register at a time would write 2 bytes per lane.
template <bool BF16>
__device__ __forceinline__ void transpose_chunk(const uint32_t (&r)[32], int lane, uint4 (&v)[4]) {
  uint32_t s[16];                                // a pair of features, row 2 i + bit 0 of the lane
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const uint32_t p = pack_16bit(BF16, __uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
    const uint32_t q = __shfl_xor_sync(kFullMask, p, 1);
    s[i] = (lane & 1) ? __byte_perm(q, p, 0x7632) : __byte_perm(p, q, 0x5410);
  }
  uint2 u[8];                                    // four features, row 4 j + two bits of the lane
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const bool up = (lane & 2) != 0;
    const uint32_t got = __shfl_xor_sync(kFullMask, up ? s[2 * j] : s[2 * j + 1], 2);
    u[j] = up ? make_uint2(got, s[2 * j + 1]) : make_uint2(s[2 * j], got);
  }
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    const bool up = (lane & 4) != 0;
    const uint2 give = up ? u[2 * m] : u[2 * m + 1];
    const uint2 got = make_uint2(__shfl_xor_sync(kFullMask, give.x, 4), __shfl_xor_sync(kFullMask, give.y, 4));
    v[m] = up ? make_uint4(got.x, got.y, u[2 * m + 1].x, u[2 * m + 1].y) : make_uint4(u[2 * m].x, u[2 * m].y, got.x, got.y);
  }
}

// A producer that gave up lets the loads that it issued land before shared memory is released (they take microseconds).
__device__ __forceinline__ void drain_wait() {
  unsigned long long t0, t1;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t0));
  do { asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t1)); } while (t1 - t0 < 200000ull);
}

// Tensor maps (gemm_sm100.cu).  dims and box innermost first; strides in bytes, of dimensions 1 and up.
CUtensorMap make_swizzled_map(const void* base, int elem_bytes, int rank, const uint64_t* dims, const uint64_t* strides, const uint32_t* box);

}  // namespace sm100
}  // namespace msccl
