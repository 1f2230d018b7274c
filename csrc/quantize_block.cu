// Quantisation to e4m3 with one fp32 scale per block: 128 values of a row (activations) or 128 x 128 values (weights).
//
//   scale = max(largest magnitude, 2^-100) / 448,   q = e4m3(x / scale)
//
// Both quotients are correctly rounded fp32 divisions, then one rounding to e4m3 (nearest even): the bytes follow from this
// definition alone.  Infinite values make the scale infinite (the block becomes NaN and zeros), NaN makes the whole block NaN:
// neither can vanish.  The floor keeps the scale of a block of zeros, or of values below 2^-100, a normal number.
//
// A row's 128 bf16 values are 16 lanes x 16 bytes in, 16 lanes x 8 bytes out.  fp32 is bound by memory (8192 x 14336: 99 us, 5.9 TB/s; a
// weight of 8 x 14336 x 4096: 327 us, 7.2 TB/s), 16-bit types by the instructions for each value (93 us, 3.8 TB/s; 327 us, 4.3 TB/s).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "expert_ops.h"

namespace msccl {
namespace sm100 {

namespace {

constexpr int kQThreads = 256;

template <typename T> __device__ __forceinline__ void load8(const T* p, float (&v)[8]);
template <> __device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 r = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
template <> __device__ __forceinline__ void load8<__half>(const __half* p, float (&v)[8]) {
  const uint4 r = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
template <> __device__ __forceinline__ void load8<float>(const float* p, float (&v)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}

// Magnitudes compare as unsigned bit patterns: infinity is above every number and NaN above infinity.
__device__ __forceinline__ uint32_t largest_bits(const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
  return m;
}
__device__ __forceinline__ float block_scale(uint32_t bits) {
  const float floor_value = 0x1p-100f;
  return __fdiv_rn(__uint_as_float(max(bits, __float_as_uint(floor_value))), 448.0f);
}
__device__ __forceinline__ uint2 to_e4m3(const float (&v)[8]) {
  uint32_t p[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) p[i] = __nv_cvt_float2_to_fp8x2(make_float2(v[2 * i], v[2 * i + 1]), __NV_SATFINITE, __NV_E4M3);
  return make_uint2(p[0] | p[1] << 16, p[2] | p[3] << 16);
}
// x / scale, correctly rounded: the quotient from the correctly rounded reciprocal, corrected once by its exact remainder (Markstein,
// "Computation of elementary functions on the IBM RISC System/6000 processor", 1990, theorem on division).  Scales are between
// 2^-109 and 2^120, so the reciprocal is a normal number.  The remainder is a multiple of more than 2^-48 |q| scale and has to be one of
// 2^-149 to be exact; quotients below 2^-11 are zero in e4m3 whatever the last bits are.  So scales below 2^-60 are multiplied by 2^64 first,
// and x with them, which is exact (without that, blocks whose largest magnitude is near 2^-99 had bytes off by one at ties).  In every thread:
// calls of 8192 x 14336 take 95 us instead of 91, with a branch around it 93, or 97 where it is taken.  An infinite
// or NaN scale takes the division itself.  Eight divisions per thread took 123 us for 8192 x 14336.
__device__ __forceinline__ uint2 quantize8(const float (&v)[8], float scale) {
  float q[8];
  if (scale < INFINITY) {
    const float lift = scale < 0x1p-60f ? 0x1p64f : 1.0f, divisor = scale * lift, reciprocal = __frcp_rn(divisor);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = v[i] * lift;
      q[i] = x * reciprocal;
      q[i] = fmaf(fmaf(q[i], divisor, -x), -reciprocal, q[i]);      // the remainder negated: a zero keeps its sign this way
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = __fdiv_rn(v[i], scale);
  }
  return to_e4m3(q);
}

// 16 lanes take one block of one row; threadIdx.x runs along the row (whole blocks), threadIdx.y over rows.  (Blocks numbered through, a
// division of 64-bit numbers per thread, took 123 us for 8192 x 14336 instead of 92; several rows per thread gain nothing.)
template <typename T>
__global__ void __launch_bounds__(kQThreads)
quantize_rows_kernel(const T* __restrict__ x, long long ldx, uint8_t* __restrict__ q, float* __restrict__ scales, int rows, int k,
                     long long s_row, long long s_block) {
  const long long row = static_cast<long long>(blockIdx.x) * blockDim.y + threadIdx.y;
  const int col = (blockIdx.y * blockDim.x + threadIdx.x) * 8, b = col / 128;
  if (row >= rows || b * 128 >= k) return;                          // uniform for those 16 lanes
  const unsigned int mask = 0xffffu << ((threadIdx.y * blockDim.x + threadIdx.x) & 16);
  float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
  if (col < k) load8(x + row * ldx + col, v);
  uint32_t m = largest_bits(v);
#pragma unroll
  for (int off = 8; off > 0; off >>= 1) m = max(m, __shfl_xor_sync(mask, m, off));
  const float scale = block_scale(m);
  if (col < k) *reinterpret_cast<uint2*>(q + row * k + col) = quantize8(v, scale);
  if (threadIdx.x % 16 == 0) scales[row * s_row + b * s_block] = scale;
}

template <typename T>
__global__ void __launch_bounds__(kQThreads)
quantize_blocks_kernel(const T* __restrict__ w, long long ldw, long long lde, uint8_t* __restrict__ q, float* __restrict__ scales, int n, int k) {
  __shared__ uint32_t part[kQThreads / 32];
  const int kb = blockIdx.x, nb = blockIdx.y, e = blockIdx.z;
  const int col = kb * 128 + static_cast<int>(threadIdx.x % 16) * 8, row0 = nb * 128 + static_cast<int>(threadIdx.x / 16);
  float v[8][8];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = row0 + 16 * i;
    if (row < n && col < k) load8(w + e * lde + row * ldw + col, v[i]);
    else
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
    m = max(m, largest_bits(v[i]));
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, off));
  if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kQThreads / 32; ++i) m = max(m, part[i]);
  const float scale = block_scale(m);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = row0 + 16 * i;
    if (row < n && col < k) *reinterpret_cast<uint2*>(q + (static_cast<long long>(e) * n + row) * k + col) = quantize8(v[i], scale);
  }
  if (threadIdx.x == 0) scales[(static_cast<long long>(e) * gridDim.y + nb) * gridDim.x + kb] = scale;
}

}  // namespace

#define MSCCL_BY_ELEM(elem, ...)                                        \
  switch (elem) {                                                       \
    case kElemF32: { using T = float; __VA_ARGS__; break; }             \
    case kElemBF16: { using T = __nv_bfloat16; __VA_ARGS__; break; }    \
    case kElemF16: { using T = __half; __VA_ARGS__; break; }            \
    default: return cudaErrorInvalidValue;                              \
  }

// x: [rows, k] (pitch ldx elements), q: [rows, k] contiguous, scales: [rows, ceil(k / 128)] with the strides given.
// k % 16 == 0, rows 16-byte aligned.
cudaError_t launch_quantize_rows(const void* x, long long ldx, void* q, float* scales, long long s_row, long long s_block, int rows, int k,
                                 int elem, cudaStream_t stream) {
  if (rows < 1 || k < 16 || k % 16 != 0) return cudaErrorInvalidValue;
  const int blocks = (k + 127) / 128, across = blocks < kQThreads / 16 ? blocks : kQThreads / 16;
  const dim3 threads(16 * across, kQThreads / (16 * across));
  const dim3 grid((rows + threads.y - 1) / threads.y, (blocks + across - 1) / across);
  if (grid.y > 65535) return cudaErrorInvalidValue;
  MSCCL_BY_ELEM(elem, (quantize_rows_kernel<T><<<grid, threads, 0, stream>>>(static_cast<const T*>(x), ldx, static_cast<uint8_t*>(q), scales,
                                                                          rows, k, s_row, s_block)));
  return cudaGetLastError();
}

// w: [groups, n, k] (pitch ldw, matrix stride lde), q: the same contiguous, scales: [groups, ceil(n / 128), ceil(k / 128)].
cudaError_t launch_quantize_blocks(const void* w, long long ldw, long long lde, void* q, float* scales, int groups, int n, int k, int elem,
                                   cudaStream_t stream) {
  if (groups < 1 || groups > 65535 || n < 1 || (n + 127) / 128 > 65535 || k < 16 || k % 16 != 0) return cudaErrorInvalidValue;
  const dim3 grid((k + 127) / 128, (n + 127) / 128, groups);
  MSCCL_BY_ELEM(elem, (quantize_blocks_kernel<T><<<grid, kQThreads, 0, stream>>>(static_cast<const T*>(w), ldw, lde, static_cast<uint8_t*>(q),
                                                                              scales, n, k)));
  return cudaGetLastError();
}

}  // namespace sm100
}  // namespace msccl
