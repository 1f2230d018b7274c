// Global norm of a list of gradients and their clipping, in two launches:
//
//   norm    every CTA adds the squares of its chunks and writes one partial sum;
//   scale   every CTA adds the partial sums (in the same order), forms min(1, max_norm / (norm + 1e-6)) and, unless that is 1
//           and the result stays in place, multiplies its chunks by it.  CTA 0 writes the norm.
//
// No atomics and no counters: which CTA takes which chunk is a function of the sizes, so results are the same bits on every
// call, and the only workspace is the partial sums.  With many tensors the list travels in the kernel arguments (32 bytes each),
// so nothing is copied to the device before the launch and a captured graph holds its own list.
//
// Squares are added in fp32 over the 4 or 8 elements of one 16-byte load and in fp64 from there: one conversion per load, and
// a sum of 2^30 elements loses nothing.  A group whose fp32 sum leaves [2^-80, 2^120] (tiny, huge, infinite or NaN values; a group
// of zeros too) is added again in fp64, where no square of an fp32 number over- or underflows.
//
// Both launches are bound by HBM.  (Walking the chunks backwards in the second, for what the norm left in L2, gains nothing.)
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "expert_ops.h"
#include "gemm_sm100.h"

namespace msccl {
namespace sm100 {

namespace {

constexpr int kGradThreads = 256;
// CTAs per SM.  256 Mi bf16 elements: the norm takes 99 us with 8 and 85 (6.3 TB/s) with 6, scaling into fp32 270 us (6.0 TB/s) with 8
// and 285 with 6.
constexpr int kNormCtas = 6, kScaleCtas = 8;
constexpr int kGradMaxCtas = 2048;
constexpr int kChunk = 16384;                   // elements
constexpr int kFewTensors = 100;                // this list fits the 4 KB of arguments that every launch may carry

template <int MAX>
struct GradList {
  int count, chunks;
  GradTensor t[MAX];
};

template <int MAX>
__device__ __forceinline__ int find_tensor(const GradList<MAX>& list, int chunk) {
  int lo = 0, hi = list.count - 1;              // the last tensor whose first chunk is not behind `chunk`
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (list.t[mid].first_chunk <= chunk) lo = mid; else hi = mid - 1;
  }
  return lo;
}

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
  T v[N];
};

template <typename T, int N>
__device__ __forceinline__ double squares(const Vec<T, N>& x) {
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float f = to_f32(x.v[i]);
    s = fmaf(f, f, s);
  }
  if (s > 0x1p-80f && s < 0x1p120f) return s;
  double d = 0.0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const double f = to_f32(x.v[i]);
    d = fma(f, f, d);
  }
  return d;
}

// Elements [0, n) from `p`, any alignment of an element: single elements up to a 16-byte boundary, 16 bytes a load, the rest.
template <typename T>
__device__ __forceinline__ double chunk_squares(const T* p, int n) {
  constexpr int N = 16 / sizeof(T), U = 4;
  const int head = min(n, static_cast<int>((16 - reinterpret_cast<uintptr_t>(p) % 16) % 16 / sizeof(T)));
  const int vecs = (n - head) / N;
  double sum = 0.0;
  if (threadIdx.x < head) sum += squares(Vec<T, 1>{p[threadIdx.x]});
  const Vec<T, N>* body = reinterpret_cast<const Vec<T, N>*>(p + head);
  int i = threadIdx.x;
  for (; i + (U - 1) * kGradThreads < vecs; i += U * kGradThreads) {
    Vec<T, N> x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = body[i + u * kGradThreads];
#pragma unroll
    for (int u = 0; u < U; ++u) sum += squares(x[u]);
  }
  for (; i < vecs; i += kGradThreads) sum += squares(body[i]);
  const int tail = head + vecs * N + threadIdx.x;
  if (tail < n) sum += squares(Vec<T, 1>{p[tail]});
  return sum;
}

__device__ __forceinline__ double block_sum(double v) {      // the same in every thread
  __shared__ double part[kGradThreads / 32];
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int w = 0; w < kGradThreads / 32; ++w) s += part[w];
  return s;
}

template <int MAX>
__global__ void __launch_bounds__(kGradThreads)
grad_norm_kernel(const __grid_constant__ GradList<MAX> list, double* __restrict__ partials) {
  double sum = 0.0;
  for (int c = blockIdx.x; c < list.chunks; c += gridDim.x) {
    const GradTensor& t = list.t[find_tensor(list, c)];
    const long long lo = static_cast<long long>(c - t.first_chunk) * kChunk;
    const int n = static_cast<int>(min(static_cast<long long>(kChunk), t.numel - lo));
    if (t.src_type == kElemF32) sum += chunk_squares(static_cast<const float*>(t.src) + lo, n);
    else if (t.src_type == kElemBF16) sum += chunk_squares(static_cast<const __nv_bfloat16*>(t.src) + lo, n);
    else sum += chunk_squares(static_cast<const __half*>(t.src) + lo, n);
  }
  sum = block_sum(sum);
  if (threadIdx.x == 0) partials[blockIdx.x] = sum;
}

__device__ __forceinline__ double sum_partials(const double* __restrict__ partials, int count) {
  double v = 0.0;
  for (int i = threadIdx.x; i < count; i += kGradThreads) v += partials[i];
  return block_sum(v);
}

__global__ void __launch_bounds__(kGradThreads) grad_sum_kernel(const double* __restrict__ partials, int count, double* sum, float* norm) {
  const double s = sum_partials(partials, count);
  if (threadIdx.x == 0) {
    if (sum != nullptr) *sum = s;
    if (norm != nullptr) *norm = static_cast<float>(sqrt(s));
  }
}

// A factor below 2^-126 (gradients of 1e37) has few bits or none in fp32 although its products may be ordinary numbers.  So it
// comes in two parts: a power of two and the rest.  The first is 1 for all others, and where it is not, what a multiplication by it
// may round is far below the least product that fp32 holds.
struct Factor {
  float power, rest;
  __device__ __forceinline__ explicit Factor(double ratio) {
    power = ratio >= 0x1p-126 || !(ratio > 0.0) ? 1.0f : ratio >= 0x1p-190 ? 0x1p-64f : 0x1p-126f;
    rest = ratio > 1.0 ? 1.0f : static_cast<float>(ratio / power);            // a NaN stays one
  }
  __device__ __forceinline__ float operator*(float v) const { return v * power * rest; }
};

template <typename S, typename D>
__device__ __forceinline__ void chunk_scale(const S* src, D* dst, int n, Factor factor) {
  // The wider of the two types moves 16 bytes per lane, so that every access of a warp is one stretch of memory (8 elements a lane
  // would write fp32 as two halves of a 32-byte sector at different times: 256 Mi bf16 -> fp32 356 us, now 270).  Element by
  // element where the two sides cannot be aligned together.
  constexpr int N = 16 / (sizeof(S) > sizeof(D) ? sizeof(S) : sizeof(D)), U = 8;
  constexpr uintptr_t as = sizeof(S) * N, ad = sizeof(D) * N;
  int head = static_cast<int>((as - reinterpret_cast<uintptr_t>(src) % as) % as / sizeof(S));
  if (reinterpret_cast<uintptr_t>(dst + head) % ad != 0) head = n;
  head = min(head, n);
  for (int i = threadIdx.x; i < head; i += kGradThreads) dst[i] = from_f32<D>(factor * to_f32(src[i]));
  const int vecs = (n - head) / N;
  const Vec<S, N>* sv = reinterpret_cast<const Vec<S, N>*>(src + head);
  Vec<D, N>* dv = reinterpret_cast<Vec<D, N>*>(dst + head);
  int i = threadIdx.x;
  for (; i + (U - 1) * kGradThreads < vecs; i += U * kGradThreads) {
    Vec<S, N> x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = sv[i + u * kGradThreads];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      Vec<D, N> y;
#pragma unroll
      for (int e = 0; e < N; ++e) y.v[e] = from_f32<D>(factor * to_f32(x[u].v[e]));
      dv[i + u * kGradThreads] = y;
    }
  }
  for (; i < vecs; i += kGradThreads) {
    const Vec<S, N> x = sv[i];
    Vec<D, N> y;
#pragma unroll
    for (int e = 0; e < N; ++e) y.v[e] = from_f32<D>(factor * to_f32(x.v[e]));
    dv[i] = y;
  }
  for (int t = head + vecs * N + threadIdx.x; t < n; t += kGradThreads) dst[t] = from_f32<D>(factor * to_f32(src[t]));
}

template <typename S>
__device__ __forceinline__ void chunk_scale_to(const GradTensor& t, long long lo, int n, Factor factor) {
  const S* src = static_cast<const S*>(t.src) + lo;
  if (t.dst_type == kElemF32) chunk_scale(src, static_cast<float*>(t.dst) + lo, n, factor);
  else if (t.dst_type == kElemBF16) chunk_scale(src, static_cast<__nv_bfloat16*>(t.dst) + lo, n, factor);
  else chunk_scale(src, static_cast<__half*>(t.dst) + lo, n, factor);
}

template <int MAX>
__global__ void __launch_bounds__(kGradThreads, 5)           // at most 48 registers: with 50 (four CTAs) those 275 us are 287
grad_scale_kernel(const __grid_constant__ GradList<MAX> list, const double* __restrict__ partials, int partial_count, double max_norm,
                  float* __restrict__ norm_out) {
  const double norm = sqrt(sum_partials(partials, partial_count));
  if (blockIdx.x == 0 && threadIdx.x == 0 && norm_out != nullptr) *norm_out = static_cast<float>(norm);
  const Factor factor(max_norm / (norm + 1e-6));
  for (int c = blockIdx.x; c < list.chunks; c += gridDim.x) {
    const GradTensor& t = list.t[find_tensor(list, c)];
    if (factor.rest == 1.0f && factor.power == 1.0f && t.src == t.dst) continue;
    const long long lo = static_cast<long long>(c - t.first_chunk) * kChunk;
    const int n = static_cast<int>(min(static_cast<long long>(kChunk), t.numel - lo));
    if (t.src_type == kElemF32) chunk_scale_to<float>(t, lo, n, factor);
    else if (t.src_type == kElemBF16) chunk_scale_to<__nv_bfloat16>(t, lo, n, factor);
    else chunk_scale_to<__half>(t, lo, n, factor);
  }
}

template <int MAX>
GradList<MAX> make_list(const GradTensor* tensors, int count) {
  GradList<MAX> list;
  list.count = count;
  int chunks = 0;
  for (int i = 0; i < count; ++i) {
    list.t[i] = tensors[i];
    list.t[i].first_chunk = chunks;
    chunks += static_cast<int>((tensors[i].numel + kChunk - 1) / kChunk);
  }
  list.chunks = chunks;
  return list;
}

bool list_ok(const GradTensor* tensors, int count) {
  if (count < 1 || count > kGradTensorsPerLaunch) return false;
  long long chunks = 0;
  for (int i = 0; i < count; ++i) {
    if (tensors[i].numel < 1 || tensors[i].src_type < 0 || tensors[i].src_type > kElemF16) return false;
    chunks += (tensors[i].numel + kChunk - 1) / kChunk;
  }
  return chunks < (1ll << 30);
}

int grad_grid(const GradTensor* tensors, int count, int per_sm) {
  long long chunks = 0;
  for (int i = 0; i < count; ++i) chunks += (tensors[i].numel + kChunk - 1) / kChunk;
  long long g = sm_count() * per_sm;
  if (g > kGradMaxCtas) g = kGradMaxCtas;
  return static_cast<int>(g < chunks ? g : chunks);
}

}  // namespace

// Partial sums that a launch for this list writes: one for each of its CTAs.
int grad_norm_partials(const GradTensor* tensors, int count) { return list_ok(tensors, count) ? grad_grid(tensors, count, kNormCtas) : 0; }

cudaError_t launch_grad_norm(const GradTensor* tensors, int count, double* partials, cudaStream_t stream) {
  if (!list_ok(tensors, count)) return cudaErrorInvalidValue;
  const int grid = grad_grid(tensors, count, kNormCtas);
  if (count <= kFewTensors) grad_norm_kernel<kFewTensors><<<grid, kGradThreads, 0, stream>>>(make_list<kFewTensors>(tensors, count), partials);
  else grad_norm_kernel<kGradTensorsPerLaunch><<<grid, kGradThreads, 0, stream>>>(make_list<kGradTensorsPerLaunch>(tensors, count), partials);
  return cudaGetLastError();
}

cudaError_t launch_grad_sum(const double* partials, int count, double* sum, float* norm, cudaStream_t stream) {
  if (count < 1) return cudaErrorInvalidValue;
  grad_sum_kernel<<<1, kGradThreads, 0, stream>>>(partials, count, sum, norm);
  return cudaGetLastError();
}

cudaError_t launch_grad_scale(const GradTensor* tensors, int count, const double* partials, int partial_count, double max_norm, float* norm,
                              cudaStream_t stream) {
  if (!list_ok(tensors, count) || partial_count < 1) return cudaErrorInvalidValue;
  const int grid = grad_grid(tensors, count, kScaleCtas);
  if (count <= kFewTensors)
    grad_scale_kernel<kFewTensors><<<grid, kGradThreads, 0, stream>>>(make_list<kFewTensors>(tensors, count), partials, partial_count,
                                                                           max_norm, norm);
  else
    grad_scale_kernel<kGradTensorsPerLaunch><<<grid, kGradThreads, 0, stream>>>(make_list<kGradTensorsPerLaunch>(tensors, count), partials,
                                                                                     partial_count, max_norm, norm);
  return cudaGetLastError();
}

}  // namespace sm100
}  // namespace msccl
