// Rows around the experts of a MoE layer on one GPU, forward and backward.
//
//   sort      the copies (token, j) of every token ordered by expert, stable; expert_start[e] .. expert_start[e + 1] are the rows
//             of expert e.  Copies whose expert id is outside [0, experts) are dropped: they come last, behind
//             expert_start[experts].  position[copy] is the row of a copy (the inverse of sorted_copy).
//   scatter   xs[position[t, j]] = x[t]                         (zero in dropped rows)
//   combine   y[t] = sum_j w[t, j] ys[position[t, j]]           (dropped copies contribute nothing and are not read)
//   backward  of scatter: combine with w = 1; of combine: dys[position[t, j]] = w[t, j] dy[t], dw[t, j] = <dy[t], ys[position[t, j]]>.
//
// Positions and the number of kept rows come from the device and may be anything: a row outside [0, tokens * topk) is neither read nor
// written.
//
// All four are memory bound.  One CTA takes one token, so that a row of x (of dy) is read once and written topk times, where a
// CTA per copy would read it topk times; sums over j and over the row stay in fp32 registers and have one fixed order.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "expert_ops.h"

namespace msccl {
namespace sm100 {

namespace {

constexpr int kSortThreads = 1024;             // copies per CTA
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortMaxExperts = 512;
constexpr int kRowsMaxTopk = 8;
constexpr long long kMaxCopies = 1 << 22;
constexpr int kRowThreads = 256;

// Every CTA orders its own 1024 copies.  It needs the expert counts of all copies and of the copies before its own.  Up to 32 CTAs
// count them themselves (n ids from L2) instead of waiting for other CTAs, so that one launch does and nothing has to be cleared; with
// more a launch before this one has written the counts of each CTA's copies to `counts` (131072 copies, 256 experts: 144 us
// without, under 17 with it).  Counts are integers: the order of the shared-memory additions does not show.
constexpr int kSortAlone = 32;

template <typename Id>
__device__ __forceinline__ int bucket_of(const Id* __restrict__ expert_of, int i, int n, int experts) {
  if (i >= n) return -1;
  const Id id = expert_of[i];
  return id >= 0 && id < static_cast<Id>(experts) ? static_cast<int>(id) : experts;
}

template <typename Id>
__global__ void __launch_bounds__(kSortThreads, 1)
count_copies_kernel(const Id* __restrict__ expert_of, int n, int experts, int* __restrict__ counts) {
  __shared__ int here[kSortMaxExperts + 1];
  for (int i = threadIdx.x; i <= experts; i += kSortThreads) here[i] = 0;
  __syncthreads();
  const int e = bucket_of(expert_of, blockIdx.x * kSortThreads + threadIdx.x, n, experts);
  const unsigned int same = __match_any_sync(0xffffffffu, e);
  if (e >= 0 && (same & ((1u << (threadIdx.x % 32)) - 1u)) == 0) atomicAdd(&here[e], __popc(same));
  __syncthreads();
  for (int i = threadIdx.x; i <= experts; i += kSortThreads) counts[static_cast<long long>(blockIdx.x) * (experts + 1) + i] = here[i];
}

template <typename Id>
__global__ void __launch_bounds__(kSortThreads, 1)
sort_copies_kernel(const Id* __restrict__ expert_of, int n, int experts, const int* __restrict__ counts, int* __restrict__ sorted_copy,
                   int* __restrict__ expert_start, int* __restrict__ position) {
  __shared__ int total[kSortMaxExperts + 1], before[kSortMaxExperts + 1], start[kSortMaxExperts + 2];
  __shared__ unsigned short in_warp[kSortWarps][kSortMaxExperts + 1];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int buckets = experts + 1;             // the last one: dropped copies
  for (int i = threadIdx.x; i < buckets; i += kSortThreads) total[i] = before[i] = 0;
  for (int i = threadIdx.x; i < kSortWarps * (kSortMaxExperts + 1); i += kSortThreads) (&in_warp[0][0])[i] = 0;
  __syncthreads();
  const int own = blockIdx.x * kSortThreads;
  int my_bucket = -1;
  unsigned int my_rank = 0;
  if (counts != nullptr) {
    my_bucket = bucket_of(expert_of, own + static_cast<int>(threadIdx.x), n, experts);
    const unsigned int same = __match_any_sync(0xffffffffu, my_bucket);
    my_rank = __popc(same & ((1u << lane) - 1u));
    if (my_bucket >= 0 && my_rank == 0) in_warp[warp][my_bucket] = static_cast<unsigned short>(__popc(same));
    // two threads for each bucket: CTAs before this one, and the others
    for (int i = threadIdx.x; i < 2 * buckets; i += kSortThreads) {
      const int e = i % buckets, lo = i < buckets ? 0 : blockIdx.x, hi = i < buckets ? blockIdx.x : gridDim.x;
      int sum = 0;
#pragma unroll 8
      for (int c = lo; c < hi; ++c) sum += counts[static_cast<long long>(c) * buckets + e];
      if (i < buckets) before[e] = sum;
      atomicAdd(&total[e], sum);
    }
  } else {
    for (int base = 0; base < n; base += kSortThreads) {
      const int e = bucket_of(expert_of, base + static_cast<int>(threadIdx.x), n, experts);
      const unsigned int same = __match_any_sync(0xffffffffu, e);
      const unsigned int rank = __popc(same & ((1u << lane) - 1u));
      if (e >= 0 && rank == 0) {
        atomicAdd(&total[e], __popc(same));
        if (base < own) atomicAdd(&before[e], __popc(same));
        if (base == own) in_warp[warp][e] = static_cast<unsigned short>(__popc(same));
      }
      if (base == own) { my_bucket = e; my_rank = rank; }
    }
  }
  __syncthreads();
  if (warp == 0) {                             // exclusive prefix of the totals
    int run = 0;
    for (int b0 = 0; b0 < buckets; b0 += 32) {
      const int v = b0 + lane < buckets ? total[b0 + lane] : 0;
      int incl = v;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, incl, off);
        if (lane >= off) incl += up;
      }
      if (b0 + lane < buckets) start[b0 + lane] = run + incl - v;
      run += __shfl_sync(0xffffffffu, incl, 31);
    }
  } else if (threadIdx.x - 32 < buckets) {     // exclusive prefix over this CTA's warps, per bucket
    const int e = threadIdx.x - 32;
    int run = 0;
    for (int w = 0; w < kSortWarps; ++w) {
      const int c = in_warp[w][e];
      in_warp[w][e] = static_cast<unsigned short>(run);
      run += c;
    }
  }
  __syncthreads();
  if (blockIdx.x == 0)
    for (int e = threadIdx.x; e <= experts; e += kSortThreads) expert_start[e] = start[e];
  if (my_bucket >= 0) {
    const int copy = own + threadIdx.x;
    const int row = start[my_bucket] + before[my_bucket] + in_warp[warp][my_bucket] + static_cast<int>(my_rank);
    sorted_copy[row] = copy;
    position[copy] = row;
  }
}

// 16 bytes of a row as fp32 values and back (one rounding to nearest even).
template <typename T> struct Pack;
template <> struct Pack<float> {
  static constexpr int kN = 4;
  static __device__ __forceinline__ void load(uint4 v, float (&f)[4]) {
    f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ uint4 store(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};
template <> struct Pack<__nv_bfloat16> {
  static constexpr int kN = 8;
  static __device__ __forceinline__ void load(uint4 v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint4 store(const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 p = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&p);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <> struct Pack<__half> {
  static constexpr int kN = 8;
  static __device__ __forceinline__ void load(uint4 v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = p.x;
      f[2 * i + 1] = p.y;
    }
  }
  static __device__ __forceinline__ uint4 store(const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 p = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&p);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// CTAs per SM that the row kernels leave room for: left to itself the compiler keeps more addresses in registers (16384 tokens x 2 copies of
// 4096 bf16: scatter 70 us at 40 registers, 64 at 32; 4096 x 8: combine 47 at 79, 46 at 64, backward 98 at 90, 89 at 80).
constexpr int kScatterCtas = 8;
constexpr int combine_ctas(int k) { return k == 8 ? 4 : 6; }
constexpr int combine_backward_ctas(int k) { return k == 8 ? 3 : k == 1 ? 6 : 4; }

// The row of copy j of this CTA's token, or -1.
__device__ __forceinline__ int row_of(const int* __restrict__ position, int topk, int j) {
  if (j >= topk) return -1;
  const int row = position[static_cast<long long>(blockIdx.x) * topk + j];
  return static_cast<unsigned int>(row) < gridDim.x * static_cast<unsigned int>(topk) ? row : -1;
}

template <typename T>
__global__ void __launch_bounds__(kRowThreads, kScatterCtas)
scatter_rows_kernel(const T* __restrict__ x, long long ldx, T* __restrict__ out, const int* __restrict__ position,
                    const int* __restrict__ rows_kept, int topk, int hidden) {
  const long long t = blockIdx.x;
  const int kept = *rows_kept, vecs = hidden / Pack<T>::kN;
  int rows[kRowsMaxTopk];
#pragma unroll
  for (int j = 0; j < kRowsMaxTopk; ++j) rows[j] = row_of(position, topk, j);
  const uint4* src = reinterpret_cast<const uint4*>(x + t * ldx);
  for (int v = threadIdx.x; v < vecs; v += blockDim.x) {
    const uint4 val = src[v];
#pragma unroll
    for (int j = 0; j < kRowsMaxTopk; ++j)
      if (rows[j] >= 0)
        reinterpret_cast<uint4*>(out + static_cast<long long>(rows[j]) * hidden)[v] = rows[j] < kept ? val : make_uint4(0, 0, 0, 0);
  }
}

// K >= topk copies and V vectors of a row per thread and step, K * V loads in flight (one vector of a token with two copies kept HBM at
// 4.0 TB/s).
template <typename T, int K, bool WEIGHTED>
__global__ void __launch_bounds__(kRowThreads, combine_ctas(K))
combine_rows_kernel(const T* __restrict__ ys, long long ldy, const float* __restrict__ weights, T* __restrict__ out,
                    const int* __restrict__ position, const int* __restrict__ rows_kept, int topk, int hidden) {
  constexpr int N = Pack<T>::kN, V = K <= 2 ? 4 / K : 1;
  const long long t = blockIdx.x;
  const int kept = *rows_kept, vecs = hidden / N;
  int rows[K];
  float w[K];
#pragma unroll
  for (int j = 0; j < K; ++j) {
    rows[j] = row_of(position, topk, j);
    if (rows[j] >= kept) rows[j] = -1;
    w[j] = WEIGHTED && j < topk ? weights[t * topk + j] : 1.0f;
  }
  for (int v0 = threadIdx.x; v0 < vecs; v0 += V * blockDim.x) {
    uint4 val[V][K];
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int j = 0; j < K; ++j)
        if (rows[j] >= 0 && v0 + i * blockDim.x < vecs)
          val[i][j] = reinterpret_cast<const uint4*>(ys + static_cast<long long>(rows[j]) * ldy)[v0 + i * blockDim.x];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (v0 + i * blockDim.x >= vecs) break;
      float sum[N];
#pragma unroll
      for (int c = 0; c < N; ++c) sum[c] = 0.0f;
#pragma unroll
      for (int j = 0; j < K; ++j)
        if (rows[j] >= 0) {
          float f[N];
          Pack<T>::load(val[i][j], f);
#pragma unroll
          for (int c = 0; c < N; ++c) sum[c] = WEIGHTED ? fmaf(w[j], f[c], sum[c]) : sum[c] + f[c];
        }
      reinterpret_cast<uint4*>(out + t * hidden)[v0 + i * blockDim.x] = Pack<T>::store(sum);
    }
  }
}

template <typename T, int K>
__global__ void __launch_bounds__(kRowThreads, combine_backward_ctas(K))
combine_backward_kernel(const T* __restrict__ dy, long long lddy, const T* __restrict__ ys, long long ldy, const float* __restrict__ weights,
                        T* __restrict__ dys, float* __restrict__ dweights, const int* __restrict__ position,
                        const int* __restrict__ rows_kept, int topk, int hidden) {
  constexpr int N = Pack<T>::kN, V = K <= 2 ? 2 : 1;
  __shared__ float partial[kRowThreads / 32][K];
  const long long t = blockIdx.x;
  const int kept = *rows_kept, vecs = hidden / N;
  int rows[K];
  float w[K], dot[K];
#pragma unroll
  for (int j = 0; j < K; ++j) {
    rows[j] = row_of(position, topk, j);
    w[j] = j < topk ? weights[t * topk + j] : 0.0f;
    dot[j] = 0.0f;
  }
  const uint4* src = reinterpret_cast<const uint4*>(dy + t * lddy);
  for (int v0 = threadIdx.x; v0 < vecs; v0 += V * blockDim.x) {
    uint4 gv[V], val[V][K];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int v = v0 + i * blockDim.x;
      if (v >= vecs) break;
      gv[i] = src[v];
#pragma unroll
      for (int j = 0; j < K; ++j)
        if (rows[j] >= 0 && rows[j] < kept && dweights != nullptr) val[i][j] = reinterpret_cast<const uint4*>(ys + static_cast<long long>(rows[j]) * ldy)[v];
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int v = v0 + i * blockDim.x;
      if (v >= vecs) break;
      float g[N];
      Pack<T>::load(gv[i], g);
#pragma unroll
      for (int j = 0; j < K; ++j) {
        if (rows[j] < 0) continue;
        float f[N];
        if (rows[j] < kept) {
          if (dweights != nullptr) {
            Pack<T>::load(val[i][j], f);
#pragma unroll
            for (int c = 0; c < N; ++c) dot[j] = fmaf(f[c], g[c], dot[j]);
          }
#pragma unroll
          for (int c = 0; c < N; ++c) f[c] = w[j] * g[c];
        } else {
#pragma unroll
          for (int c = 0; c < N; ++c) f[c] = 0.0f;
        }
        if (dys != nullptr) reinterpret_cast<uint4*>(dys + static_cast<long long>(rows[j]) * hidden)[v] = Pack<T>::store(f);
      }
    }
  }
  if (dweights == nullptr) return;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
#pragma unroll
  for (int j = 0; j < K; ++j) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], off);
    if (lane == 0) partial[warp][j] = dot[j];
  }
  __syncthreads();
  if (threadIdx.x < topk) {
    float sum = 0.0f;
    for (int i = 0; i < blockDim.x / 32; ++i) sum += partial[i][threadIdx.x];
    dweights[t * topk + threadIdx.x] = sum;
  }
}

bool rows_ok(int tokens, int topk, int hidden, int elem) {
  const int n = elem == kElemF32 ? 4 : 8;
  return tokens >= 1 && topk >= 1 && topk <= kRowsMaxTopk && static_cast<long long>(tokens) * topk <= kMaxCopies && hidden >= n && hidden % n == 0;
}

// One thread per 16 bytes of a row, whole warps, at most kRowThreads.
int row_threads(int hidden, int elem) {
  const int vecs = hidden / (elem == kElemF32 ? 4 : 8);
  const int t = (vecs + 31) / 32 * 32;
  return t < kRowThreads ? t : kRowThreads;
}

}  // namespace

// Integers of workspace that launch_sort_copies needs.
long long sort_copies_workspace(long long n, int experts) {
  const long long ctas = (n + kSortThreads - 1) / kSortThreads;
  return ctas > kSortAlone ? ctas * (experts + 1) : 0;
}

// expert_of: n ids (int32, or int64 with wide_ids).
cudaError_t launch_sort_copies(const void* expert_of, bool wide_ids, long long n, int experts, int* sorted_copy, int* expert_start,
                               int* position, int* workspace, cudaStream_t stream) {
  if (n < 1 || n > kMaxCopies || experts < 1 || experts > kSortMaxExperts) return cudaErrorInvalidValue;
  const int grid = static_cast<int>((n + kSortThreads - 1) / kSortThreads), count = static_cast<int>(n);
  int* counts = sort_copies_workspace(n, experts) > 0 ? workspace : nullptr;
  auto run = [&](auto* ids) {
    using Id = std::remove_const_t<std::remove_pointer_t<decltype(ids)>>;
    if (counts != nullptr) count_copies_kernel<Id><<<grid, kSortThreads, 0, stream>>>(ids, count, experts, counts);
    sort_copies_kernel<Id><<<grid, kSortThreads, 0, stream>>>(ids, count, experts, counts, sorted_copy, expert_start, position);
  };
  if (wide_ids) run(static_cast<const long long*>(expert_of));
  else run(static_cast<const int*>(expert_of));
  return cudaGetLastError();
}

#define MSCCL_BY_ELEM(elem, ...)                                        \
  switch (elem) {                                                       \
    case kElemF32: { using T = float; __VA_ARGS__; break; }             \
    case kElemBF16: { using T = __nv_bfloat16; __VA_ARGS__; break; }    \
    case kElemF16: { using T = __half; __VA_ARGS__; break; }            \
    default: return cudaErrorInvalidValue;                              \
  }

#define MSCCL_BY_COPIES(topk, ...)                                      \
  if (topk == 1) { constexpr int K = 1; __VA_ARGS__; }                  \
  else if (topk == 2) { constexpr int K = 2; __VA_ARGS__; }             \
  else if (topk <= 4) { constexpr int K = 4; __VA_ARGS__; }             \
  else { constexpr int K = 8; __VA_ARGS__; }

cudaError_t launch_scatter_rows(const void* x, long long ldx, void* out, const int* position, const int* rows_kept, int tokens, int topk,
                                int hidden, int elem, cudaStream_t stream) {
  if (!rows_ok(tokens, topk, hidden, elem)) return cudaErrorInvalidValue;
  MSCCL_BY_ELEM(elem, (scatter_rows_kernel<T><<<tokens, row_threads(hidden, elem), 0, stream>>>(
                          static_cast<const T*>(x), ldx, static_cast<T*>(out), position, rows_kept, topk, hidden)));
  return cudaGetLastError();
}

// weights == nullptr: plain sum (the gradient of scatter).
cudaError_t launch_combine_rows(const void* ys, long long ldy, const float* weights, void* out, const int* position, const int* rows_kept,
                                int tokens, int topk, int hidden, int elem, cudaStream_t stream) {
  if (!rows_ok(tokens, topk, hidden, elem)) return cudaErrorInvalidValue;
  const int threads = row_threads(hidden, elem);
  MSCCL_BY_ELEM(elem, MSCCL_BY_COPIES(topk, {
    auto kernel = weights != nullptr ? combine_rows_kernel<T, K, true> : combine_rows_kernel<T, K, false>;
    kernel<<<tokens, threads, 0, stream>>>(static_cast<const T*>(ys), ldy, weights, static_cast<T*>(out), position, rows_kept, topk, hidden);
  }));
  return cudaGetLastError();
}

// dys or dweights may be nullptr when only the other is asked for.
cudaError_t launch_combine_backward(const void* dy, long long lddy, const void* ys, long long ldy, const float* weights, void* dys,
                                    float* dweights, const int* position, const int* rows_kept, int tokens, int topk, int hidden,
                                    int elem, cudaStream_t stream) {
  if (!rows_ok(tokens, topk, hidden, elem)) return cudaErrorInvalidValue;
  MSCCL_BY_ELEM(elem, MSCCL_BY_COPIES(topk, (combine_backward_kernel<T, K><<<tokens, row_threads(hidden, elem), 0, stream>>>(
                                               static_cast<const T*>(dy), lddy, static_cast<const T*>(ys), ldy, weights, static_cast<T*>(dys),
                                               dweights, position, rows_kept, topk, hidden))));
  return cudaGetLastError();
}

}  // namespace sm100
}  // namespace msccl
