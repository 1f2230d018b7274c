// Host API of the operators of an expert layer: row exchange (moe_rows.cu), grouped products
// (grouped_gemm.cu, grouped_wgrad.cu), block-scaled fp8 (fp8_block_gemm.cu, quantize_block.cu), gradient norm (grad_norm.cu).
#pragma once
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace msccl {
namespace sm100 {

// Element types of the operators: the numbers the Python side passes.
enum ElemType : int { kElemF32 = 0, kElemBF16 = 1, kElemF16 = 2 };

// ---- rows around the experts
cudaError_t launch_sort_copies(const void* expert_of, bool wide_ids, long long n, int experts, int* sorted_copy, int* expert_start,
                               int* position, int* workspace, cudaStream_t stream);
long long sort_copies_workspace(long long n, int experts);
cudaError_t launch_scatter_rows(const void* x, long long ldx, void* out, const int* position, const int* rows_kept, int tokens, int topk,
                                int hidden, int elem, cudaStream_t stream);
cudaError_t launch_combine_rows(const void* ys, long long ldy, const float* weights, void* out, const int* position, const int* rows_kept,
                                int tokens, int topk, int hidden, int elem, cudaStream_t stream);
cudaError_t launch_combine_backward(const void* dy, long long lddy, const void* ys, long long ldy, const float* weights, void* dys,
                                    float* dweights, const int* position, const int* rows_kept, int tokens, int topk, int hidden,
                                    int elem, cudaStream_t stream);

// ---- products of the rows of every group with the group's matrix (grouped_gemm.cu, grouped_wgrad.cu)
cudaError_t launch_grouped_gemm(const void* x, long long ldx, const void* w, long long ldw, long long lde, const int* offsets, void* out,
                                long long ldo, int rows, int groups, int n, int k, bool backward, int elem, int bn, bool zero_rest,
                                int* error_words, cudaStream_t stream);
cudaError_t launch_grouped_wgrad(const void* dy, long long lddy, const void* x, long long ldx, const int* offsets, void* out, long long ldo,
                                 long long lde, int rows, int groups, int n, int k, int elem, bool f32_out, int* error_words,
                                 cudaStream_t stream);

// ---- 8-bit floating point with fp32 scales per block of 128 (fp8_block_gemm.cu, quantize_block.cu)
cudaError_t launch_quantize_rows(const void* x, long long ldx, void* q, float* scales, long long s_row, long long s_block, int rows, int k,
                                 int elem, cudaStream_t stream);
cudaError_t launch_quantize_blocks(const void* w, long long ldw, long long lde, void* q, float* scales, int groups, int n, int k, int elem,
                                   cudaStream_t stream);
cudaError_t launch_fp8_block_gemm(const void* a, long long lda, const float* sa, long long sa_row, long long sa_block, const void* w,
                                  long long ldw, long long lde, const float* sb, const int* offsets, void* out, long long ldo, int rows,
                                  int groups, int n, int k, int bn, bool few_rows, bool zero_rest, int* error_words, cudaStream_t stream);

// ---- gradient norm and clipping
struct GradTensor {
  const void* src;
  void* dst;               // clipped values (may be src); unused by the norm
  long long numel;
  int first_chunk;         // chunks of the tensors before this one in the same launch
  short src_type, dst_type;
};
constexpr int kGradTensorsPerLaunch = 1000;      // 32 bytes each: a launch takes up to 32764 bytes of arguments
int grad_norm_partials(const GradTensor* tensors, int count);     // doubles that launch_grad_norm writes for this list
cudaError_t launch_grad_norm(const GradTensor* tensors, int count, double* partials, cudaStream_t stream);
cudaError_t launch_grad_sum(const double* partials, int count, double* sum, float* norm, cudaStream_t stream);
cudaError_t launch_grad_scale(const GradTensor* tensors, int count, const double* partials, int partial_count, double max_norm, float* norm,
                              cudaStream_t stream);

}  // namespace sm100
}  // namespace msccl
