"""Hand-written sm_100a compute kernels (tcgen05 GEMM and its fused variants, the operators of an expert layer) as PyTorch callables."""
from msccl.ops.gemm import gemm_bf16, GemmKernelError, check_gemm_errors  # noqa: F401
from msccl.ops.fp8_block import gemm_fp8_block, grouped_gemm_fp8_block, quantize_fp8_block, quantize_fp8_block_weight  # noqa: F401
from msccl.ops.grad_norm import clip_grad_norm  # noqa: F401
from msccl.ops.grouped import grouped_gemm, grouped_gemm_dgrad, grouped_gemm_wgrad  # noqa: F401
from msccl.ops.moe_rows import combine_rows, gather_rows, sort_copies  # noqa: F401
