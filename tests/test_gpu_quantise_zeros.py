"""Zeros keep their sign in the quantisation: x / scale does."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize('top', [0.0, 2.0 ** -99, 1.0, 60000.0, float('inf')])
def test_signs_of_zeros(top, dtype):
    from msccl.ops.fp8_block import quantize_fp8_block, quantize_fp8_block_weight
    x = torch.zeros(3, 144, dtype=dtype, device='cuda')
    x[:, ::2] = -0.0
    x[1, 5], x[1, 130] = top, -top
    for q, _ in (quantize_fp8_block(x), quantize_fp8_block_weight(x)):
        zero = x == 0
        assert torch.equal(q.view(torch.uint8)[zero], torch.where(torch.signbit(x), 0x80, 0).to(torch.uint8)[zero])
