"""Incoming gradients, which may be any view, as the kernels take them."""
import pytest
import torch

from msccl.ops._launch import check_matrix
from msccl.ops.moe_rows import _kernel_rows

BASE = torch.arange(4096, dtype=torch.float32)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('view', [
    lambda b: b.unfold(0, 64, 8)[:20],                     # windows that overlap: rows of 64 that start 8 apart
    lambda b: b.as_strided((20, 64), (56, 1)),
    lambda b: b[:64].expand(20, 64),
    lambda b: b[:1].expand(20, 64),
    lambda b: b[:1280].view(64, 20).t(),
    lambda b: b[3:1283].view(20, 64),                      # off the 16-byte boundary
    lambda b: b[:20 * 66].view(20, 66)[:, :64],
    lambda b: b.as_strided((1, 64), (8, 1)),               # the stride of a single row means nothing
    lambda b: b[:1280].view(20, 64),
    lambda b: b[:20 * 72].view(20, 72)[:, 8:],
])
def test_a_gradient_meets_the_checks_of_an_operand(view, dtype):
    g = view(BASE.to(dtype).clone())
    got = _kernel_rows(g, dtype)
    rows, columns, _ = check_matrix(got, 'dy', (dtype,), 8)
    assert (rows, columns) == g.shape and torch.equal(got, g)
