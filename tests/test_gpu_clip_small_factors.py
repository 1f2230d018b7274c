"""Clipping by a factor that fp32 does not hold in full: the values are held, so they are to be right."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('max_norm', [1e-1, 1e-3, 1e-6, 1e-8, 1e-15, 1e-20, 1e-30, 1e-36])
def test_subnormal_factors(max_norm, dtype):
    from msccl.ops.grad_norm import clip_grad_norm
    gen = torch.Generator(device='cuda').manual_seed(0)
    g = (torch.randn(1000, device='cuda', generator=gen) * 1e37).to(dtype)
    g[:200] *= 1e-10
    g[200:300] *= 1e-37
    want_norm = math.sqrt(float((g.double() ** 2).sum()))
    factor = max_norm / (want_norm + 1e-6)
    assert factor < 2.0 ** -126 or max_norm == 1e-1
    ideal = g.double() * factor
    for out_type in (torch.float32, torch.bfloat16):
        out = torch.empty_like(g, dtype=out_type)
        clip_grad_norm([g], max_norm, out=[out])
        # the norm: 6 steps of 2^-24 (groups of 8 squares); the factor's and the product's rounding; the result's, and half of the least
        # number of the type
        step, least = torch.finfo(out_type).eps / 2, torch.finfo(out_type).smallest_normal * torch.finfo(out_type).eps
        assert torch.all((out.double() - ideal).abs() <= (step + 9 * 2.0 ** -24) * ideal.abs() + least)
    clip_grad_norm([g], max_norm)
    least = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    assert torch.all((g.double() - ideal).abs() <= (torch.finfo(dtype).eps / 2 + 9 * 2.0 ** -24) * ideal.abs() + least)
