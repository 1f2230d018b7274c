"""Quantisation where a quotient is a tie of e4m3, or within a step of one, over the whole range of scales: byte for byte against divisions on
the CPU."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _definition(x, block_rows):
    rows, k = x.shape
    b = x.view(rows // block_rows, block_rows, k // 128, 128)
    scale = b.abs().amax((1, 3), keepdim=True).clamp_min(2.0 ** -100) / torch.tensor(448.0)
    return (b / scale).to(torch.float8_e4m3fn).view(rows, k).view(torch.uint8), scale[:, 0, :, 0]


def _near_ties(exponent):
    """Rows of one block each: a random maximum of that exponent, and values whose quotients are at most two steps of fp32 from the middle of two
    numbers of e4m3 (or from such a number)."""
    gen = torch.Generator().manual_seed(exponent + 200)
    numbers = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    middles = torch.cat([(numbers[1:] + numbers[:-1]) / 2, numbers])
    rows = 512
    top = torch.ldexp(1 + torch.rand(rows, 1, generator=gen), torch.tensor(exponent)).float()
    scale = top.clamp_min(2.0 ** -100) / torch.tensor(448.0)
    q = middles[torch.randint(0, len(middles), (rows, 128), generator=gen)]
    x = (q * scale.double()).float()
    bits = x.view(torch.int32) + torch.randint(-2, 3, x.shape, generator=gen)
    x = torch.where(bits > 0, bits, 0).int().view(torch.float32).minimum(top)
    x = torch.where(torch.rand(x.shape, generator=gen) < 0.5, -x, x)
    x[:, 0] = top[:, 0]
    return x


@pytest.mark.parametrize('exponent', [-126, -112, -101, -100, -99, -98, -95, -92, -90, -86, -84, -83, -82, -81, -80, -75, -60, 0, 60, 127])
def test_bytes_near_ties(exponent):
    from msccl.ops.fp8_block import quantize_fp8_block, quantize_fp8_block_weight
    x = _near_ties(exponent)
    x = x[torch.isfinite(x).all(1)]
    assert len(x) > 400
    q, s = quantize_fp8_block(x.cuda())
    want_q, want_s = _definition(x, 1)
    nonzero = x != 0
    assert torch.equal(s.cpu(), want_s)
    assert torch.equal(q.cpu().view(torch.uint8)[nonzero], want_q[nonzero])
    x = x[:384]
    q, s = quantize_fp8_block_weight(x.cuda())
    want_q, want_s = _definition(x, 128)
    assert torch.equal(s.cpu(), want_s)
    assert torch.equal(q.cpu().view(torch.uint8)[x != 0], want_q[x != 0])


def test_a_tie_at_a_small_scale():
    """The quotient of this pair rounds to a tie; an fp32 remainder of it is not exact."""
    from msccl.ops.fp8_block import quantize_fp8_block
    x = torch.zeros(1, 128)
    x[0, 0], x[0, 1] = float.fromhex('0x1.c0110ap-99'), float.fromhex('0x1.c01108p-115')
    q, s = quantize_fp8_block(x.cuda())
    want_q, want_s = _definition(x, 1)
    assert torch.equal(s.cpu(), want_s) and torch.equal(q.cpu().view(torch.uint8)[:, :2], want_q[:, :2])
