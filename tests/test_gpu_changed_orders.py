"""Positions and offsets that hold other values than ``sort_copies`` gave them: the kernels keep to their operands."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('tokens,topk', [(5, 1), (40, 2), (33, 3), (20, 8)])
def test_rows_outside_are_passed_by(tokens, topk, dtype):
    from msccl.ops.moe_rows import combine_rows, gather_rows, sort_copies
    gen = torch.Generator(device='cuda').manual_seed(topk)
    rows, hidden = tokens * topk, 72
    good = sort_copies(torch.randint(0, 4, (tokens, topk), device='cuda', generator=gen), 4)
    x, dy = torch.randn(tokens, hidden, device='cuda', generator=gen).to(dtype), torch.randn(tokens, hidden, device='cuda', generator=gen).to(dtype)
    ys, dxs = torch.randn(rows, hidden, device='cuda', generator=gen).to(dtype), torch.randn(rows, hidden, device='cuda', generator=gen).to(dtype)
    weights = torch.rand(tokens, topk, device='cuda', generator=gen)
    outside = torch.rand(tokens, topk, device='cuda', generator=gen) < 0.3
    outside[0, 0] = True
    far = torch.tensor([-1, rows, rows + 1, 1 << 30, -(1 << 31), (1 << 31) - 1], device='cuda')
    position = torch.where(outside, far[torch.randint(0, 6, (tokens, topk), device='cuda', generator=gen)], good.position).int()
    for last in (rows, 1 << 30):                           # the number of kept rows, and one that no order has
        offsets = good.offsets.clone()
        offsets[-1] = last
        order = good._replace(position=position, offsets=offsets)
        leaves = [t.clone().requires_grad_() for t in (x, ys, weights)]
        xs, y = gather_rows(leaves[0], order), combine_rows(leaves[1], leaves[2], order)
        dx, dys, dweights = torch.autograd.grad((xs, y), leaves, (dxs, dy))
        inside = ~outside
        at = position[inside].long()
        token = torch.arange(tokens, device='cuda')[:, None].expand(tokens, topk)[inside]
        assert torch.equal(xs[at], x[token])
        # as if those copies had a weight of zero and, in the gather, no gradient
        w = torch.where(inside, weights, 0.0)
        safe = torch.where(inside, position, 0).long()
        want = (ys.double()[safe] * w[:, :, None]).sum(1)
        step = torch.finfo(dtype).eps / 2
        assert torch.all((y.double() - want).abs() <= step * (1 + 2.0 ** -8) * want.abs() + 2 * topk * 2.0 ** -24 * (ys.double()[safe].abs() * w[:, :, None]).sum(1))
        want = (dxs.double()[safe] * inside[:, :, None]).sum(1)
        assert torch.all((dx.double() - want).abs() <= step * (1 + 2.0 ** -8) * want.abs() + topk * 2.0 ** -24 * (dxs.double()[safe].abs() * inside[:, :, None]).sum(1))
        assert torch.all(dweights[outside] == 0)
        assert torch.equal(dys[at], (dy.float()[token] * weights[inside][:, None]).to(dtype))
    # no kept rows at all: nothing is read
    offsets.fill_(-7)
    order = good._replace(offsets=offsets)
    assert torch.all(gather_rows(x, order) == 0) and torch.all(combine_rows(ys.fill_(float('nan')), weights, order) == 0)
