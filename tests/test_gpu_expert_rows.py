"""Rows around the experts, gradient norm and clipping against 64-bit references."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _chosen(gen, tokens, topk, experts, dropped, dtype=torch.int32):
    e = torch.randint(0, experts, (tokens, topk), device='cuda', generator=gen)
    if dropped:
        e[torch.rand(tokens, topk, device='cuda', generator=gen) < 0.3] = -1
        e[torch.rand(tokens, topk, device='cuda', generator=gen) < 0.1] = experts
    return e.to(dtype)


def _plain_order(chosen, experts):
    key = torch.where((chosen >= 0) & (chosen < experts), chosen, experts).reshape(-1).long()
    order = torch.argsort(key, stable=True)
    position = torch.empty_like(order)
    position[order] = torch.arange(order.numel(), device='cuda')
    counts = torch.bincount(key, minlength=experts + 1)
    return order, torch.cat([counts.new_zeros(1), counts.cumsum(0)[:experts]]), position


@pytest.mark.parametrize('tokens,topk,experts', [(1, 1, 1), (1, 8, 8), (16, 2, 8), (511, 3, 5), (512, 2, 512), (1024, 1, 64), (4097, 2, 8),
                                                 (16384, 8, 256)])
@pytest.mark.parametrize('dropped', [False, True])
def test_sort_copies(tokens, topk, experts, dropped):
    from msccl.ops.moe_rows import sort_copies
    gen = torch.Generator(device='cuda').manual_seed(tokens)
    for dtype in (torch.int32, torch.int64):
        chosen = _chosen(gen, tokens, topk, experts, dropped, dtype)
        order = sort_copies(chosen, experts)
        want = _plain_order(chosen, experts)
        assert torch.equal(order.sorted_copy.long(), want[0]) and torch.equal(order.offsets.long(), want[1])
        assert torch.equal(order.position.reshape(-1).long(), want[2]) and order.position.shape == (tokens, topk)
    # ids that lie apart in memory, and 64-bit ids that would wrap into the range
    wide = torch.zeros(tokens, topk * 2, dtype=torch.int64, device='cuda')
    wide[:, ::2] = chosen
    assert torch.equal(sort_copies(wide[:, ::2], experts).sorted_copy, order.sorted_copy)
    assert int(sort_copies(torch.full((tokens, topk), 1 << 32, device='cuda'), experts).offsets[-1]) == 0


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize('tokens,topk,experts,hidden', [(1, 1, 1, 8), (1, 2, 4, 4096), (37, 3, 5, 264), (300, 8, 16, 1000), (129, 2, 8, 2056)])
@pytest.mark.parametrize('dropped', [False, True])
def test_rows_and_their_gradients(tokens, topk, experts, hidden, dropped, dtype):
    from msccl.ops.moe_rows import combine_rows, gather_rows, sort_copies
    gen = torch.Generator(device='cuda').manual_seed(hidden)

    def normal(*shape):
        return torch.randn(*shape, device='cuda', generator=gen).to(dtype)
    chosen = _chosen(gen, tokens, topk, experts, dropped)
    order = sort_copies(chosen, experts)
    sorted_copy, offsets, position = _plain_order(chosen, experts)
    kept = int(offsets[-1])
    x, ys, dxs, dy = normal(tokens, hidden), normal(tokens * topk, hidden), normal(tokens * topk, hidden), normal(tokens, hidden)
    weights = torch.rand(tokens, topk, device='cuda', generator=gen)
    ys[kept:] = float('nan')                               # the results of dropped copies are nobody's
    dxs[kept:] = float('nan')
    x.requires_grad_(), ys.requires_grad_(), weights.requires_grad_()
    xs, y = gather_rows(x, order), combine_rows(ys, weights, order)
    dx, dys, dweights = torch.autograd.grad((xs, y), (x, ys, weights), (dxs, dy))
    with torch.no_grad():
        used = (position < kept).view(tokens, topk, 1)
        back = position.view(tokens, topk)

        def copies(t):
            return torch.where(used, t.double()[back], 0.0)
        w = weights.double()[:, :, None]
        want_xs = torch.zeros_like(xs)
        want_xs[:kept] = x[sorted_copy[:kept] // topk]
        assert torch.equal(xs, want_xs)
        # a product and a sum of fp32 for each copy (2^-24 each), one rounding to the type
        step, f32 = torch.finfo(dtype).eps / 2, 2.0 ** -24
        low = 2.0 ** -25 if dtype == torch.float16 else 0.0

        def near(got, want, magnitude, operations, half_step):
            assert torch.all((got.double() - want).abs() <= half_step * want.abs() * (1 + 2.0 ** -8) + operations * f32 * magnitude + low)
        near(y, (copies(ys) * w).sum(1), (copies(ys).abs() * w).sum(1), 2 * topk, step)
        near(dx, copies(dxs).sum(1), copies(dxs).abs().sum(1), topk, step)
        want_dys = torch.zeros(tokens * topk, hidden, dtype=torch.float64, device='cuda')
        want_dys[:kept] = dy.double()[sorted_copy[:kept] // topk] * weights.double().reshape(-1)[sorted_copy[:kept]][:, None]
        near(dys, want_dys, want_dys.abs(), 1, step)
        products = copies(ys) * dy.double()[:, None, :]
        near(dweights, products.sum(-1), products.abs().sum(-1), hidden, f32)
        # without gradients, and one of the two
        assert torch.equal(gather_rows(x, order), xs) and torch.equal(combine_rows(ys, weights, order), y)
    only = torch.autograd.grad(combine_rows(ys.detach(), weights, order), weights, dy)[0]
    assert torch.equal(only, dweights)
    assert torch.equal(torch.autograd.grad(combine_rows(ys, weights.detach(), order), ys, dy)[0], dys)


def test_gradients_are_difference_quotients():
    """Both operators are linear in each operand: f(a + d) - f(a) = <gradient, d>, exactly for small whole numbers in fp32."""
    from msccl.ops.moe_rows import combine_rows, gather_rows, sort_copies
    gen = torch.Generator(device='cuda').manual_seed(9)

    def whole(*shape):
        return torch.randint(-4, 5, shape, device='cuda', generator=gen).float()
    order = sort_copies(_chosen(gen, 40, 3, 6, True), 6)
    x, ys, weights, cx, cy = whole(40, 20), whole(120, 20), whole(40, 3), whole(120, 20), whole(40, 20)
    for f, operand, c in ((lambda t: gather_rows(t, order), x, cx), (lambda t: combine_rows(t, weights, order), ys, cy),
                          (lambda t: combine_rows(ys, t, order), weights, cy)):
        leaf = operand.clone().requires_grad_()
        (f(leaf) * c).sum().backward()
        d = whole(*operand.shape)
        assert ((f(operand + d) - f(operand)).double() * c.double()).sum() == (leaf.grad.double() * d.double()).sum()


def test_rows_with_strides_and_expanded_gradients():
    from msccl.ops.moe_rows import combine_rows, gather_rows, sort_copies
    gen = torch.Generator(device='cuda').manual_seed(0)
    order = sort_copies(_chosen(gen, 50, 2, 4, False), 4)
    big = torch.randn(50, 80, device='cuda', generator=gen).bfloat16()
    x = big[:, 8:72].detach().requires_grad_()
    xs = gather_rows(x, order)
    assert torch.equal(xs, gather_rows(x.detach().contiguous(), order))
    xs.sum().backward()                                    # expanded ones, strides of zero
    assert torch.all(x.grad == 2)
    ys = torch.randn(100, 80, device='cuda', generator=gen).bfloat16()[:, 8:72]
    weights = torch.rand(2, 50, device='cuda', generator=gen).t()
    assert torch.equal(combine_rows(ys, weights, order), combine_rows(ys.contiguous(), weights.contiguous(), order))
    dy = torch.randn(64, 50, device='cuda', generator=gen).bfloat16().t()
    g = torch.autograd.grad(gather_rows(x, order), x, dy.repeat_interleave(2, 0)[order.sorted_copy.long()].t().contiguous().t())[0]
    assert torch.equal(g, (dy.float() * 2).bfloat16())


# ------------------------------------------------------------------------------------------------------------ norm and clipping
def _norm64(tensors):
    return math.sqrt(sum(float((t.double() ** 2).sum()) for t in tensors))


def _near_norm(got, want):
    # groups of 8 squares in fp32 (8 roundings of 2^-24 of a sum of positive terms), half of that in the root; the result's rounding
    assert abs(float(got) - want) <= (4 + 1 + 1) * 2.0 ** -24 * want


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('sizes', [[1], [7], [16384], [16385, 0, 3], [100000, 1, 65536, 33], list(range(1, 300)), [5] * 1003])
def test_norm_and_clipping(sizes, dtype):
    from msccl.ops.grad_norm import clip_grad_norm, grad_norm
    gen = torch.Generator(device='cuda').manual_seed(len(sizes))
    flat = torch.randn(sum(sizes) + len(sizes), device='cuda', generator=gen).to(dtype)
    grads, at = [], 1
    for s in sizes:                                        # packed back to back: any alignment
        grads.append(flat[at:at + s])
        at += s
    start = flat.clone()
    want = _norm64(grads)
    _near_norm(grad_norm(grads), want)
    # no clipping: nothing changes
    _near_norm(clip_grad_norm(grads, want * 2 + 1), want)
    assert torch.equal(flat, start)
    # into other tensors of each type
    for out_type in (torch.float32, torch.bfloat16, torch.float16):
        holder = torch.full((sum(sizes) + len(sizes) + 2,), 7.0, dtype=out_type, device='cuda')
        outs, at = [], 2
        for s in sizes:
            outs.append(holder[at:at + s])
            at += s
        norm = clip_grad_norm(grads, want / 4, out=outs)
        _near_norm(norm, want)
        factor = (want / 4) / (want + 1e-6)
        step = torch.finfo(out_type).eps / 2
        low = 2.0 ** -25 if out_type == torch.float16 else 0.0
        for g, o in zip(grads, outs):
            # the factor: the norm's 5 roundings and its own; then a product in fp32 and the result's rounding
            assert torch.all((o.double() - g.double() * factor).abs() <= (step + 8 * 2.0 ** -24) * g.double().abs() * factor + low)
        assert torch.all(holder[:2] == 7) and torch.all(holder[at:] == 7) and torch.equal(flat, start)
        assert torch.equal(clip_grad_norm(grads, want / 4, out=outs), norm)
    # in place: the same values as into tensors of the same type
    outs = [torch.empty_like(g) for g in grads]
    clip_grad_norm(grads, want / 4, out=outs)
    clip_grad_norm(grads, want / 4)
    assert all(torch.equal(g, o) for g, o in zip(grads, outs))
    assert flat[0] == start[0] and torch.equal(flat[at - 1:], start[at - 1:])


@pytest.mark.parametrize('values', [[1e30, 1e30, 3e30], [1e-30, 2e-30, 2e-30], [1e-42, 0.0, 0.0], [3e38, 3e38, 1.0], [0.0, 0.0, 0.0]])
def test_norm_of_extreme_values(values):
    from msccl.ops.grad_norm import clip_grad_norm, grad_norm
    g = torch.zeros(1000, device='cuda')
    g[5:8] = torch.tensor(values, device='cuda')
    want = _norm64([g])
    got = float(grad_norm([g]))
    if want > torch.finfo(torch.float32).max:
        assert got == math.inf
    else:
        assert abs(got - want) <= 8 * 2.0 ** -24 * want + 2.0 ** -149
    clip_grad_norm([g], 1.0)
    factor = min(1.0, 1.0 / (want + 1e-6))
    assert torch.allclose(g[5:8].double(), torch.tensor(values, dtype=torch.float64, device='cuda') * factor, rtol=1e-6, atol=1e-44)


def test_infinite_and_nan_gradients():
    from msccl.ops.grad_norm import clip_grad_norm
    for bad in (math.inf, -math.inf, math.nan):
        grads = [torch.ones(100, device='cuda'), torch.ones(33, device='cuda').bfloat16()]
        grads[1][7] = bad
        norm = clip_grad_norm(grads, 1.0)
        if math.isnan(bad):
            assert math.isnan(norm) and all(torch.all(torch.isnan(g)) for g in grads)
        else:
            assert norm == math.inf and torch.all(grads[0] == 0) and torch.isnan(grads[1][7]) and torch.all(grads[1][:7] == 0)


def test_mixed_types_dense_orders_and_reduction():
    from msccl.ops.grad_norm import clip_grad_norm, grad_norm
    gen = torch.Generator(device='cuda').manual_seed(0)
    grads = [torch.randn(40, 30, device='cuda', generator=gen).t(), None, torch.randn(4, 3, 5, 7, device='cuda', generator=gen).half()
             .to(memory_format=torch.channels_last), torch.randn(17, device='cuda', generator=gen).bfloat16(), torch.zeros(0, device='cuda')]
    live = [g for g in grads if g is not None]
    start = [g.clone() for g in live]
    want = _norm64(live)
    _near_norm(grad_norm(grads), want)
    norm = clip_grad_norm(grads, want)                     # the factor is want / (want + 1e-6)
    _near_norm(norm, want)
    # two processes that hold the same gradients: the sum of squares doubles
    norm = clip_grad_norm([g.copy_(s) for g, s in zip(live, start)], want, reduce=lambda t: t.mul_(2))
    _near_norm(norm, want * math.sqrt(2))
    for g, s in zip(live, start):
        step = torch.finfo(g.dtype).eps / 2
        ideal = s.double() * (want / (want * math.sqrt(2) + 1e-6))
        assert torch.all((g.double() - ideal).abs() <= (step + 8 * 2.0 ** -24) * ideal.abs() + (2.0 ** -25 if g.dtype == torch.float16 else 0))
    empty = torch.zeros(0, device='cuda')
    assert grad_norm([empty]) == 0 and clip_grad_norm([empty], 1.0) == 0
    assert clip_grad_norm([empty], 1.0, reduce=lambda t: t.add_(9.0)) == 3


def test_refused_lists():
    from msccl.ops.grad_norm import clip_grad_norm
    t = torch.ones(100, device='cuda')
    for call in (lambda: clip_grad_norm([t, t], 1.0), lambda: clip_grad_norm([t[:60], t[50:]], 1.0), lambda: clip_grad_norm([t, t.cpu()], 1.0),
                 lambda: clip_grad_norm([t[::2]], 1.0), lambda: clip_grad_norm([t[:50]], 1.0, out=[t[1:51]]),
                 lambda: clip_grad_norm([t, t], 1.0, out=[torch.empty_like(t)]), lambda: clip_grad_norm([t], 1.0, out=[t[:50]]),
                 lambda: clip_grad_norm([t.view(10, 10)], 1.0, out=[torch.empty(10, 10, device='cuda').t()]),
                 lambda: clip_grad_norm([t.view(torch.bfloat16)[:100]], 1.0, out=[t]), lambda: clip_grad_norm([t[:1].expand(5)], 1.0)):
        with pytest.raises(ValueError):
            call()
    clip_grad_norm([t], 1.0, out=[t])                      # the gradient itself is fine
    clip_grad_norm([t[:50], t[50:]], 1.0)


def test_large_list_in_a_graph():
    from msccl.ops.grad_norm import clip_grad_norm
    gen = torch.Generator(device='cuda').manual_seed(0)
    grads = [torch.randn(1000 + i, device='cuda', generator=gen) for i in range(150)]
    outs = [torch.empty_like(g) for g in grads]
    clip_grad_norm(grads, 1.0, out=outs)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        norm = clip_grad_norm(grads, 1.0, out=outs)
    for scale in (1.0, 3.0):
        for t in grads:
            t.mul_(scale)
        g.replay()
        want = _norm64(grads)
        _near_norm(norm, want)
        assert abs(_norm64(outs) - want / (want + 1e-6)) <= 1e-6


def test_far_elements():
    from msccl.ops.grad_norm import clip_grad_norm
    t = torch.zeros((1 << 31) + 40000, device='cuda', dtype=torch.bfloat16)
    t[5], t[1 << 31], t[-1] = 3.0, 4.0, 12.0
    assert clip_grad_norm([t], 6.5) == 13.0
    assert [float(v) for v in (t[5], t[1 << 31], t[-1])] == [1.5, 2.0, 6.0]
