"""The operators on a stream that is given, with their gradients; under checkpointing and saved-tensor hooks; gradients of unusual layouts."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _whole(gen, *shape, dtype=torch.bfloat16):
    return torch.randint(-2, 3, shape, device='cuda', generator=gen).to(dtype)


def _layer_operands(gen):
    from msccl.ops.moe_rows import sort_copies
    order = sort_copies(torch.randint(-1, 4, (200, 2), device='cuda', generator=gen), 4)
    return order, _whole(gen, 200, 64), _whole(gen, 4, 128, 64), torch.randint(0, 3, (200, 2), device='cuda', generator=gen).float()


def _run(order, x, w, weights, stream=None):
    from msccl.ops import combine_rows, gather_rows, grouped_gemm
    xs = gather_rows(x, order, stream=stream)
    return combine_rows(grouped_gemm(xs, w, order.offsets, stream=stream), weights, order, stream=stream)


def test_forward_and_backward_on_a_given_stream():
    from msccl.ops import check_gemm_errors
    gen = torch.Generator(device='cuda').manual_seed(0)
    order, *operands = _layer_operands(gen)
    dy = _whole(gen, 200, 128)
    leaves = [t.clone().requires_grad_() for t in operands]
    want_y = _run(order, *leaves)
    want = torch.autograd.grad(want_y, leaves, dy)
    for _ in range(3):
        leaves = [t.clone().requires_grad_() for t in operands]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        y = _run(order, *leaves, stream=side)
        torch.cuda.current_stream().wait_stream(side)
        got = torch.autograd.grad(y, leaves, dy)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(y, want_y) and all(torch.equal(a, b) for a, b in zip(got, want))
    check_gemm_errors()


def test_clipping_and_fp8_on_a_given_stream():
    from msccl.ops import check_gemm_errors, clip_grad_norm, gemm_fp8_block, quantize_fp8_block, quantize_fp8_block_weight
    gen = torch.Generator(device='cuda').manual_seed(1)
    grads = [torch.randn(5000 + i, device='cuda', generator=gen) for i in range(9)]
    outs = [[torch.empty_like(g) for g in grads] for _ in range(2)]
    x, w = torch.randn(70, 512, device='cuda', generator=gen), torch.randn(264, 512, device='cuda', generator=gen)
    norm = clip_grad_norm(grads, 1.0, out=outs[0])
    y = gemm_fp8_block(*quantize_fp8_block(x), *quantize_fp8_block_weight(w))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    norm2 = clip_grad_norm(grads, 1.0, out=outs[1], stream=side)
    out = torch.empty(70, 264, dtype=torch.bfloat16, device='cuda')
    gemm_fp8_block(*quantize_fp8_block(x, stream=side), *quantize_fp8_block_weight(w, stream=side), out=out, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    check_gemm_errors()
    assert torch.equal(norm, norm2) and all(torch.equal(a, b) for a, b in zip(*outs)) and torch.equal(out, y)


@pytest.mark.parametrize('how', ['checkpoint', 'save_on_cpu', 'strided'])
def test_gradients_with_what_autograd_keeps_elsewhere(how):
    from torch.utils.checkpoint import checkpoint
    from msccl.ops import check_gemm_errors
    gen = torch.Generator(device='cuda').manual_seed(2)
    order, *operands = _layer_operands(gen)
    dy = _whole(gen, 200, 128)
    leaves = [t.clone().requires_grad_() for t in operands]
    want = torch.autograd.grad(_run(order, *leaves), leaves, dy)
    if how == 'checkpoint':
        y = checkpoint(_run, order, *leaves, use_reentrant=False)
    elif how == 'save_on_cpu':
        with torch.autograd.graph.save_on_cpu():
            y = _run(order, *leaves)
    else:
        # hooks that give the kernels' operands back with other strides, and off the boundary of 16 bytes
        def unpack(t):
            big = torch.zeros(*t.shape[:-1], t.shape[-1] + 3, dtype=t.dtype, device=t.device)
            big[..., 1:-2] = t
            return big[..., 1:-2]
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            y = _run(order, *leaves)
    got = torch.autograd.grad(y, leaves, dy)
    check_gemm_errors()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize('pitch', [8, 56, 64])
def test_gradients_whose_rows_overlap(pitch):
    """Windows of one stretch of memory as the gradient of a product and of both row operators."""
    from msccl.ops import check_gemm_errors, combine_rows, gather_rows, grouped_gemm
    gen = torch.Generator(device='cuda').manual_seed(3)
    order, x, w, weights = _layer_operands(gen)
    base = _whole(gen, 400 * pitch + 128)
    for call, leaf, shape in ((lambda t: gather_rows(t, order), x, (400, 64)),
                              (lambda t: grouped_gemm(t, w, order.offsets), _whole(gen, 400, 64), (400, 128)),
                              (lambda t: grouped_gemm(_one, t, order.offsets), w, (400, 128)),
                              (lambda t: combine_rows(t, weights, order), _whole(gen, 400, 64), (200, 64))):
        _one = _whole(torch.Generator(device='cuda').manual_seed(4), 400, 64)
        dy = base.as_strided(shape, (pitch, 1))
        leaf = leaf.clone().requires_grad_()
        y = call(leaf)
        got, = torch.autograd.grad(y, leaf, dy, retain_graph=True)
        want, = torch.autograd.grad(y, leaf, dy.contiguous())
        assert torch.equal(got, want)
    check_gemm_errors()
