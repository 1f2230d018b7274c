"""Clipping writes through raw pointers; autograd has to know of it all the same."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _saved(out):
    """A tensor in whose graph ``out``, the gradient or the clipped copy, is saved."""
    leaf = torch.ones_like(out).requires_grad_()
    return (leaf * out).sum()


@pytest.mark.parametrize('count', [1, 150])
def test_a_saved_gradient_that_is_clipped_is_noticed(count):
    from msccl.ops import clip_grad_norm
    grads = [torch.full((10,), 2.0, device='cuda') for _ in range(count)]
    loss = _saved(grads[-1])
    clip_grad_norm(grads, 1.0)
    with pytest.raises(RuntimeError, match='inplace'):
        loss.backward()
    # into other tensors: those are written, the gradients are not
    outs = [torch.empty_like(g) for g in grads]
    loss, kept = _saved(outs[0]), _saved(grads[0])
    clip_grad_norm(grads, 1.0, out=outs)
    with pytest.raises(RuntimeError, match='inplace'):
        loss.backward()
    kept.backward()


def test_gradients_with_a_graph():
    from msccl.ops import clip_grad_norm
    x = torch.linspace(1, 2, 10, device='cuda').requires_grad_()
    g, = torch.autograd.grad((x ** 3).sum(), x, create_graph=True)
    penalty = (g * g).sum()
    clip_grad_norm([g], 1.0)
    with pytest.raises(RuntimeError, match='inplace'):
        penalty.backward()


def test_views_of_a_bucket():
    from msccl.ops import clip_grad_norm
    flat = torch.ones(32, device='cuda')
    loss = _saved(flat[8:16])
    clip_grad_norm([flat], 1.0)
    with pytest.raises(RuntimeError, match='inplace'):
        loss.backward()


def test_the_norm_alone_and_inference_tensors():
    from msccl.ops.grad_norm import clip_grad_norm, grad_norm
    g = torch.ones(16, device='cuda')
    loss = _saved(g)
    assert grad_norm([g]) == 4
    loss.backward()
    with torch.inference_mode():
        g = torch.full((16,), 2.0, device='cuda')
    clip_grad_norm([g, None], 4.0)
    with torch.inference_mode():
        assert torch.all((g - 1).abs() <= 2.0 ** -20)
