"""``FlatGradients.clip_grad_norm`` on the CPU, with a plain clip in place of the kernels: the buckets are what it scales, so the
parameters' gradients have to be views of them."""
import pytest
import torch

from msccl.parallel import FlatGradients, data_parallel


def _plain_clip(tensors, max_norm, reduce=None):
    norm = torch.sqrt(sum((t.double() ** 2).sum() for t in tensors)).float()
    for t in tensors:
        t.mul_(min(1.0, max_norm / (float(norm) + 1e-6)))
    return norm


@pytest.fixture
def model(monkeypatch):
    monkeypatch.setattr(data_parallel, 'clip_grad_norm', _plain_clip)
    params = [torch.nn.Parameter(torch.full((n,), 2.0)) for n in (5, 12)]
    return params, FlatGradients(params, lambda n, d: torch.empty(n, dtype=d), bucket_bytes=32)


def _backward(params):
    sum(p.square().sum() for p in params).backward()


def test_buckets_are_clipped(model):
    params, flat = model
    assert len(flat.buckets) == 2
    _backward(params)
    assert abs(float(flat.clip_grad_norm(1.0)) - 4 * 17 ** 0.5) <= 1e-5
    assert abs(sum(float((p.grad ** 2).sum()) for p in params) - 1.0) <= 1e-5


@pytest.mark.parametrize('which', [0, 1])
def test_a_replaced_gradient_is_refused(model, which):
    params, flat = model
    torch.optim.SGD(params[which:which + 1], lr=0.1).zero_grad()       # its default sets .grad to None
    with pytest.raises(RuntimeError, match='replaced'):
        flat.clip_grad_norm(1.0)
    _backward(params)                                                  # autograd makes a tensor of its own
    before = [p.grad.clone() for p in params]
    with pytest.raises(RuntimeError, match='replaced'):
        flat.clip_grad_norm(1.0)
    assert all(torch.equal(p.grad, b) for p, b in zip(params, before))
    calls = []
    with pytest.raises(RuntimeError, match='replaced'):
        flat.all_reduce_gradients(calls.append, 2)
    assert not calls, 'a bucket was summed before the gradients of a later one were looked at'


def test_a_parameter_without_elements(monkeypatch):
    monkeypatch.setattr(data_parallel, 'clip_grad_norm', _plain_clip)
    params = [torch.nn.Parameter(torch.ones(n)) for n in (4, 0, 4)]
    flat = FlatGradients(params, lambda n, d: torch.empty(n, dtype=d))
    _backward(params)
    assert abs(float(flat.clip_grad_norm(1.0)) - 32 ** 0.5) <= 1e-5
    flat.all_reduce_gradients(lambda t: None, 1)
