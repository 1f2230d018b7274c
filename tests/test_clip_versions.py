"""The version counters of clipped tensors, on the CPU with the launches replaced."""
import pytest
import torch

from msccl.ops.grad_norm import clip_grad_norm, grad_norm


class _Tensors(list):
    def partials(self):
        return 1

    def overlapping(self):
        return False


class _Native:
    def GradList(self, gradients, out, dtypes, same_dense_layout):
        return _Tensors(g for g in gradients if g.numel())

    def grad_norm(self, *a):
        pass

    grad_sum = grad_scale = grad_norm


@pytest.fixture(autouse=True)
def without_a_gpu(monkeypatch):
    import contextlib
    import sys
    m = sys.modules['msccl.ops.grad_norm']
    monkeypatch.setattr(m, 'load', _Native)
    monkeypatch.setattr(m, 'on_stream', lambda *a: contextlib.nullcontext())
    monkeypatch.setattr(m, 'stream_handle', lambda i: 0)


def test_what_is_written_gets_a_new_version():
    g, h, o, p = (torch.ones(4) for _ in range(4))
    clip_grad_norm([g, None, h], 1.0)
    assert g._version == h._version == 1
    clip_grad_norm([g, None, h], 1.0, out=[o, None, p])
    assert g._version == h._version == 1 and o._version == p._version == 1
    grad_norm([g, h])
    assert g._version == h._version == 1


def test_a_refused_call_writes_nothing(monkeypatch):
    g = torch.ones(4)
    monkeypatch.setattr(_Tensors, 'overlapping', lambda self: True)
    with pytest.raises(ValueError):
        clip_grad_norm([g], 1.0)
    assert g._version == 0
