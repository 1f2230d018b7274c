"""What a backward pass reads may come back from a saved-tensor hook with other strides, or off the boundary of 16 bytes: the kernels get
none of that.  On the CPU, with the launches replaced by checks of their arguments."""
import contextlib
import ctypes

import pytest
import torch

from msccl.ops import grouped, moe_rows
from msccl.ops.moe_rows import CopyOrder

UNIT = 8                                                   # bf16 elements of 16 bytes


class _Native:
    """Pointers and strides in the places where the bindings have them."""
    calls = []

    def grouped_gemm(self, x, ldx, w, ldw, lde, offsets, out, ldo, rows, groups, n, k, backward, *rest):
        self.calls.append('dx' if backward else 'y')
        assert not (x % 16 or w % 16 or out % 16 or ldx % UNIT or ldw % UNIT or lde % UNIT or ldo % UNIT)
        assert ldx >= (n if backward else k) and ldw >= k and lde >= (n - 1) * ldw + k

    def grouped_wgrad(self, dy, lddy, x, ldx, offsets, out, ldo, lde, rows, groups, n, k, *rest):
        self.calls.append('dw')
        assert not (dy % 16 or x % 16 or out % 16 or lddy % UNIT or ldx % UNIT) and lddy >= n and ldx >= k

    def scatter_rows(self, *a):
        pass

    def combine_rows(self, *a):
        pass

    def combine_backward(self, dy, lddy, ys, ldy, weights, *rest):
        self.calls.append('combine')
        assert not (dy % 16 or ys % 16 or lddy % UNIT or ldy % UNIT) and self.weights[0].data_ptr() != 0
        hidden, read = rest[6], torch.frombuffer((ctypes.c_float * 6).from_address(weights), dtype=torch.float32)
        assert hidden == 16 and torch.equal(read, self.weights[0].reshape(-1)), 'weights are read as they lie in memory'


@pytest.fixture
def native(monkeypatch):
    native = _Native()
    native.calls = []
    for m in (grouped, moe_rows):
        monkeypatch.setattr(m, 'load', lambda: native)
        monkeypatch.setattr(m, 'check_devices', lambda *a: 0)
        monkeypatch.setattr(m, 'on_stream', lambda *a: contextlib.nullcontext())
        monkeypatch.setattr(m, 'stream_handle', lambda i: 0)
    monkeypatch.setattr(grouped, 'error_words', lambda i: 0)
    return native


def _off_the_boundary(t):
    big = torch.zeros(*t.shape[:-1], t.shape[-1] + 3, dtype=t.dtype)
    big[..., 1:-2] = t
    return big[..., 1:-2]


def _overlapping(t):
    return t.reshape(-1)[:1].expand(t.shape) if t.dtype == torch.bfloat16 else t.t().contiguous().t()


def _odd_rows(t):
    big = torch.zeros(*t.shape[:-1], t.shape[-1] + 4, dtype=t.dtype)
    big[..., :-4] = t
    return big[..., :-4]


@pytest.mark.parametrize('unpack', [lambda t: t, _off_the_boundary, _overlapping, _odd_rows])
def test_operands_of_the_backward_pass(native, unpack):
    offsets = torch.tensor([0, 2, 6], dtype=torch.int32)
    order = CopyOrder(torch.arange(6, dtype=torch.int32), offsets, torch.arange(6, dtype=torch.int32).view(3, 2))
    x, w = torch.ones(6, 16).bfloat16().requires_grad_(), torch.ones(2, 8, 16).bfloat16().requires_grad_()
    ys, weights = torch.ones(6, 16).bfloat16().requires_grad_(), torch.arange(6.0).view(3, 2).requires_grad_()
    native.weights = [weights.detach()]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        y, z = grouped.grouped_gemm(x, w, offsets), moe_rows.combine_rows(ys, weights, order)
    torch.autograd.grad((y, z), (x, w, ys, weights), (torch.ones_like(y), torch.ones_like(z)))
    assert native.calls.count('combine') == 1 and {'y', 'dx', 'dw'} <= set(native.calls)
