"""Operands with a forward-mode tangent: the operators have no rule for one, so they say so instead of dropping it.  On the CPU, with the
launches replaced."""
import contextlib

import pytest
import torch
import torch.autograd.forward_ad as fw

from msccl.ops import grouped, moe_rows
from msccl.ops.moe_rows import CopyOrder


@pytest.fixture
def calls(monkeypatch):
    for module in (grouped, moe_rows):
        monkeypatch.setattr(module, 'check_devices', lambda *a: 0)
        monkeypatch.setattr(module, 'on_stream', lambda *a: contextlib.nullcontext())
    monkeypatch.setattr(grouped, '_launch', lambda x, w, *a: torch.zeros(x.shape[0], w.shape[1], dtype=x.dtype))
    monkeypatch.setattr(moe_rows, '_scatter', lambda x, order: torch.zeros(6, 16))
    monkeypatch.setattr(moe_rows, '_combine', lambda ys, weights, order: torch.zeros(3, 16))
    offsets = torch.tensor([0, 2, 6], dtype=torch.int32)
    order = CopyOrder(torch.arange(6, dtype=torch.int32), offsets, torch.arange(6, dtype=torch.int32).view(3, 2))
    rows = dict(x=torch.ones(6, 16).bfloat16(), w=torch.ones(2, 8, 16).bfloat16())
    ys = dict(ys=torch.ones(6, 16), weights=torch.ones(3, 2))
    return [(lambda x, w: grouped.grouped_gemm(x, w, offsets), rows), (lambda x: moe_rows.gather_rows(x, order), dict(x=torch.ones(3, 16))),
            (lambda ys, weights: moe_rows.combine_rows(ys, weights, order), ys)]


@pytest.mark.parametrize('grad_mode', [True, False])
@pytest.mark.parametrize('which', [0, 1, 2])
def test_a_tangent_is_refused(calls, which, grad_mode):
    f, operands = calls[which]
    with fw.dual_level(), torch.set_grad_enabled(grad_mode):
        f(**operands)                                      # no tangent among the operands
        for name, t in operands.items():
            dual = fw.make_dual(t, torch.ones_like(t))
            with pytest.raises(NotImplementedError):
                f(**{**operands, name: dual})
    f(**operands)


def test_a_tangent_and_a_given_result(calls):
    _, operands = calls[0]
    with fw.dual_level():
        dual = fw.make_dual(operands['x'], torch.ones(6, 16).bfloat16())
        with pytest.raises(ValueError, match='gradient'):
            grouped.grouped_gemm(dual, operands['w'], torch.tensor([0, 2, 6], dtype=torch.int32), out=torch.zeros(6, 8).bfloat16())
