"""The words in which the kernels report a wait that ran out are zero before any stream can read them (CPU, with the device replaced)."""
import contextlib
import types

import pytest
import torch

from msccl.ops import _launch, gemm


def test_the_words_are_zero_before_they_are_handed_out(monkeypatch):
    events = []
    monkeypatch.setattr(gemm, '_error_words', {})
    monkeypatch.setattr(_launch, '_words', {})
    zeros = torch.zeros
    monkeypatch.setattr(torch, 'zeros', lambda *a, device=None, **k: events.append(('zeros', device)) or zeros(*a, **k))
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: False)
    monkeypatch.setattr(torch.cuda, 'Stream', lambda device, priority: types.SimpleNamespace(
        synchronize=lambda: events.append(('synchronize', device))))
    monkeypatch.setattr(torch.cuda, 'stream', contextlib.nullcontext)
    monkeypatch.setattr(torch.cuda, 'current_stream', lambda *a: pytest.fail('work of the current stream may wait for this thread'))
    address = _launch.error_words(1)
    assert events == [('zeros', 'cuda:1'), ('synchronize', 1)]
    assert _launch.error_words(1) == address == gemm._errors('cuda:1').data_ptr() and len(events) == 2
