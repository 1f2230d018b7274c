"""The workspace of a large sort lives until the kernels that use it have been launched (CPU, with the launch replaced)."""
import contextlib
import weakref

import pytest
import torch

from msccl.ops import moe_rows


@pytest.mark.parametrize('copies', [16, 40000])
def test_every_buffer_is_alive_at_the_launch(monkeypatch, copies):
    made, launched = [], []
    empty = torch.empty

    def recorded(*a, **k):
        t = empty(*a, **k)
        made.append((t.data_ptr(), weakref.ref(t)))
        return t

    class Native:
        def sort_copies_workspace(self, n, experts):
            return 100 if n > 32768 else 0

        def sort_copies(self, ids, wide, n, experts, sorted_copy, offsets, position, counts, stream):
            launched.append(counts)
            assert (counts == 0) == (n <= 32768)
            assert not counts or any(t() is not None and address == counts for address, t in made), 'the workspace is gone'

    monkeypatch.setattr(moe_rows, 'load', Native)
    monkeypatch.setattr(moe_rows, 'check_devices', lambda *a: 0)
    monkeypatch.setattr(moe_rows, 'on_stream', lambda *a: contextlib.nullcontext())
    monkeypatch.setattr(moe_rows, 'stream_handle', lambda i: 0)
    monkeypatch.setattr(moe_rows.torch, 'empty', recorded)
    moe_rows.sort_copies(torch.zeros(copies, 1, dtype=torch.int32), 4)
    assert len(launched) == 1
