"""Orders of copies that ``sort_copies`` did not make: refused where their shapes and types show it (on CPU tensors, before the device is
looked at)."""
import pytest
import torch

from msccl.ops.moe_rows import CopyOrder, combine_rows, gather_rows

TOKENS, K = 6, 2
GOOD = CopyOrder(torch.arange(12, dtype=torch.int32), torch.tensor([0, 5, 12], dtype=torch.int32), torch.arange(12, dtype=torch.int32).view(TOKENS, K))
BAD = [
    GOOD._replace(position=GOOD.position[:4]),                         # the first tokens of an order
    GOOD._replace(position=GOOD.position[:, :1]),
    GOOD._replace(position=GOOD.position[:, :1].contiguous()),
    GOOD._replace(position=GOOD.position.long()),
    GOOD._replace(position=GOOD.position.t().contiguous().t()),
    GOOD._replace(position=GOOD.position.reshape(-1)),
    GOOD._replace(position=GOOD.position[:0], sorted_copy=GOOD.sorted_copy[:0]),
    GOOD._replace(position=torch.zeros(1, 9, dtype=torch.int32), sorted_copy=torch.zeros(9, dtype=torch.int32)),
    GOOD._replace(offsets=GOOD.offsets[:0]),
    GOOD._replace(offsets=GOOD.offsets[:1]),
    GOOD._replace(offsets=GOOD.offsets.long()),
    GOOD._replace(offsets=GOOD.offsets.view(1, 3)),
    GOOD._replace(offsets=torch.zeros(6, dtype=torch.int32)[::2]),
    GOOD._replace(sorted_copy=GOOD.sorted_copy[:10]),
]


@pytest.mark.parametrize('order', BAD)
def test_refused(order):
    tokens = order.position.shape[0]
    k = order.position.shape[1] if order.position.dim() == 2 else 1
    with pytest.raises(ValueError, match='order'):
        gather_rows(torch.zeros(tokens, 16), order)
    with pytest.raises(ValueError, match='order'):
        combine_rows(torch.zeros(tokens * k, 16), torch.zeros(tokens, k), order)


def test_a_whole_one_reaches_the_device_check():
    for call in (lambda: gather_rows(torch.zeros(TOKENS, 16), GOOD), lambda: combine_rows(torch.zeros(12, 16), torch.zeros(TOKENS, K), GOOD)):
        with pytest.raises(ValueError, match='CUDA'):
            call()
