"""Sizes that no forward pass of ``GroupedMoE`` takes are refused when the layer is made."""
import pytest
import torch

from msccl.parallel import GroupedMoE


@pytest.mark.parametrize('sizes,words', [
    (dict(hidden=32, ffn=16, num_experts=16, topk=9), 'topk'), (dict(hidden=32, ffn=16, num_experts=4, topk=0), 'topk'),
    (dict(hidden=32, ffn=16, num_experts=2, topk=3), 'topk'), (dict(hidden=8, ffn=8, num_experts=513, topk=2), 'experts'),
    (dict(hidden=8, ffn=8, num_experts=0, topk=1), 'experts'), (dict(hidden=36, ffn=16, num_experts=4), 'hidden'),
    (dict(hidden=32, ffn=12, num_experts=4), 'ffn'), (dict(hidden=0, ffn=16, num_experts=4), 'hidden'),
])
def test_refused(sizes, words):
    with pytest.raises(ValueError, match=words):
        GroupedMoE(device='cpu', **sizes)


@pytest.mark.parametrize('sizes', [dict(hidden=8, ffn=8, num_experts=1, topk=1), dict(hidden=8, ffn=8, num_experts=512, topk=8),
                                   dict(hidden=24, ffn=40, num_experts=3, topk=3)])
def test_taken(sizes):
    layer = GroupedMoE(device='cpu', **sizes)
    assert layer.w_gate_up.shape == (sizes['num_experts'], 2 * sizes['ffn'], sizes['hidden'])
    assert GroupedMoE(device='cpu', dtype=torch.float32, **sizes).bfloat16().w_down.dtype == torch.bfloat16
