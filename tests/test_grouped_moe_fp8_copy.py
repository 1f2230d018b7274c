"""The fp8 copy of a ``GroupedMoE`` follows the layer or is gone: on the CPU, with a plain quantisation in place of the kernels."""
import copy
import io

import pytest
import torch

from msccl.parallel import GroupedMoE, grouped_moe


def _plain_quantise(w, stream=None):
    return w.float().to(torch.float8_e4m3fn), torch.ones(*w.shape[:-2], 1, 1)


@pytest.fixture
def layer(monkeypatch):
    monkeypatch.setattr(grouped_moe, 'quantize_fp8_block_weight', _plain_quantise)
    return GroupedMoE(32, 16, 4, 2, device='cpu', std=1.0).quantize()


X = torch.zeros(2, 32, dtype=torch.bfloat16)


def _bytes(layer):
    return [t.view(torch.uint8).clone() for t in layer._fp8]


def _same(a, b):
    return len(a) == len(b) and all(torch.equal(s, t) for s, t in zip(a, b))


def test_loaded_weights_end_the_copy(layer):
    other = GroupedMoE(32, 16, 4, 2, device='cpu', std=1.0, seed=1)
    layer.load_state_dict(other.state_dict())
    with pytest.raises(RuntimeError, match='quantize'):
        layer(X, precision='fp8')
    layer.quantize()
    assert _same(_bytes(layer), _bytes(other.quantize()))


def test_loading_into_a_larger_model_ends_it_too(layer):
    model = torch.nn.Sequential(torch.nn.Linear(2, 2), layer)
    model.load_state_dict({k: torch.zeros_like(v) for k, v in model.state_dict().items()})
    with pytest.raises(RuntimeError, match='quantize'):
        layer(X, precision='fp8')


def test_a_state_without_the_experts_leaves_it(layer):
    before = _bytes(layer)
    layer.load_state_dict({'w_router': torch.zeros_like(layer.w_router)}, strict=False)
    model = torch.nn.Sequential(torch.nn.Linear(2, 2), layer)
    model.load_state_dict({'0.weight': torch.zeros(2, 2), 'w_down': layer.w_down}, strict=False)
    assert _same(_bytes(layer), before)
    layer.load_state_dict({'w_down': torch.zeros_like(layer.w_down)}, strict=False)
    assert layer._fp8 is None


def test_a_move_takes_the_copy_along(layer):
    before = _bytes(layer)
    assert _same(_bytes(layer.cpu()), before) and _same(_bytes(layer.to(torch.bfloat16)), before)
    assert _same(_bytes(torch.nn.Sequential(layer).to('cpu', torch.bfloat16)[0]), before)
    layer.to('meta')                                       # another device, as far as there is one here
    assert all(t.device.type == 'meta' for t in layer._fp8)
    assert [t.dtype for t in layer._fp8] == [torch.float8_e4m3fn, torch.float32] * 2


@pytest.mark.parametrize('convert', [lambda l: l.half(), lambda l: l.float(), lambda l: l.to(torch.float16)])
def test_another_type_ends_it(layer, convert):
    convert(layer)
    with pytest.raises(RuntimeError, match='quantize'):
        layer(X, precision='fp8')


def test_copies_of_the_layer(layer):
    saved = io.BytesIO()
    torch.save(layer, saved)
    saved.seek(0)
    for other in (copy.deepcopy(layer), torch.load(saved, weights_only=False)):
        assert _same(_bytes(other), _bytes(layer))
    assert set(layer.state_dict()) == {'w_router', 'w_gate_up', 'w_down'}
