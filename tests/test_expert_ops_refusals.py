"""What the expert-layer operators refuse, before anything is launched: on CPU tensors, the last of their checks being the device."""
import pytest
import torch

from msccl.ops.fp8_block import (dequantize_fp8_block, gemm_fp8_block, grouped_gemm_fp8_block, quantize_fp8_block,
                                 quantize_fp8_block_weight)
from msccl.ops.grad_norm import _same_dense_layout, clip_grad_norm, grad_norm
from msccl.ops.grouped import grouped_gemm, grouped_gemm_dgrad, grouped_gemm_wgrad
from msccl.ops.moe_rows import CopyOrder, combine_rows, gather_rows, sort_copies

BF16, F8 = torch.bfloat16, torch.float8_e4m3fn


def _refused(call, words):
    with pytest.raises(ValueError, match=words):
        call()


def _z(*shape, dtype=BF16):
    return torch.zeros(*shape, dtype=dtype)


OFFSETS = torch.zeros(4, dtype=torch.int32)


@pytest.mark.parametrize('x,w,offsets,words', [
    (_z(5, 16), _z(3, 8, 16, dtype=torch.float32), OFFSETS, 'w must be'),
    (_z(5, 16, dtype=torch.float16), _z(3, 8, 16), OFFSETS, 'x must be'),
    (_z(5, 16), _z(8, 16), OFFSETS, 'dimensions'),
    (_z(5, 24), _z(3, 8, 16), OFFSETS, 'columns'),
    (_z(5, 12), _z(3, 8, 12), OFFSETS, 'multiple of 8'),
    (_z(5, 16), _z(3, 12, 16), OFFSETS, 'multiples of 8'),
    (_z(5, 16), _z(3, 0, 16), OFFSETS, 'multiples of 8'),
    (_z(16, 5).t(), _z(3, 8, 16), OFFSETS, 'contiguous'),
    (_z(5, 20)[:, :16], _z(3, 8, 16), OFFSETS, '16 bytes'),
    (_z(5, 24)[:, 4:20], _z(3, 8, 16), OFFSETS, 'boundary'),
    (_z(1, 16).expand(5, 16), _z(3, 8, 16), OFFSETS, 'overlap'),
    (_z(5, 16), _z(1, 8, 16).expand(3, 8, 16), OFFSETS, 'overlap'),
    (_z(5, 16), _z(3, 8, 16), OFFSETS.long(), 'offsets'),
    (_z(5, 16), _z(3, 8, 16), OFFSETS[:3], 'offsets'),
    (_z(5, 16), _z(3, 8, 16), torch.zeros(8, dtype=torch.int32)[::2], 'offsets'),
    (_z(5, 16), _z(513, 8, 16), torch.zeros(514, dtype=torch.int32), 'experts'),
    (_z(5, 16), _z(3, 8, 16), OFFSETS, 'CUDA'),
])
def test_grouped_gemm(x, w, offsets, words):
    _refused(lambda: grouped_gemm(x, w, offsets), words)


def test_grouped_gemm_results_and_gradients():
    x, w = _z(5, 16), _z(3, 8, 16)
    _refused(lambda: grouped_gemm(x, w, OFFSETS, out=_z(5, 16)), 'out must be')
    _refused(lambda: grouped_gemm(x, w, OFFSETS, out=_z(5, 8, dtype=torch.float32)), 'out must be')
    _refused(lambda: grouped_gemm_dgrad(_z(5, 16), _z(3, 16, 16), OFFSETS, out=_z(6, 16)[:5, :].t()[:, :5]), 'contiguous|out must|multiple')
    square = _z(5, 16)
    _refused(lambda: grouped_gemm(square, _z(3, 16, 16), OFFSETS, out=square), 'overlaps')
    _refused(lambda: grouped_gemm_dgrad(_z(5, 16), w, OFFSETS), 'columns')
    _refused(lambda: grouped_gemm_wgrad(_z(5, 8), _z(4, 16), OFFSETS), 'rows')
    _refused(lambda: grouped_gemm_wgrad(_z(5, 8), x, OFFSETS, dtype=torch.float16), 'asked for')
    _refused(lambda: grouped_gemm_wgrad(_z(5, 8), x, OFFSETS, out=_z(3, 8, 16), dtype=torch.float32), 'type asked for')
    _refused(lambda: grouped_gemm_wgrad(_z(5, 8), x, OFFSETS, out=_z(3, 16, 8)), 'out must be')
    _refused(lambda: grouped_gemm_wgrad(_z(5, 8), x, OFFSETS[:1]), 'experts')
    _refused(lambda: grouped_gemm_wgrad(_z(5, 8), x, OFFSETS), 'CUDA')


def test_sizes_beyond_the_index_arithmetic():
    rows = (1 << 30) + 8
    x = torch.empty(rows, 16, dtype=BF16, device='meta')
    _refused(lambda: grouped_gemm(x, _z(3, 8, 16), OFFSETS), 'limited')
    _refused(lambda: grouped_gemm_wgrad(x, x, OFFSETS), 'limited')
    a = torch.empty(rows, 16, dtype=F8, device='meta')
    _refused(lambda: gemm_fp8_block(a, torch.zeros(rows, 1, device='meta'), _z(8, 16, dtype=F8), torch.zeros(1, 1)), 'limited')


def _order(tokens, topk):
    return CopyOrder(torch.zeros(tokens * topk, dtype=torch.int32), torch.zeros(5, dtype=torch.int32), torch.zeros(tokens, topk, dtype=torch.int32))


def test_rows():
    ids = torch.zeros(3, 2, dtype=torch.int64)
    for bad, words in ((ids.float(), 'int32 or int64'), (ids.view(-1), 'tokens, k'), (torch.zeros(0, 2, dtype=torch.int64), 'at least one'),
                       (torch.zeros(2, 9, dtype=torch.int64), 'k <= 8'), (torch.zeros(1, dtype=torch.int64).expand((1 << 22) + 1, 1), 'at most'),
                       (ids, 'CUDA')):
        _refused(lambda: sort_copies(bad, 4), words)
    _refused(lambda: sort_copies(ids, 0), 'num_experts')
    _refused(lambda: sort_copies(ids, 513), 'num_experts')
    order, weights = _order(3, 2), torch.zeros(3, 2)
    for x, words in ((_z(4, 16), 'tokens'), (_z(3, 12), 'multiple of 8'), (_z(3, 16, dtype=torch.float64), 'must be'), (_z(16, 3).t(), 'contiguous'),
                     (_z(3, 16), 'CUDA')):
        _refused(lambda: gather_rows(x, order), words)
    for ys, w, words in ((_z(5, 16), weights, 'copies'), (_z(6, 16), weights.double(), 'weights'), (_z(6, 16), weights[:, :1], 'weights'),
                         (_z(6, 6, dtype=torch.float32), weights, 'multiple of 4'), (_z(6, 16), weights, 'CUDA')):
        _refused(lambda: combine_rows(ys, w, order), words)


def test_fp8():
    a, sa, w, sw = _z(5, 144, dtype=F8), torch.zeros(5, 2), _z(40, 144, dtype=F8), torch.zeros(1, 2)
    for call, words in (
            (lambda: gemm_fp8_block(a.view(torch.uint8), sa, w, sw), 'a must be'), (lambda: gemm_fp8_block(a, sa.double(), w, sw), 'scales of a'),
            (lambda: gemm_fp8_block(a, sa[:, :1], w, sw), 'scales of a'), (lambda: gemm_fp8_block(a, sa, w, sw[:, :1]), 'scales of w'),
            (lambda: gemm_fp8_block(a, sa, w, torch.zeros(2, 1).t().expand(1, 2)[:, ::1].half()), 'scales of w'),
            (lambda: gemm_fp8_block(a, sa, w[:, :128], sw), 'inner'), (lambda: gemm_fp8_block(a, sa, w[:36], sw), 'multiple of 8'),
            (lambda: gemm_fp8_block(a[:, :136], sa, w[:, :136], sw), 'multiple of 16'),
            (lambda: gemm_fp8_block(a, sa, w, sw, out=_z(5, 40, dtype=torch.float16)), 'out must be'),
            (lambda: gemm_fp8_block(a, sa, w, sw, out=_z(5, 48)), 'out must be'), (lambda: gemm_fp8_block(a, sa, w[None], sw[None]), 'dimensions'),
            (lambda: gemm_fp8_block(a, sa, w, sw), 'CUDA'),
            (lambda: grouped_gemm_fp8_block(a, sa, w[None], sw[None], OFFSETS), 'offsets'),
            (lambda: grouped_gemm_fp8_block(a, sa, w[None], sw[None], None), 'offsets'),
            (lambda: grouped_gemm_fp8_block(a, sa, w[None], sw, OFFSETS[:2]), 'scales of w'),
            (lambda: grouped_gemm_fp8_block(a, sa, w[None], sw[None], OFFSETS[:2]), 'CUDA'),
            (lambda: quantize_fp8_block(_z(5, 24)), 'multiple of 16'), (lambda: quantize_fp8_block(_z(5, 16, dtype=torch.int8)), 'must be'),
            (lambda: quantize_fp8_block(_z(5, 16)), 'CUDA'), (lambda: quantize_fp8_block_weight(_z(16)), 'n, k'),
            (lambda: quantize_fp8_block_weight(_z(0, 16)), 'empty'), (lambda: quantize_fp8_block_weight(_z(3, 16, 16)), 'CUDA')):
        _refused(call, words)


def test_dequantisation_expands_either_kind_of_scale():
    q = torch.ones(3, 200, 300).to(F8)
    rows = torch.arange(3 * 200 * 3).float().view(3, 200, 3)
    blocks = torch.arange(3 * 2 * 3).float().view(3, 2, 3)
    assert torch.equal(dequantize_fp8_block(q, rows)[1, 150], rows[1, 150].repeat_interleave(128)[:300])
    assert torch.equal(dequantize_fp8_block(q, blocks)[2, :, 299], blocks[2, :, 2].repeat_interleave(128)[:200])


def test_gradient_lists():
    g = torch.zeros(10)
    for call, words in ((lambda: grad_norm([]), 'no gradients'), (lambda: clip_grad_norm([None], 1.0), 'no gradients'),
                        (lambda: clip_grad_norm([g], -1.0), 'max_norm'), (lambda: clip_grad_norm([g], float('nan')), 'max_norm'),
                        (lambda: clip_grad_norm([g], 1.0, out=[g, g]), 'as many'), (lambda: grad_norm([g.double()]), 'float32'),
                        (lambda: clip_grad_norm([g], 1.0, out=[g.long()]), 'output 0'), (lambda: grad_norm([g]), 'CUDA')):
        _refused(call, words)


def test_dense_layouts():
    t = torch.zeros(4, 3, 5)
    assert _same_dense_layout(t, t) and _same_dense_layout(t.permute(2, 0, 1), t.permute(2, 0, 1)) and _same_dense_layout(t[:, :1], t[:, :1]) is False
    assert not _same_dense_layout(t.transpose(0, 1), t.transpose(0, 1).contiguous())
    assert not _same_dense_layout(t[..., :4], t[..., :4]) and not _same_dense_layout(torch.zeros(1).expand(3), torch.zeros(3))
    assert _same_dense_layout(torch.zeros(5, 1, 2)[:, :, :], torch.zeros(5, 1, 2))
