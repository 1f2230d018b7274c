"""Products in 8-bit floating point (e4m3) with fp32 scales: one per 128 values of an activation row, one per 128 x 128 values of a
weight (``csrc/fp8_block_gemm.cu``, ``csrc/quantize_block.cu``).  Weights are quantised once, activations per call:

    wq, ws = quantize_fp8_block_weight(w)                 # w [n, k], or [experts, n, k]
    xq, xs = quantize_fp8_block(x)                        # x [rows, k]
    y = gemm_fp8_block(xq, xs, wq, ws)                    # bf16 [rows, n]
    y = grouped_gemm_fp8_block(xq, xs, wq, ws, offsets)   # rows of expert e: offsets[e] .. offsets[e + 1]

Beside the MX format of ``msccl.ops.gemm`` (a power of two per 32 values, applied inside the tensor core) these scales are any
fp32 numbers, the form in which block-quantised checkpoints come.  (The scales of an activation and of a weight are multiplied with each
other first: that product has to be a normal fp32 number.)  There are no gradients: this is the path for serving.
"""
import torch
from torch.autograd.graph import increment_version

from msccl.ops._launch import (ELEMS, check, check_apart, check_devices, check_matrices, check_matrix, check_offsets, check_sizes, error_words,
                               on_stream, stream_handle)
from msccl.ops.moe_rows import MAX_EXPERTS
from msccl.runtime.native import load

BLOCK = 128
_E4M3 = torch.float8_e4m3fn


def _blocks(size):
    return -(-size // BLOCK)


def _weight(w, dtypes):
    """Matrices, rows, columns, row stride and matrix stride of a [n, k] or [experts, n, k] weight."""
    if w.dim() == 3:
        return check_matrices(w, 'w', dtypes, 16)
    n, k, pitch = check_matrix(w, 'w', dtypes, 16)
    return 1, n, k, pitch, n * pitch


def quantize_fp8_block(x, stream=None):
    """``x`` [rows, k] fp32, bf16 or fp16 (k a multiple of 16) -> ``(q, scales)``: e4m3 [rows, k] and float32 [rows, ceil(k / 128)].
    ``scale = max(largest magnitude, 2 ** -100) / 448`` over the block, ``q = e4m3(x / scale)``, each rounded once.  The scales
    of neighbouring rows lie next to each other in memory, as the product reads them.  A NaN or an infinity makes its block NaN
    (or zero beside an infinity)."""
    rows, k, pitch = check_matrix(x, 'x', ELEMS, 16)
    index = check_devices('x', x)
    with on_stream(index, stream, (x,)):
        q = torch.empty((rows, k), dtype=_E4M3, device=x.device)
        scales = torch.empty((_blocks(k), rows), dtype=torch.float32, device=x.device).t()
        if rows:
            load().quantize_rows(x.data_ptr(), pitch, q.data_ptr(), scales.data_ptr(), 1, rows, rows, k, ELEMS[x.dtype], stream_handle(index))
    return q, scales


def quantize_fp8_block_weight(w, stream=None):
    """``w`` [n, k] or [experts, n, k] -> e4m3 of the same shape and float32 scales [.., ceil(n / 128), ceil(k / 128)], by the rule of
    ``quantize_fp8_block`` over blocks of 128 x 128."""
    check(w.dim() in (2, 3), f'w must be [n, k] or [experts, n, k] (got {w.dim()} dimensions)')
    experts, n, k, pitch, between = _weight(w, ELEMS)
    check(w.numel() > 0, 'w is empty')
    index = check_devices('w', w)
    check(experts <= 65535, f'at most 65535 matrices at once (got {experts})')
    with on_stream(index, stream, (w,)):
        q = torch.empty(w.shape, dtype=_E4M3, device=w.device)
        scales = torch.empty(*w.shape[:-2], _blocks(n), _blocks(k), dtype=torch.float32, device=w.device)
        load().quantize_blocks(w.data_ptr(), pitch, between, q.data_ptr(), scales.data_ptr(), experts, n, k,
                               ELEMS[w.dtype], stream_handle(index))
    return q, scales


def dequantize_fp8_block(q, scales):
    """fp32 values of a ``quantize_fp8_block`` or ``quantize_fp8_block_weight`` pair (on any device)."""
    s = scales.repeat_interleave(BLOCK, -1)[..., :q.shape[-1]]
    if scales.shape[-2] != q.shape[-2]:
        s = s.repeat_interleave(BLOCK, -2)[..., :q.shape[-2], :]
    return q.float() * s


def _tile_columns(rows, groups, n):
    """The widest tiles of which there are about as many as SMs.  16 x 4096 x 14336: 32 columns 25 us (128 tiles), 64 columns 27, 128
    columns 34; 16 x 14336 x 4096: 128 columns 22.5 (112 tiles), 64 columns 22.6, 32 columns 28."""
    row_tiles = rows // 128 + min(rows, groups)
    for bn in (128, 64):
        if row_tiles * -(-n // bn) >= 100:
            return bn
    return 32


def _product(a, sa, w, sw, offsets, out, stream, dims):
    check(w.dim() == dims, f'w must have {dims} dimensions (got {w.dim()})')
    groups, n, k, w_pitch, w_stride = _weight(w, (_E4M3,))
    if n <= 0 or n % 8:
        raise ValueError(f'the rows of a weight must be a positive multiple of 8 (got {n})')
    rows, columns, a_pitch = check_matrix(a, 'a', (_E4M3,), 16)
    if columns != k:
        raise ValueError(f'inner dimensions differ (a {columns}, w {k})')
    check_sizes(rows, n, k)
    k_blocks = _blocks(k)
    if sa.dtype != torch.float32 or sa.shape != (rows, k_blocks):
        raise ValueError(f'the scales of a must be float32 [{rows}, {k_blocks}] (got {sa.dtype} {list(sa.shape)})')
    want = (_blocks(n), k_blocks) if dims == 2 else (groups, _blocks(n), k_blocks)
    if sw.dtype != torch.float32 or sw.shape != want or not sw.is_contiguous():
        raise ValueError(f'the scales of w must be contiguous float32 {list(want)} (got {sw.dtype} {list(sw.shape)})')
    if offsets is not None:
        if not 1 <= groups <= MAX_EXPERTS:
            raise ValueError(f'between 1 and {MAX_EXPERTS} experts are supported (got {groups})')
        check_offsets(offsets, groups)
    out_pitch = n
    if out is not None:
        *shape, out_pitch = check_matrix(out, 'out', (torch.bfloat16,), 8)
        check(shape == [rows, n], f'out must be [{rows}, {n}] (got {shape})')
        check_apart(out, a=a, sa=sa, w=w, sw=sw)
    index = check_devices('a sa w sw offsets out', a, sa, w, sw, offsets, out)
    with on_stream(index, stream, (a, sa, w, sw, offsets, out)):
        zero_rest = out is None and offsets is not None
        if out is None:
            out = torch.empty((rows, n), dtype=torch.bfloat16, device=a.device)
        else:
            increment_version(out)
        if rows:
            load().fp8_block_gemm(a.data_ptr(), a_pitch, sa.data_ptr(), *sa.stride(), w.data_ptr(), w_pitch, w_stride, sw.data_ptr(),
                                  0 if offsets is None else offsets.data_ptr(), out.data_ptr(), out_pitch, rows, groups, n, k,
                                  _tile_columns(rows, groups, n), rows <= 32, zero_rest, error_words(index), stream_handle(index))
    return out


def gemm_fp8_block(a, sa, w, sw, out=None, stream=None):
    """bf16 [rows, n] = dequant(a) @ dequant(w).T, sums in fp32.  ``a`` [rows, k] with ``sa`` [rows, ceil(k / 128)] (any strides) from
    ``quantize_fp8_block``; ``w`` [n, k] with ``sw`` from ``quantize_fp8_block_weight``; k a multiple of 16, n of 8."""
    return _product(a, sa, w, sw, None, out, stream, 2)


def grouped_gemm_fp8_block(a, sa, w, sw, offsets, out=None, stream=None):
    """The same with a weight for each expert: rows ``offsets[e] .. offsets[e + 1]`` times ``w[e]``.  ``offsets`` and rows of no expert
    as in ``msccl.ops.grouped``."""
    check(offsets is not None, 'offsets are needed')
    return _product(a, sa, w, sw, offsets, out, stream, 3)
