"""Matrix products grouped by expert with ragged sizes: the rows of expert ``e`` (``offsets[e] .. offsets[e + 1]`` of a row-sorted
matrix, as ``sort_copies`` gives them) times that expert's weights, forward and both gradients (``csrc/grouped_gemm.cu``,
``csrc/grouped_wgrad.cu``).  Any number of rows per expert, none included; there is no capacity and no padding.

``offsets`` [experts + 1] int32 stays on the device: no call waits for it.  Values are clamped to the rows and to their running
maximum.  Rows that belong to no expert come out as zeros, or, in an ``out`` that the caller gives, are left as they were.  ``out`` may not
reach into the stretch of memory between an input's first and last element.
"""
import torch
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from msccl.ops._launch import (ELEMS, check, check_apart, check_devices, check_matrices, check_matrix, check_offsets, check_sizes, differentiated,
                               error_words, matrix_stride, on_stream, pitch, stream_handle)
from msccl.ops.moe_rows import MAX_EXPERTS, _kernel_rows
from msccl.runtime.native import load

_TYPES = (torch.bfloat16, torch.float16)


def _tile_rows(rows, experts):
    """The most rows of a tile, from the mean size of a group (the sizes themselves are on the device): tiles of 64 leave room for more
    of the weights on their way, tiles of 256 read them less often.  Microseconds with 64 / 256 rows, forward: 32 rows x 8 experts of
    14336 x 4096 165 / 178; 4096 x 64 of 1024 x 2048 71 / 73; 1024 x 8 of 4096 x 4096 81 / 72; 8192 x 8 of 14336 x 4096 1097 / 611."""
    return 64 if rows <= 48 * min(rows, experts) else 256


def _check_experts(experts):
    if not 1 <= experts <= MAX_EXPERTS:
        raise ValueError(f'between 1 and {MAX_EXPERTS} experts are supported (got {experts})')


def _launch(x, w, offsets, out, backward, index, experts, n, k, rows, x_pitch, w_pitch, w_stride):
    """``out`` is None or a pair of a tensor and its row stride."""
    dtype = x.dtype
    if out is None:
        columns = k if backward else n
        result, out_pitch = torch.empty((rows, columns), dtype=dtype, device=x.device), columns
    else:
        result, out_pitch = out
    if rows:
        load().grouped_gemm(x.data_ptr(), x_pitch, w.data_ptr(), w_pitch, w_stride, offsets.data_ptr(), result.data_ptr(), out_pitch, rows,
                            experts, n, k, backward, ELEMS[dtype], _tile_rows(rows, experts), out is None, error_words(index),
                            stream_handle(index))
    return result


def _product(x, w, offsets, backward):
    """The same for operands that have been checked before."""
    experts, n, k = w.shape
    return _launch(x, w, offsets, None, backward, x.get_device(), experts, n, k, x.shape[0], pitch(x), pitch(w), matrix_stride(w))


def _weight_gradient(dy, x, offsets, out=None, dtype=None):
    experts, n, k = offsets.numel() - 1, dy.shape[1], x.shape[1]
    if out is None:
        out = torch.empty(experts, n, k, dtype=dtype or x.dtype, device=x.device)
    else:
        increment_version(out)
    if x.shape[0] == 0:
        return out.zero_()
    index = x.get_device()
    load().grouped_wgrad(dy.data_ptr(), pitch(dy), x.data_ptr(), pitch(x), offsets.data_ptr(), out.data_ptr(), pitch(out), matrix_stride(out),
                         x.shape[0], experts, n, k, ELEMS[x.dtype], out.dtype == torch.float32, error_words(index), stream_handle(index))
    return out


class _Grouped(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, offsets):
        ctx.save_for_backward(x, w, offsets)
        return _product(x, w, offsets, False)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w, offsets = ctx.saved_tensors
        with on_stream(dy.get_device(), None):
            dy, offsets = _kernel_rows(dy, x.dtype), offsets.contiguous()
            dx = _product(dy, _kernel_rows(w, x.dtype), offsets, True) if ctx.needs_input_grad[0] else None
            dw = _weight_gradient(dy, _kernel_rows(x, x.dtype), offsets) if ctx.needs_input_grad[1] else None
        return dx, dw, None


def _checked(x, name, w, offsets, out, backward):
    """Everything that ``_launch`` needs to know of the operands, from ``out`` on."""
    experts, n, k, w_pitch, w_stride = check_matrices(w, 'w', _TYPES, 8)
    width, columns = (n, k) if backward else (k, n)
    _check_experts(experts)
    if n <= 0 or n % 8:
        raise ValueError(f'both dimensions of a weight must be positive multiples of 8 (got {n})')
    rows, x_columns, x_pitch = check_matrix(x, name, (w.dtype,), 8)
    if x_columns != width:
        raise ValueError(f'{name} has {x_columns} columns, the weights expect {width}')
    check_sizes(rows, n, k)
    check_offsets(offsets, experts)
    target = None
    if out is not None:
        *shape, out_pitch = check_matrix(out, 'out', (w.dtype,), 8)
        check(shape == [rows, columns], f'out must be [{rows}, {columns}] (got {shape})')
        check_apart(out, **{name: x, 'w': w})
        target = (out, out_pitch)
    index = check_devices(f'{name} w offsets out', x, w, offsets, out)
    return target, backward, index, experts, n, k, rows, x_pitch, w_pitch, w_stride


def grouped_gemm(x, w, offsets, out=None, stream=None):
    """``y[t] = w[e] @ x[t]`` for the rows ``t`` of every expert ``e``: ``x`` [rows, k], ``w`` [experts, n, k] (both bf16 or both fp16,
    n and k multiples of 8, rows contiguous), result [rows, n] of the same type, fp32 sums.  Differentiable in ``x`` and ``w``; with
    ``out`` the result has no gradient."""
    known = _checked(x, 'x', w, offsets, out, False)
    if differentiated(x, w):
        check(out is None, 'a result written to out has no gradient: detach x and w, or leave out away')
        with on_stream(known[2], stream, (x, w, offsets)):
            return _Grouped.apply(x, w, offsets)
    with on_stream(known[2], stream, (x, w, offsets, out)):
        if out is not None:
            increment_version(out)
        return _launch(x, w, offsets, *known)


def grouped_gemm_dgrad(dy, w, offsets, out=None, stream=None):
    """``dx[t] = w[e].T @ dy[t]``: ``dy`` [rows, n], ``w`` [experts, n, k], result [rows, k].  No gradient of its own."""
    known = _checked(dy, 'dy', w, offsets, out, True)
    with on_stream(known[2], stream, (dy, w, offsets, out)):
        if out is not None:
            increment_version(out)
        return _launch(dy, w, offsets, *known)


def grouped_gemm_wgrad(dy, x, offsets, out=None, dtype=None, stream=None):
    """``dw[e] = sum of outer(dy[t], x[t])`` over the rows of expert ``e`` (zeros where it has none): ``dy`` [rows, n], ``x``
    [rows, k], result [experts, n, k] of their type or, with ``dtype=torch.float32`` (or such an ``out``), the fp32 sums."""
    rows, k, _ = check_matrix(x, 'x', _TYPES, 8)
    dy_rows, n, _ = check_matrix(dy, 'dy', (x.dtype,), 8)
    check(rows == dy_rows, f'dy has {dy_rows} rows, x {rows}')
    check_sizes(rows, n, k)
    experts = offsets.numel() - 1
    _check_experts(experts)
    check_offsets(offsets, experts)
    check(dtype in (None, x.dtype, torch.float32), f'the gradient is {x.dtype} or float32 (asked for {dtype})')
    if out is not None:
        shape = check_matrices(out, 'out', (x.dtype, torch.float32), 8)[:3]
        check(shape == (experts, n, k) and dtype in (None, out.dtype), f'out must be [{experts}, {n}, {k}] of the type asked for')
        check_apart(out, dy=dy, x=x)
    index = check_devices('dy x offsets out', dy, x, offsets, out)
    with on_stream(index, stream, (dy, x, offsets, out)):
        return _weight_gradient(dy, x, offsets, out, dtype)
