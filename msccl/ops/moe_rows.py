"""Rows around the experts of a MoE layer on one GPU: token copies sorted by expert, their rows gathered, the experts' results
combined (``csrc/moe_rows.cu``).  Unlike ``FusedMoE``, which exchanges rows between GPUs inside its GEMM kernels, there is no
capacity, and ``gather_rows`` and ``combine_rows`` have gradients.

    order = sort_copies(experts, num_experts)             # experts [tokens, k], as the router chose them
    xs = gather_rows(x, order)                            # [tokens * k, hidden], rows of expert e: order.offsets[e] .. [e + 1]
    ys = grouped_gemm(xs, w, order.offsets)
    y = combine_rows(ys, weights, order)                  # y[t] = sum_j weights[t, j] * (result of copy j of token t)
"""
from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from msccl.ops._launch import ELEMS, check_devices, check_matrix, differentiated, on_stream, pitch, stream_handle
from msccl.runtime.native import load

MAX_EXPERTS, MAX_TOPK, MAX_COPIES = 512, 8, 1 << 22
_INT32 = torch.int32


class CopyOrder(NamedTuple):
    """``sorted_copy`` [tokens * k] int32: copies (``token * k + j``) ordered by expert, equal ones by number, dropped ones last.
    ``offsets`` [num_experts + 1] int32: the rows of each expert; rows from ``offsets[-1]`` on belong to dropped copies.
    ``position`` [tokens, k] int32: the row of each copy.  The tensors are made by ``sort_copies`` and are not to be changed.
    (One that was changed gives wrong rows, but none outside the operands is read or written.)"""
    sorted_copy: torch.Tensor
    offsets: torch.Tensor
    position: torch.Tensor


def sort_copies(experts, num_experts, stream=None):
    """Stable order of the copies ``experts`` [tokens, k] (int32 or int64) by expert, in one launch (two
    with more than 32768 copies).  A copy whose id is outside
    ``[0, num_experts)`` is dropped: the gather gives it a row of zeros behind the last expert's, the combination ignores it."""
    if experts.dim() != 2 or experts.dtype not in (torch.int32, torch.int64):
        raise ValueError('experts must be a [tokens, k] int32 or int64 tensor')
    tokens, topk = experts.shape
    copies = tokens * topk
    if tokens < 1 or not 1 <= topk <= MAX_TOPK or copies > MAX_COPIES:
        raise ValueError(f'sort_copies needs at least one token, k <= {MAX_TOPK} and at most {MAX_COPIES} copies (got {tokens} x {topk})')
    if not 1 <= num_experts <= MAX_EXPERTS:
        raise ValueError(f'num_experts must be within 1 and {MAX_EXPERTS} (got {num_experts})')
    index = check_devices('experts', experts)
    with on_stream(index, stream, (experts,)):
        experts = experts.contiguous()
        native = load()
        workspace = native.sort_copies_workspace(copies, num_experts) if copies > 1024 else 0
        table = torch.empty(2 * copies + num_experts + 1, dtype=torch.int32, device=experts.device)
        sorted_copy, position, offsets = table.split((copies, copies, num_experts + 1))
        counts = torch.empty(workspace, dtype=torch.int32, device=experts.device) if workspace else None     # alive until the launch
        native.sort_copies(experts.data_ptr(), experts.dtype == torch.int64, copies, num_experts, sorted_copy.data_ptr(),
                           offsets.data_ptr(), position.data_ptr(), 0 if counts is None else counts.data_ptr(), stream_handle(index))
    return CopyOrder(sorted_copy, offsets, position.view(tokens, topk))


def _check_rows(t, name):
    check_matrix(t, name, ELEMS, 4 if t.dtype == torch.float32 else 8)


def _check_order(order):
    """Tokens and copies of each."""
    sorted_copy, offsets, position = order
    copies = position.numel()
    if (position.dim() == 2 and position.dtype == _INT32 and position.is_contiguous() and sorted_copy.numel() == copies and 1 <= copies <= MAX_COPIES
            and offsets.dim() == 1 and offsets.dtype == _INT32 and offsets.is_contiguous() and offsets.numel() > 1):
        tokens, topk = position.shape
        if topk <= MAX_TOPK:
            return tokens, topk
    raise ValueError('order must be as sort_copies makes it, and whole: contiguous int32 position [tokens, k] (got '
                     f'{position.dtype} {list(position.shape)}), {copies} sorted copies (got {sorted_copy.numel()}) and offsets [experts + 1] (got '
                     f'{offsets.dtype} {list(offsets.shape)})')


def _rows_kept(order):
    return order.offsets.data_ptr() + 4 * (order.offsets.numel() - 1)


def _scatter(x, order):
    tokens, topk = order.position.shape
    out = torch.empty(tokens * topk, x.shape[1], dtype=x.dtype, device=x.device)
    load().scatter_rows(x.data_ptr(), pitch(x), out.data_ptr(), order.position.data_ptr(), _rows_kept(order), tokens, topk, x.shape[1],
                        ELEMS[x.dtype], stream_handle(x.get_device()))
    return out


def _combine(ys, weights, order):
    tokens, topk = order.position.shape
    out = torch.empty(tokens, ys.shape[1], dtype=ys.dtype, device=ys.device)
    load().combine_rows(ys.data_ptr(), pitch(ys), 0 if weights is None else weights.data_ptr(), out.data_ptr(), order.position.data_ptr(),
                        _rows_kept(order), tokens, topk, ys.shape[1], ELEMS[ys.dtype], stream_handle(ys.get_device()))
    return out


def _kernel_rows(t, dtype):
    """``t`` as the kernels take it (``check_matrix``, ``check_matrices``), copied if need be.  An incoming gradient may be an expanded or
    otherwise strided tensor, with rows that overlap; a saved operand may have been unpacked by a hook into any layout."""
    if t.dtype != dtype:
        t = t.to(dtype)
    if t.is_contiguous() and not t.data_ptr() % 16:          # the usual case; the columns are whole units
        return t
    unit = 16 // t.element_size()
    stride, extent = t.stride(), t.shape[-1]
    good = stride[-1] == 1
    for dim in range(t.dim() - 2, -1, -1):
        step = stride[dim] if t.shape[dim] > 1 else extent
        good = good and step >= extent and not step % unit
        extent = (t.shape[dim] - 1) * step + extent
    if not good:
        t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


class _Gather(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, order):
        ctx.order, ctx.dtype = order, x.dtype
        return _scatter(x, order)

    @staticmethod
    @once_differentiable
    def backward(ctx, dxs):
        with on_stream(dxs.get_device(), None):
            return _combine(_kernel_rows(dxs, ctx.dtype), None, ctx.order), None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ys, weights, order):
        ctx.order = order
        ctx.save_for_backward(ys, weights)
        return _combine(ys, weights, order)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        ys, weights = ctx.saved_tensors
        order = ctx.order
        tokens, topk = order.position.shape
        with on_stream(dy.get_device(), None):
            dy, ys, weights = _kernel_rows(dy, ys.dtype), _kernel_rows(ys, ys.dtype), weights.contiguous()
            dys = torch.empty(ys.shape, dtype=ys.dtype, device=ys.device) if ctx.needs_input_grad[0] else None
            dweights = torch.empty(weights.shape, dtype=weights.dtype, device=ys.device) if ctx.needs_input_grad[1] else None
            load().combine_backward(dy.data_ptr(), pitch(dy), ys.data_ptr(), pitch(ys), weights.data_ptr(),
                                    0 if dys is None else dys.data_ptr(), 0 if dweights is None else dweights.data_ptr(),
                                    order.position.data_ptr(), _rows_kept(order), tokens, topk, ys.shape[1], ELEMS[ys.dtype],
                                    stream_handle(ys.get_device()))
        return dys, dweights, None


def gather_rows(x, order, stream=None):
    """``xs[order.position[t, j]] = x[t]``: the row of every copy, ordered by expert; zeros in the rows of dropped copies.
    ``x`` [tokens, hidden] fp32, bf16 or fp16, rows of whole 16-byte units.  The gradient of a token is the sum of its copies'
    (fp32, in the order of ``j``, rounded once)."""
    _check_rows(x, 'x')
    tokens, _ = _check_order(order)
    if x.shape[0] != tokens:
        raise ValueError(f'x has {x.shape[0]} rows, the order {tokens} tokens')
    index = check_devices('x order.position order.offsets', x, order.position, order.offsets)
    with on_stream(index, stream, (x, order.position, order.offsets)):
        return _Gather.apply(x, order) if differentiated(x) else _scatter(x, order)


def combine_rows(ys, weights, order, stream=None):
    """``y[t] = sum_j weights[t, j] * ys[order.position[t, j]]`` over the copies that were not dropped (those are not even read);
    fp32 sums in the order of ``j``, rounded once.  ``ys`` [tokens * k, hidden] fp32, bf16 or fp16, ``weights`` [tokens, k] fp32.
    Gradients: ``ys`` and ``weights`` (zero for dropped copies)."""
    _check_rows(ys, 'ys')
    tokens, topk = _check_order(order)
    if ys.shape[0] != tokens * topk:
        raise ValueError(f'ys has {ys.shape[0]} rows, the order {tokens * topk} copies')
    if weights.dtype != torch.float32 or weights.shape != (tokens, topk):
        raise ValueError(f'weights must be a [{tokens}, {topk}] float32 tensor')
    index = check_devices('ys weights order.position order.offsets', ys, weights, order.position, order.offsets)
    with on_stream(index, stream, (ys, weights, order.position, order.offsets)):
        weights = weights.contiguous()
        return _Combine.apply(ys, weights, order) if differentiated(ys, weights) else _combine(ys, weights, order)
