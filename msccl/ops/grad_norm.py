"""Global norm of a list of gradients and their clipping, in two launches whatever the number of tensors up to 1000
(``csrc/grad_norm.cu``).  ``FlatGradients.clip_grad_norm`` calls it on its buckets."""
import math

import torch
from torch.autograd.graph import increment_version

from msccl.ops._launch import ELEMS, check, on_stream, stream_handle
from msccl.runtime.native import load

_DTYPES = tuple(sorted(ELEMS, key=ELEMS.get))


def _same_dense_layout(g, out):
    """Do ``g``'s elements fill one stretch of memory (in any order of the dimensions), and ``out``'s in the same order?"""
    def dims(t):
        return sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1)
    expected = 1
    for stride, size in dims(g):
        if stride != expected:
            return False
        expected *= size
    return g.shape == out.shape and [s for s, n in zip(g.stride(), g.shape) if n != 1] == [s for s, n in zip(out.stride(), out.shape) if n != 1]


def _collect(gradients, out):
    gradients = list(gradients)
    if out is None:
        gradients = [g for g in gradients if g is not None]
    else:
        out = list(out)
        check(len(out) == len(gradients), f'{len(gradients)} gradients need as many outputs (got {len(out)})')
        kept = [(g, o) for g, o in zip(gradients, out) if g is not None]
        gradients, out = [g for g, _ in kept], [o for _, o in kept]
    if not gradients:
        raise ValueError('no gradients')
    return load().GradList(gradients, out, _DTYPES, _same_dense_layout), gradients, out


def grad_norm(gradients, stream=None):
    """The 2-norm over all elements of ``gradients`` (fp32, bf16 or fp16 CUDA tensors of one device, dense in memory; ``None``
    entries are skipped) as a float32 tensor without dimensions.  Sums are formed in fp32 over 16 bytes and in fp64 from there,
    in an order that depends on the sizes only."""
    tensors, gradients, _ = _collect(gradients, None)
    device = gradients[0].device
    with on_stream(device.index, stream, gradients):
        norm = torch.empty((), dtype=torch.float32, device=device)
        if len(tensors) == 0:
            return norm.zero_()
        partials = torch.empty(tensors.partials(), dtype=torch.float64, device=device)
        load().grad_norm(tensors, partials.data_ptr(), stream_handle(device.index))
        load().grad_sum(partials.data_ptr(), partials.numel(), 0, norm.data_ptr(), stream_handle(device.index))
    return norm


def clip_grad_norm(gradients, max_norm, out=None, reduce=None, stream=None):
    """Scale ``gradients`` by ``min(1, max_norm / (norm + 1e-6))`` where ``norm`` is that of ``grad_norm``, and return it.

    In place, or into ``out`` (a tensor for each gradient, of the same size and memory order and any of the three types: the
    bf16 gradients of a step into the fp32 ones of the optimizer).  In place nothing is written on a step that needs no clipping.
    ``reduce(t)`` sums the one-element float64 tensor ``t`` (this process's sum of squares) over the processes that hold the other
    parts of the gradients, in place; gradients that are the same on every rank need none.  An infinite norm gives zeros (and NaN
    where the gradient is infinite; NaN everywhere if ``max_norm`` is infinite too), a NaN gives NaN everywhere.  No tensor may share memory with another one that is written.
    For autograd this is a write under ``no_grad``: a backward pass that needs a written tensor as it was raises."""
    max_norm = float(max_norm)
    check(not math.isnan(max_norm) and max_norm >= 0, f'max_norm must not be negative or NaN (got {max_norm})')
    tensors, gradients, out = _collect(gradients, out)
    if tensors.overlapping():
        raise ValueError('a tensor that is written shares memory with another one')
    device = gradients[0].device
    with on_stream(device.index, stream, gradients + (out or [])):
        norm = torch.empty((), dtype=torch.float32, device=device)
        if len(tensors) == 0 and reduce is None:
            return norm.zero_()
        partials = torch.empty(max(tensors.partials(), 1), dtype=torch.float64, device=device)
        if len(tensors):
            load().grad_norm(tensors, partials.data_ptr(), stream_handle(device.index))
        else:
            partials.zero_()
        increment_version(gradients if out is None else out)
        count = partials.numel()
        if reduce is not None:
            total = torch.empty(1, dtype=torch.float64, device=device)
            load().grad_sum(partials.data_ptr(), count, total.data_ptr(), 0, stream_handle(device.index))
            reduce(total)
            partials, count = total, 1
        if len(tensors):
            load().grad_scale(tensors, partials.data_ptr(), count, max_norm, norm.data_ptr(), stream_handle(device.index))
        else:
            load().grad_sum(partials.data_ptr(), count, 0, norm.data_ptr(), stream_handle(device.index))
    return norm
