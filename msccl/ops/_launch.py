"""What the expert-layer operators share: element types, argument checks, and the device and stream of a call.

A call on a few tokens takes a handful of microseconds on the GPU, so the checks of a valid call are a few comparisons each;
messages are only put together once one has failed.
"""
import contextlib

import torch
from torch.autograd import forward_ad

ELEMS = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}        # ElemType of csrc/expert_ops.h


@contextlib.contextmanager
def _elsewhere(index, stream):
    with torch.cuda.device(index):
        if stream is None:
            yield
        else:
            with torch.cuda.stream(stream):
                yield


MAX_ROWS = 1 << 30                                      # kMaxRows of csrc/grouped_common.cuh
_HERE = contextlib.nullcontext()
# the public torch.cuda.current_device() and current_stream().cuda_stream give the same numbers in five microseconds more
_current_device = getattr(torch._C, '_cuda_getDevice', None) or torch.cuda.current_device
_raw_stream = getattr(torch._C, '_cuda_getCurrentRawStream', None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def on_stream(index, stream, tensors=()):
    """Context in which a call on tensors of device ``index`` allocates and launches: that device is current and, with ``stream``,
    that stream too.  ``tensors`` (``None`` ones apart) then stay allocated until the work on ``stream`` that was queued
    meanwhile is done."""
    if stream is None:
        return _HERE if _current_device() == index else _elsewhere(index, None)
    if stream.device.index != index:
        raise ValueError(f'the stream belongs to {stream.device}, the tensors to cuda:{index}')
    for t in tensors:
        if t is not None:
            t.record_stream(stream)
    return _elsewhere(index, stream)


def stream_handle(index):
    return _raw_stream(index)


def check(condition, message):
    if not condition:
        raise ValueError(message)


def differentiated(a, b=None):
    """Does autograd follow an operand, backward or forward?  (A tangent is followed without ``requires_grad``, and under ``no_grad`` too.)
    The operators have backward rules only: their autograd functions then raise ``NotImplementedError``."""
    if torch.is_grad_enabled() and (a.requires_grad or (b is not None and b.requires_grad)):
        return True
    if getattr(forward_ad, '_current_level', 0) < 0:        # no forward mode is active: the usual case, for the price of a comparison
        return False
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in (a, b))


def check_matrix(t, name, dtypes, unit):
    """``t`` [rows, columns]: contiguous rows of a multiple of ``unit`` elements that start on 16-byte boundaries and do not overlap.
    Returns rows, columns and the row stride (that of a single row, which no index uses, is its length)."""
    shape, stride, dtype = t.shape, t.stride(), t.dtype
    if dtype in dtypes and len(shape) == 2:
        rows, columns = shape
        pitch = stride[0] if rows > 1 else columns
        if columns > 0 and not columns % unit and stride[1] == 1 and pitch >= columns and not (
                pitch * dtype.itemsize % 16 or t.data_ptr() % 16):
            return rows, columns, pitch
    _refuse(t, name, dtypes, unit, 2)


def check_matrices(t, name, dtypes, unit):
    """``t`` [count, rows, columns]: ``check_matrix`` for each, and matrices that do not overlap.  Returns count, rows, columns, the row
    stride and the matrix stride."""
    shape, stride, dtype = t.shape, t.stride(), t.dtype
    if dtype in dtypes and len(shape) == 3:
        count, rows, columns = shape
        pitch = stride[1] if rows > 1 else columns
        between = stride[0] if count > 1 else rows * pitch
        if columns > 0 and not columns % unit and stride[2] == 1 and pitch >= columns and between >= rows * pitch - (pitch - columns) and not (
                pitch * dtype.itemsize % 16 or between * dtype.itemsize % 16 or t.data_ptr() % 16):
            return count, rows, columns, pitch, between
    _refuse(t, name, dtypes, unit, 3)


def _refuse(t, name, dtypes, unit, dims):
    if t.dtype not in dtypes:
        raise ValueError(f'{name} must be {" or ".join(str(d) for d in dtypes)} (got {t.dtype})')
    if t.dim() != dims:
        raise ValueError(f'{name} must have {dims} dimensions (got {t.dim()})')
    if t.shape[-1] <= 0 or t.shape[-1] % unit:
        raise ValueError(f'the last dimension of {name} must be a positive multiple of {unit} (got {t.shape[-1]})')
    if t.stride(-1) != 1:
        raise ValueError(f'the rows of {name} must be contiguous')
    if t.data_ptr() % 16:
        raise ValueError(f'{name} must start on a 16-byte boundary')
    raise ValueError(f'the strides of {name} must be multiples of 16 bytes and its rows must not overlap (strides {t.stride()})')


def check_sizes(rows, n, k):
    if rows > MAX_ROWS or n > MAX_ROWS or k > MAX_ROWS:
        raise ValueError(f'rows and dimensions of a product are limited to {MAX_ROWS} (got {rows}, {n}, {k})')


def check_offsets(offsets, experts):
    if offsets.dtype != torch.int32 or offsets.shape != (experts + 1,) or offsets.stride(0) != 1:
        raise ValueError(f'offsets must be a contiguous [{experts + 1}] int32 tensor (got {list(offsets.shape)} {offsets.dtype})')


def check_devices(names, *tensors):
    """All tensors (``None`` ones apart) are on one CUDA device; returns its index.  ``names``: theirs, for the message."""
    index = tensors[0].get_device()
    if index < 0 or not tensors[0].is_cuda:
        raise ValueError(f'{names.split()[0]} must be a CUDA tensor')
    for i, t in enumerate(tensors):
        if t is not None and t.get_device() != index:
            raise ValueError(f'{names.split()[i]} is on {t.device}, {names.split()[0]} on cuda:{index}')
    return index


def check_apart(out, **inputs):
    """``out`` shares no memory with an input."""
    lo, hi = span(out)
    for name, t in inputs.items():
        a, b = span(t)
        if lo < b and a < hi:
            raise ValueError(f'out overlaps {name}')


def span(t):
    """First and last byte address (exclusive) of a tensor with non-negative strides."""
    if t.numel() == 0:
        return t.data_ptr(), t.data_ptr()
    return t.data_ptr(), t.data_ptr() + t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))


def pitch(t):
    """Row stride in elements; that of a matrix with one row is its length."""
    return t.stride(-2) if t.shape[-2] > 1 else t.shape[-1]


def matrix_stride(t):
    """Distance between the matrices of a [count, n, k] tensor in elements."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1] * pitch(t)


_words = {}


def error_words(index):
    """Address of the words in which the GEMM kernels of device ``index`` report a wait that ran out (``check_gemm_errors``)."""
    address = _words.get(index)
    if address is None:
        from msccl.ops.gemm import _error_words, _errors
        if index not in _error_words and torch.cuda.is_current_stream_capturing():
            raise RuntimeError('call a GEMM of this package once on the device before capturing one into a graph')
        address = _words[index] = _errors(torch.device('cuda', index)).data_ptr()
    return address
