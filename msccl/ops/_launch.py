"""What the expert-layer operators share: element types, argument checks, and the device and stream of a call."""
import contextlib

import torch

ELEMS = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}        # ElemType of csrc/expert_ops.h


@contextlib.contextmanager
def _elsewhere(device, stream):
    with torch.cuda.device(device):
        if stream is None:
            yield
        else:
            with torch.cuda.stream(stream):
                yield


_HERE = contextlib.nullcontext()


def on_stream(device, stream, *tensors):
    """Context in which a call on tensors of ``device`` allocates and launches: that device is current and, with ``stream``,
    that stream too.  ``tensors`` then stay allocated until the work on ``stream`` that was queued meanwhile is done."""
    if stream is None:
        return _HERE if torch.cuda.current_device() == device.index else _elsewhere(device, None)
    if stream.device != device:
        raise ValueError(f'the stream belongs to {stream.device}, the tensors to {device}')
    for t in tensors:
        t.record_stream(stream)
    return _elsewhere(device, stream)


def stream_handle():
    return torch.cuda.current_stream().cuda_stream


def check(condition, message):
    if not condition:
        raise ValueError(message)


def check_matrix(t, name, dtypes, unit, dims=2):
    """``t`` has ``dims`` dimensions, its rows are contiguous, start on 16-byte boundaries and hold a multiple of ``unit`` elements.
    A stride that no index uses (one row, one matrix) may have any value."""
    check(t.dtype in dtypes, f'{name} must be {" or ".join(str(d) for d in dtypes)} (got {t.dtype})')
    check(t.dim() == dims, f'{name} must have {dims} dimensions (got {t.dim()})')
    check(t.shape[-1] > 0 and t.shape[-1] % unit == 0, f'the last dimension of {name} must be a positive multiple of {unit} (got {t.shape[-1]})')
    check(t.stride(-1) == 1, f'the rows of {name} must be contiguous')
    step = 16 // t.element_size()
    inner = t.shape[-1]
    for d in range(dims - 2, -1, -1):
        check(t.shape[d] <= 1 or t.stride(d) % step == 0 and t.stride(d) >= inner,
              f'the strides of {name} must be multiples of 16 bytes and its rows must not overlap (stride {t.stride(d)})')
        inner = max(inner, t.stride(d) * t.shape[d] if t.shape[d] > 1 else inner)
    check(t.data_ptr() % 16 == 0, f'{name} must start on a 16-byte boundary')


def check_offsets(offsets, experts):
    check(offsets.dtype == torch.int32 and offsets.shape == (experts + 1,) and offsets.is_contiguous(),
          f'offsets must be a contiguous [{experts + 1}] int32 tensor (got {list(offsets.shape)} {offsets.dtype})')


def check_devices(**tensors):
    """All tensors (``None`` ones apart) are on one CUDA device; returns it."""
    device = None
    for name, t in tensors.items():
        if t is None:
            continue
        check(t.is_cuda, f'{name} must be a CUDA tensor')
        check(device is None or t.device == device, f'{name} is on {t.device}, the other tensors on {device}')
        device = t.device
    return device


def check_apart(out, **inputs):
    """``out`` shares no memory with an input."""
    lo, hi = span(out)
    for name, t in inputs.items():
        a, b = span(t)
        check(b <= lo or hi <= a, f'out overlaps {name}')


def span(t):
    """First and last byte address (exclusive) of a tensor with non-negative strides."""
    if t.numel() == 0:
        return t.data_ptr(), t.data_ptr()
    return t.data_ptr(), t.data_ptr() + t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))


def pitch(t):
    """Row stride in elements; that of a matrix with one row is its length."""
    return t.stride(-2) if t.shape[-2] > 1 else t.shape[-1]


def error_words(device):
    """The words in which the GEMM kernels of ``device`` report a wait that ran out (``check_gemm_errors``)."""
    from msccl.ops import gemm
    if device.index not in gemm._error_words and torch.cuda.is_current_stream_capturing():
        raise RuntimeError('call a GEMM of this package once on the device before capturing one into a graph')
    return gemm._errors(device).data_ptr()
