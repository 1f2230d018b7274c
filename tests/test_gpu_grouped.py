"""Grouped products against 64-bit sums.

Small whole numbers keep every partial sum of fp32 exact (below 2^24), whatever the order, so a result has to be the exact sum
rounded once: indexing, masking and tails are checked bit for bit.  Normal values are checked within half a step of the result's
type plus the fp32 sums' bound, one part in 2^23 of the sum of magnitudes for each addition."""
import pytest
import torch

pytestmark = pytest.mark.gpu

SHAPES = [  # sizes of the groups, rows before the first and behind the last, n, k
    ([1], 0, 0, 8, 8),
    ([0, 5, 0, 0], 0, 0, 256, 64),
    ([0, 0], 0, 3, 64, 64),
    ([33, 0, 31, 1], 0, 0, 264, 72),
    ([64, 128, 65], 2, 7, 128, 136),
    ([100, 200, 0, 300], 0, 0, 520, 1000),
    ([257, 511, 1], 5, 0, 1000, 200),
    ([1] * 70, 0, 0, 40, 512),
    ([900, 2, 1200], 0, 19, 304, 256),
]


def _offsets(sizes, head):
    at = [head]
    for s in sizes:
        at.append(at[-1] + s)
    return at, torch.tensor(at, dtype=torch.int32, device='cuda')


def _whole(gen, *shape, dtype):
    return torch.randint(-3, 4, shape, device='cuda', generator=gen).to(dtype)


def _forward(x, w, at):
    y = torch.zeros(x.shape[0], w.shape[1], dtype=torch.float64, device='cuda')
    for e, (lo, hi) in enumerate(zip(at, at[1:])):
        y[lo:hi] = x[lo:hi].double() @ w[e].double().t()
    return y


def _backward(dy, w, at):
    dx = torch.zeros(dy.shape[0], w.shape[2], dtype=torch.float64, device='cuda')
    for e, (lo, hi) in enumerate(zip(at, at[1:])):
        dx[lo:hi] = dy[lo:hi].double() @ w[e].double()
    return dx


def _weight_gradient(dy, x, at):
    return torch.stack([dy[lo:hi].double().t() @ x[lo:hi].double() for lo, hi in zip(at, at[1:])])


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('sizes,head,tail,n,k', SHAPES)
def test_whole_numbers_are_exact(sizes, head, tail, n, k, dtype):
    from msccl.ops import check_gemm_errors
    from msccl.ops.grouped import grouped_gemm, grouped_gemm_dgrad, grouped_gemm_wgrad
    gen = torch.Generator(device='cuda').manual_seed(n + k)
    at, offsets = _offsets(sizes, head)
    rows, used = at[-1] + tail, slice(head, at[-1])
    x, dy = _whole(gen, rows, k, dtype=dtype), _whole(gen, rows, n, dtype=dtype)
    w = _whole(gen, len(sizes), n, k, dtype=dtype)
    want_y, want_dx, want_dw = _forward(x, w, at), _backward(dy, w, at), _weight_gradient(dy, x, at)
    # what belongs to no group must not be read into any result
    for t in (x, dy):
        t[:head] = float('nan')
        t[at[-1]:] = float('inf')
    for e, s in enumerate(sizes):
        if s == 0:
            w[e] = float('nan')
    y, dx, dw = grouped_gemm(x, w, offsets), grouped_gemm_dgrad(dy, w, offsets), grouped_gemm_wgrad(dy, x, offsets)
    dw32 = grouped_gemm_wgrad(dy, x, offsets, dtype=torch.float32)
    check_gemm_errors()
    assert torch.equal(y, want_y.to(dtype)) and torch.equal(dx, want_dx.to(dtype))
    assert torch.equal(dw, want_dw.to(dtype)) and torch.equal(dw32, want_dw.float())
    # a result that the caller gives: rows of no group and what lies beside it stay as they were
    for f, a, want, columns in ((grouped_gemm, x, want_y, n), (grouped_gemm_dgrad, dy, want_dx, k)):
        holder = torch.full((rows, columns + 16), 7.0, dtype=dtype, device='cuda')
        f(a, w, offsets, out=holder[:, 8:columns + 8])
        assert torch.equal(holder[used, 8:columns + 8], want[used].to(dtype))
        holder[used, 8:columns + 8] = 7.0
        assert torch.all(holder == 7.0)
    check_gemm_errors()


@pytest.mark.parametrize('sizes,head,tail,n,k', [SHAPES[3], SHAPES[5], SHAPES[6]])
def test_strided_operands(sizes, head, tail, n, k):
    """Rows and matrices inside larger ones: NaN between them."""
    from msccl.ops import check_gemm_errors
    from msccl.ops.grouped import grouped_gemm, grouped_gemm_dgrad, grouped_gemm_wgrad
    gen = torch.Generator(device='cuda').manual_seed(3)
    at, offsets = _offsets(sizes, head)
    rows, dtype = at[-1] + tail, torch.bfloat16

    def inside(t):
        big = torch.full([s + 8 for s in t.shape], float('nan'), dtype=dtype, device='cuda')
        view = big[tuple(slice(0, s) for s in t.shape[:-1])][..., 8:]
        view.copy_(t)
        return view
    x, dy = _whole(gen, rows, k, dtype=dtype), _whole(gen, rows, n, dtype=dtype)
    w = _whole(gen, len(sizes), n, k, dtype=dtype)
    xs, dys, ws = inside(x), inside(dy), inside(w)
    assert torch.equal(grouped_gemm(xs, ws, offsets), _forward(x, w, at).to(dtype))
    assert torch.equal(grouped_gemm_dgrad(dys, ws, offsets), _backward(dy, w, at).to(dtype))
    out = torch.full((len(sizes), n + 3, k + 8), 7.0, dtype=dtype, device='cuda')
    grouped_gemm_wgrad(dys, xs, offsets, out=out[:, :n, :k])
    check_gemm_errors()
    assert torch.equal(out[:, :n, :k], _weight_gradient(dy, x, at).to(dtype))
    assert torch.all(out[:, n:] == 7) and torch.all(out[:, :, k:] == 7)


def _within(got, want, magnitudes, terms):
    step = torch.finfo(got.dtype).eps / 2
    smallest = torch.finfo(got.dtype).smallest_normal * step if got.dtype == torch.float16 else 0.0
    assert torch.all((got.double() - want).abs() <= step * want.abs() * (1 + 2.0 ** -8) + terms * 2.0 ** -23 * magnitudes + smallest)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('sizes,n,k', [([3, 0, 40, 700, 90], 392, 1416), ([2000, 1], 256, 4096)])
def test_gradients_against_the_formulas(sizes, n, k, dtype):
    from msccl.ops import check_gemm_errors
    from msccl.ops.grouped import grouped_gemm
    gen = torch.Generator(device='cuda').manual_seed(1)
    at, offsets = _offsets(sizes, 0)
    rows = at[-1]
    x = torch.randn(rows, k, device='cuda', generator=gen).to(dtype).requires_grad_()
    w = (torch.randn(len(sizes), n, k, device='cuda', generator=gen) * 0.05).to(dtype).requires_grad_()
    dy = torch.randn(rows, n, device='cuda', generator=gen).to(dtype)
    y = grouped_gemm(x, w, offsets)
    y.backward(dy)
    check_gemm_errors()
    with torch.no_grad():
        _within(y, _forward(x, w, at), _forward(x.abs(), w.abs(), at), k)
        _within(x.grad, _backward(dy, w, at), _backward(dy.abs(), w.abs(), at), n)
        _within(w.grad, _weight_gradient(dy, x, at), _weight_gradient(dy.abs(), x.abs(), at), max(sizes))
    # an expanded gradient (of a sum) and only one operand that needs a gradient
    x2 = x.detach().requires_grad_()
    grouped_gemm(x2, w.detach(), offsets).sum().backward()
    ones = torch.ones(rows, n, dtype=dtype, device='cuda')
    _within(x2.grad, _backward(ones, w.detach(), at), _backward(ones, w.detach().abs(), at), n)


def test_gradient_is_the_difference_quotient():
    """The product is linear in each operand: f(x + d) - f(x) = <grad, d> for whole numbers, exactly."""
    from msccl.ops.grouped import grouped_gemm
    gen = torch.Generator(device='cuda').manual_seed(5)
    at, offsets = _offsets([17, 0, 50], 0)
    x, w = _whole(gen, 67, 72, dtype=torch.float16).requires_grad_(), _whole(gen, 3, 40, 72, dtype=torch.float16).requires_grad_()
    c = torch.randint(0, 2, (67, 40), device='cuda', generator=gen).half()
    (grouped_gemm(x, w, offsets) * c).sum(dtype=torch.float64).backward()

    def f(a, b):
        return (grouped_gemm(a, b, offsets).double() * c).sum()
    with torch.no_grad():
        for t, other, swap in ((x, w, False), (w, x, True)):
            d = _whole(gen, *t.shape, dtype=torch.float16)
            change = (f(other, t + d) - f(other, t)) if swap else (f(t + d, other) - f(t, other))
            assert change == (t.grad.double() * d.double()).sum()


def test_offsets_that_are_not_sorted_or_leave_the_rows_are_clamped():
    from msccl.ops import check_gemm_errors
    from msccl.ops.grouped import grouped_gemm, grouped_gemm_wgrad
    gen = torch.Generator(device='cuda').manual_seed(2)
    x, w = _whole(gen, 60, 64, dtype=torch.bfloat16), _whole(gen, 4, 64, 64, dtype=torch.bfloat16)
    for raw, meant in (([-5, 10, 4, 70, 1 << 30], [0, 10, 10, 60, 60]), ([50, 20, 20, 20, 55], [50, 50, 50, 50, 55])):
        offsets = torch.tensor(raw, dtype=torch.int32, device='cuda')
        assert torch.equal(grouped_gemm(x, w, offsets), _forward(x, w, meant).bfloat16())
        assert torch.equal(grouped_gemm_wgrad(x, x, offsets), _weight_gradient(x, x, meant).bfloat16())
    check_gemm_errors()


def test_no_rows():
    from msccl.ops.grouped import grouped_gemm, grouped_gemm_dgrad, grouped_gemm_wgrad
    w = torch.randn(3, 16, 24, device='cuda').bfloat16().requires_grad_()
    x = torch.empty(0, 24, device='cuda', dtype=torch.bfloat16).requires_grad_()
    offsets = torch.zeros(4, dtype=torch.int32, device='cuda')
    y = grouped_gemm(x, w, offsets)
    y.sum().backward()
    assert y.shape == (0, 16) and x.grad.shape == (0, 24) and torch.all(w.grad == 0)
    assert grouped_gemm_dgrad(y.detach(), w.detach(), offsets).shape == (0, 24)
    assert torch.all(grouped_gemm_wgrad(y.detach(), x.detach(), offsets) == 0)


def test_captured_and_on_another_stream():
    from msccl.ops import check_gemm_errors
    from msccl.ops.grouped import grouped_gemm, grouped_gemm_dgrad, grouped_gemm_wgrad
    gen = torch.Generator(device='cuda').manual_seed(4)
    x, w, dy = _whole(gen, 300, 128, dtype=torch.bfloat16), _whole(gen, 3, 192, 128, dtype=torch.bfloat16), _whole(gen, 300, 192, dtype=torch.bfloat16)
    at, offsets = _offsets([100, 0, 200], 0)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    y = grouped_gemm(x, w, offsets, stream=stream)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(y, _forward(x, w, at).bfloat16())
    # two graphs with the same inputs, replayed at once on two streams with other group sizes than those they were captured with
    graphs, results = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            results.append((grouped_gemm(x, w, offsets), grouped_gemm_dgrad(dy, w, offsets), grouped_gemm_wgrad(dy, x, offsets)))
        graphs.append(g)
    for sizes in ([300, 0, 0], [1, 150, 60]):
        at, other = _offsets(sizes, 0)
        offsets.copy_(other)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for _ in range(3):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        check_gemm_errors()
        for y, dx, dw in results:
            assert torch.equal(y, _forward(x, w, at).bfloat16())
            assert torch.equal(dx, _backward(dy, w, at).bfloat16())
            assert torch.equal(dw, _weight_gradient(dy, x, at).bfloat16())


@pytest.mark.parametrize('what', ['forward', 'backward'])
def test_first_call_of_a_thread(what):
    """A thread that has made no CUDA call yet, as autograd's are at first (in a process of its own: contexts outlive a test)."""
    import os
    import subprocess
    import sys
    code = """
import sys, threading, torch
from msccl.ops import check_gemm_errors
from msccl.ops.grouped import grouped_gemm
x = torch.randn(64, 64, device='cuda').bfloat16()
w = torch.randn(2, 64, 64, device='cuda').bfloat16()
offsets = torch.tensor([0, 30, 64], dtype=torch.int32, device='cuda')
failed = []
def call():
    try:
        grouped_gemm(x, w, offsets)
    except Exception as e:
        failed.append(e)
if sys.argv[1] == 'forward':
    t = threading.Thread(target=call)
    t.start()
    t.join()
else:
    x.requires_grad_()
    y = grouped_gemm(x, w, offsets)
    torch.autograd.grad(y, x, torch.ones_like(y))
check_gemm_errors()
assert not failed, failed
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, '-c', code, what], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stdout + done.stderr


def test_first_call_inside_a_capture_is_refused():
    import os
    import subprocess
    import sys
    code = """
import torch
from msccl.ops.grouped import grouped_gemm
x, w = torch.randn(8, 64, device='cuda').bfloat16(), torch.randn(1, 64, 64, device='cuda').bfloat16()
offsets = torch.tensor([0, 8], dtype=torch.int32, device='cuda')
try:
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        grouped_gemm(x, w, offsets)
except RuntimeError as e:
    assert 'before capturing' in str(e), e
else:
    raise SystemExit('not refused')
grouped_gemm(x, w, offsets)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = grouped_gemm(x, w, offsets)
graph.replay()
assert torch.equal(y, grouped_gemm(x, w, offsets))
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, '-c', code], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stdout + done.stderr


def test_kernels_skip_after_a_reported_timeout():
    """The error words as a kernel that gave up leaves them: later launches return at once, the check reports and clears."""
    from msccl.ops import GemmKernelError, check_gemm_errors
    from msccl.ops.fp8_block import gemm_fp8_block, quantize_fp8_block, quantize_fp8_block_weight
    from msccl.ops.gemm import _errors
    from msccl.ops.grouped import grouped_gemm, grouped_gemm_dgrad, grouped_gemm_wgrad
    gen = torch.Generator(device='cuda').manual_seed(7)
    x, w = _whole(gen, 100, 64, dtype=torch.bfloat16), _whole(gen, 2, 64, 64, dtype=torch.bfloat16)
    at, offsets = _offsets([30, 70], 0)
    fp8 = (*quantize_fp8_block(x), *quantize_fp8_block_weight(w[0]))
    calls = [(lambda out: grouped_gemm(x, w, offsets, out=out), (100, 64)), (lambda out: grouped_gemm_dgrad(x, w, offsets, out=out), (100, 64)),
             (lambda out: grouped_gemm_wgrad(x, x, offsets, out=out), (2, 64, 64)), (lambda out: gemm_fp8_block(*fp8, out=out), (100, 64))]
    check_gemm_errors()
    for call, shape in calls:
        out = torch.full(shape, 7.0, dtype=torch.bfloat16, device='cuda')
        _errors('cuda:0')[0] = 1
        call(out)
        with pytest.raises(GemmKernelError):
            check_gemm_errors()
        assert torch.all(out == 7.0)
        call(out)
        check_gemm_errors()
        assert not torch.all(out == 7.0)


def test_far_rows():
    """Offsets of elements beyond 2^31: 150000 rows of 16384 columns."""
    from msccl.ops import check_gemm_errors
    from msccl.ops.grouped import grouped_gemm
    gen = torch.Generator(device='cuda').manual_seed(6)
    rows, n, k = 150000, 16384, 64
    x, w = _whole(gen, rows, k, dtype=torch.bfloat16), _whole(gen, 2, n, k, dtype=torch.bfloat16)
    at, offsets = _offsets([140001, 9000], 0)
    y = grouped_gemm(x, w, offsets)
    check_gemm_errors()
    for lo, hi, e in ((0, 64, 0), (139990, 140001, 0), (140001, 140065, 1), (148990, 149001, 1)):
        assert torch.equal(y[lo:hi], (x[lo:hi].double() @ w[e].double().t()).bfloat16())
    assert torch.all(y[149001:] == 0)
