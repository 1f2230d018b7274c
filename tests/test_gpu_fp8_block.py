"""Block-scaled fp8 with fp32 scales: the quantisation byte for byte against its definition, products against 64-bit sums.

Whole numbers of e4m3 with power-of-two scales keep every fp32 sum exact, so those results are the exact sum rounded once."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _definition(x, block_rows):
    n, k = x.shape[-2:]
    padded = torch.nn.functional.pad(x.float(), (0, -k % 128, 0, -n % block_rows))
    b = padded.view(*x.shape[:-2], padded.shape[-2] // block_rows, block_rows, -1, 128)
    largest = b.abs().amax((-3, -1), keepdim=True).clamp_min(2.0 ** -100)
    scale = largest / torch.full_like(largest, 448.0)
    return (b / scale).to(torch.float8_e4m3fn).view(padded.shape)[..., :n, :k], scale[..., 0, :, 0]


def _equal(a, b):
    """Bytes or numbers; a NaN equals a NaN."""
    a, b = a.float(), b.float()
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize('rows,k', [(1, 16), (1, 128), (7, 144), (130, 992), (300, 4096)])
def test_quantisation(rows, k, dtype):
    from msccl.ops.fp8_block import dequantize_fp8_block, quantize_fp8_block, quantize_fp8_block_weight
    gen = torch.Generator(device='cuda').manual_seed(k)
    x = torch.randn(rows, k, device='cuda', generator=gen) * torch.exp2(torch.randint(-12, 12, (rows, k // 16), device='cuda', generator=gen)
                                                                        .float()).repeat_interleave(16, 1)
    x = x.to(dtype)
    if rows > 5:
        x[0] = 0
        x[1, 3], x[2, 5], x[3, :] = float('nan'), float('inf'), 1e-6
        if dtype != torch.float16:
            x[4] = 1e-35
    for t in (x, torch.cat([x, x], 1)[:, k:]):             # a view whose rows are 2 k apart
        q, s = quantize_fp8_block(t)
        want_q, want_s = _definition(x, 1)
        assert _equal(q, want_q) and _equal(s, want_s) and q.shape == x.shape and s.shape == (rows, -(-k // 128))
        q, s = quantize_fp8_block_weight(t)
        want_q, want_s = _definition(x, 128)
        assert _equal(q, want_q) and _equal(s, want_s)
    w = torch.randn(3, rows, k, device='cuda', generator=gen).to(dtype)
    q, s = quantize_fp8_block_weight(w)
    want_q, want_s = _definition(w, 128)
    assert _equal(q, want_q) and _equal(s, want_s)
    # half an e4m3 step (2^-4 of a normal value, 2^-10 of the scale below), the quotient and the scale: 2^-23 each
    back, big = dequantize_fp8_block(q, s).double(), s.double().repeat_interleave(128, 1)[:, :rows].repeat_interleave(128, 2)[..., :k]
    assert torch.all((back - w.double()).abs() <= (2.0 ** -4 + 2.0 ** -22) * w.double().abs() + 2.0 ** -10 * big * (1 + 2.0 ** -20))


def _blocks(n):
    return -(-n // 128)


def _whole(gen, *shape):
    return torch.randint(-3, 4, shape, device='cuda', generator=gen).to(torch.float8_e4m3fn)


def _powers(gen, *shape):
    return torch.exp2(torch.randint(-1, 2, shape, device='cuda', generator=gen).float())


def _expand(a, sa, w, sw):
    k, n = a.shape[1], w.shape[0]
    return (a.float().double() * sa.double().repeat_interleave(128, 1)[:, :k],
            w.float().double() * sw.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k])


@pytest.mark.parametrize('m,n,k', [(1, 8, 16), (1, 4096, 256), (16, 1000, 2000), (32, 264, 384), (33, 128, 128), (128, 256, 640), (129, 40, 144),
                                   (300, 1032, 1040), (700, 4000, 512), (2000, 2056, 272)])
def test_dense_whole_numbers_are_exact(m, n, k):
    from msccl.ops import check_gemm_errors
    from msccl.ops.fp8_block import gemm_fp8_block
    gen = torch.Generator(device='cuda').manual_seed(m)
    a, w = _whole(gen, m, k), _whole(gen, n, k)
    sa, sw = _powers(gen, m, _blocks(k)), _powers(gen, _blocks(n), _blocks(k))
    ad, wd = _expand(a, sa, w, sw)
    want = (ad @ wd.t()).bfloat16()
    assert torch.equal(gemm_fp8_block(a, sa, w, sw), want)
    assert torch.equal(gemm_fp8_block(a, sa.t().contiguous().t(), w, sw), want)
    # views inside larger tensors, a result inside one
    big_a = torch.zeros(m, k + 32, device='cuda').to(torch.float8_e4m3fn)
    big_a[:, 16:k + 16] = a
    holder = torch.full((m + 1, n + 16), 7.0, dtype=torch.bfloat16, device='cuda')
    gemm_fp8_block(big_a[:, 16:k + 16], sa, w, sw, out=holder[:m, 8:n + 8])
    check_gemm_errors()
    assert torch.equal(holder[:m, 8:n + 8], want)
    holder[:m, 8:n + 8] = 7.0
    assert torch.all(holder == 7.0)


GROUPS = [([1], 0, 0, 8, 16), ([0, 5, 0, 20], 0, 0, 256, 256), ([33, 0, 31, 1], 0, 0, 264, 144), ([64, 128, 129], 2, 7, 136, 400),
          ([257, 511, 1], 5, 0, 1000, 208), ([0, 0], 0, 3, 64, 128), ([1] * 70, 0, 0, 40, 512)]


@pytest.mark.parametrize('sizes,head,tail,n,k', GROUPS)
def test_grouped_whole_numbers_are_exact(sizes, head, tail, n, k):
    from msccl.ops import check_gemm_errors
    from msccl.ops.fp8_block import grouped_gemm_fp8_block
    gen = torch.Generator(device='cuda').manual_seed(n)
    at = [head]
    for s in sizes:
        at.append(at[-1] + s)
    rows, offsets = at[-1] + tail, torch.tensor(at, dtype=torch.int32, device='cuda')
    a, w = _whole(gen, rows, k), _whole(gen, len(sizes), n, k)
    sa, sw = _powers(gen, rows, _blocks(k)), _powers(gen, len(sizes), _blocks(n), _blocks(k))
    want = torch.zeros(rows, n, dtype=torch.bfloat16, device='cuda')
    for e, (lo, hi) in enumerate(zip(at, at[1:])):
        ad, wd = _expand(a[lo:hi], sa[lo:hi], w[e], sw[e])
        want[lo:hi] = (ad @ wd.t()).bfloat16()
    sa[:head], sa[at[-1]:] = float('nan'), float('inf')     # rows of no group
    a.view(torch.uint8)[:head], a.view(torch.uint8)[at[-1]:] = 0x7f, 0x7f
    assert torch.equal(grouped_gemm_fp8_block(a, sa, w, sw, offsets), want)
    holder = torch.full((rows, n), 7.0, dtype=torch.bfloat16, device='cuda')
    grouped_gemm_fp8_block(a, sa, w, sw, offsets, out=holder)
    check_gemm_errors()
    used = slice(head, at[-1])
    assert torch.equal(holder[used], want[used])
    holder[used] = 7.0
    assert torch.all(holder == 7.0)


@pytest.mark.parametrize('m,n,k', [(16, 512, 4096), (200, 392, 1424), (1000, 1024, 2048)])
def test_quantised_product_within_its_bound(m, n, k):
    """fp32: 128 sums in a block, its scale (two products), one sum for each block; 2^-23 of the magnitudes each.  Then bf16."""
    from msccl.ops import check_gemm_errors
    from msccl.ops.fp8_block import gemm_fp8_block, quantize_fp8_block, quantize_fp8_block_weight
    gen = torch.Generator(device='cuda').manual_seed(k)
    x = torch.randn(m, k, device='cuda', generator=gen).bfloat16()
    a, sa = quantize_fp8_block(x)
    w, sw = quantize_fp8_block_weight((torch.randn(n, k, device='cuda', generator=gen) * 0.02).bfloat16())
    d = gemm_fp8_block(a, sa, w, sw)
    check_gemm_errors()
    ad, wd = _expand(a, sa, w, sw)
    want, magnitude = ad @ wd.t(), ad.abs() @ wd.abs().t()
    assert torch.all((d.double() - want).abs() <= 2.0 ** -8 * want.abs() * (1 + 2.0 ** -8) + (128 + 2 + _blocks(k)) * 2.0 ** -23 * magnitude)
    assert torch.equal(d, gemm_fp8_block(a, sa, w, sw))


def test_captured_and_on_another_stream():
    from msccl.ops import check_gemm_errors
    from msccl.ops.fp8_block import gemm_fp8_block, quantize_fp8_block, quantize_fp8_block_weight
    gen = torch.Generator(device='cuda').manual_seed(0)
    x = torch.randn(50, 512, device='cuda', generator=gen).bfloat16()
    w, sw = quantize_fp8_block_weight(torch.randn(256, 512, device='cuda', generator=gen))
    want = gemm_fp8_block(*quantize_fp8_block(x), w, sw)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    got = gemm_fp8_block(*quantize_fp8_block(x, stream=stream), w, sw, stream=stream)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = gemm_fp8_block(*quantize_fp8_block(x), w, sw)
    x.copy_(torch.randn(50, 512, device='cuda', generator=gen))
    g.replay()
    assert torch.equal(got, gemm_fp8_block(*quantize_fp8_block(x), w, sw))
    check_gemm_errors()


def test_no_rows():
    from msccl.ops.fp8_block import gemm_fp8_block, grouped_gemm_fp8_block, quantize_fp8_block, quantize_fp8_block_weight
    w, sw = quantize_fp8_block_weight(torch.randn(3, 40, 48, device='cuda'))
    q, s = quantize_fp8_block(torch.empty(0, 48, device='cuda'))
    assert gemm_fp8_block(q, s, w[0], sw[0]).shape == (0, 40)
    assert grouped_gemm_fp8_block(q, s, w, sw, torch.zeros(4, dtype=torch.int32, device='cuda')).shape == (0, 40)
