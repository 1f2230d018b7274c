"""Persistent kernels that take many tiles one after the other, and every variant that the rules on sizes choose, on whole numbers: exact sums
rounded once (partial sums stay below 2^24)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _whole(gen, *shape, dtype):
    return torch.randint(-3, 4, shape, device='cuda', generator=gen).to(dtype)


def _ends(sizes, head=0):
    at = [head]
    for s in sizes:
        at.append(at[-1] + s)
    return at, torch.tensor(at, dtype=torch.int32, device='cuda')


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('sizes,head,tail,n,k', [
    ([800, 0, 1000, 70, 64], 3, 5, 2048, 2048),            # stores with pauses and without, ragged ends, full blocks, no rows; 320 tiles
    ([768, 767, 1, 63, 832, 0, 129], 0, 0, 1800, 2504),    # either side of the pauses' border; sizes off the tiles
    ([5] * 60, 0, 0, 1032, 776),                           # nothing but ragged ends, more than ten tiles on a pair
    ([64, 128, 64, 192] * 3, 0, 0, 1024, 2048),            # nothing but full blocks
])
def test_grouped_products(sizes, head, tail, n, k, dtype):
    from msccl.ops import check_gemm_errors
    from msccl.ops.grouped import grouped_gemm, grouped_gemm_dgrad, grouped_gemm_wgrad
    gen = torch.Generator(device='cuda').manual_seed(n)
    at, offsets = _ends(sizes, head)
    rows = at[-1] + tail
    x, dy, w = _whole(gen, rows, k, dtype=dtype), _whole(gen, rows, n, dtype=dtype), _whole(gen, len(sizes), n, k, dtype=dtype)
    y, dx, dw = grouped_gemm(x, w, offsets), grouped_gemm_dgrad(dy, w, offsets), grouped_gemm_wgrad(dy, x, offsets)
    dw32 = grouped_gemm_wgrad(dy, x, offsets, dtype=torch.float32)
    check_gemm_errors()
    for t in (y, dx):
        assert torch.all(t[:head] == 0) and torch.all(t[at[-1]:] == 0)
    for e, (lo, hi) in enumerate(zip(at, at[1:])):
        xe, dye, we = x[lo:hi].double(), dy[lo:hi].double(), w[e].double()
        assert torch.equal(y[lo:hi], (xe @ we.t()).to(dtype)) and torch.equal(dx[lo:hi], (dye @ we).to(dtype))
        want = dye.t() @ xe
        assert torch.equal(dw[e], want.to(dtype)) and torch.equal(dw32[e], want.float())


def _blocks(n):
    return -(-n // 128)


@pytest.mark.parametrize('sizes,n,k,columns', [
    ([16], 7168, 1040, 64), ([1], 6400, 144, 64), ([32], 12808, 640, 128), ([3, 0, 20, 1, 5], 2008, 528, 64),      # at most 32 rows in all
    ([4] * 8, 4096, 400, 128), ([31], 14336, 272, 128), ([9, 7], 72, 2000, 32),
    ([40], 3208, 1296, 32), ([33], 6504, 656, 64), ([200], 4096, 272, 64), ([1000, 0, 1100, 3, 700], 3080, 400, 128),
    ([70] * 12, 5000, 272, 128),
])
def test_fp8_variants(sizes, n, k, columns):
    from msccl.ops import check_gemm_errors
    from msccl.ops.fp8_block import _tile_columns, gemm_fp8_block, grouped_gemm_fp8_block
    gen = torch.Generator(device='cuda').manual_seed(k)
    at, offsets = _ends(sizes)
    rows, f8 = at[-1], torch.float8_e4m3fn
    assert _tile_columns(rows, len(sizes), n) == columns
    a, w = _whole(gen, rows, k, dtype=f8), _whole(gen, len(sizes), n, k, dtype=f8)
    sa = torch.exp2(torch.randint(-1, 2, (rows, _blocks(k)), device='cuda', generator=gen).float())
    sw = torch.exp2(torch.randint(-1, 2, (len(sizes), _blocks(n), _blocks(k)), device='cuda', generator=gen).float())
    got = [grouped_gemm_fp8_block(a, sa, w, sw, offsets)]
    if len(sizes) == 1:
        got.append(gemm_fp8_block(a, sa, w[0], sw[0]))
    check_gemm_errors()
    ad = a.float().double() * sa.double().repeat_interleave(128, 1)[:, :k]
    for e, (lo, hi) in enumerate(zip(at, at[1:])):
        we = w[e].float().double() * sw[e].double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
        want = (ad[lo:hi] @ we.t()).bfloat16()
        assert all(torch.equal(g[lo:hi], want) for g in got)


@pytest.mark.parametrize('copies,experts', [(32768, 7), (32769, 7), (32769, 512), (1 << 22, 512), (1 << 22, 1)])
def test_large_sorts(copies, experts):
    from msccl.ops.moe_rows import sort_copies
    gen = torch.Generator(device='cuda').manual_seed(copies)
    chosen = torch.randint(-1, experts + 1, (copies, 1), device='cuda', generator=gen)
    order = sort_copies(chosen, experts)
    key = torch.where((chosen >= 0) & (chosen < experts), chosen, experts).reshape(-1)
    want = torch.argsort(key, stable=True)
    assert torch.equal(order.sorted_copy.long(), want)
    assert torch.equal(order.offsets.long(), torch.cat([want.new_zeros(1), torch.bincount(key, minlength=experts + 1).cumsum(0)[:experts]]))
    assert torch.equal(order.position.reshape(-1)[want].long(), torch.arange(copies, device='cuda'))
