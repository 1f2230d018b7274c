"""Elements beyond 2^31 of an operand or a result: the last rows against the same rows on their own."""
import pytest
import torch

pytestmark = pytest.mark.gpu

ROWS, COLUMNS = 140000, 16384                              # 2.29e9 elements


@pytest.fixture(autouse=True)
def give_back_memory():
    yield
    torch.cuda.empty_cache()


def _wide():
    """Rows that differ, from a small pattern."""
    gen = torch.Generator(device='cuda').manual_seed(0)
    x = torch.empty(ROWS, COLUMNS, dtype=torch.bfloat16, device='cuda')
    block = torch.randint(-3, 4, (1000, COLUMNS), device='cuda', generator=gen).bfloat16()
    for i in range(0, ROWS, 1000):
        x[i:i + 1000] = block * (1 + i // 1000 % 5)
    return x


LAST = slice(ROWS - 300, ROWS)


def test_rows_and_quantisation():
    from msccl.ops import combine_rows, gather_rows, quantize_fp8_block, sort_copies
    x = _wide()
    q, s = quantize_fp8_block(x)
    want_q, want_s = quantize_fp8_block(x[LAST])
    assert torch.equal(q[LAST].view(torch.uint8), want_q.view(torch.uint8)) and torch.equal(s[LAST], want_s)
    del q, s
    order = sort_copies(torch.arange(ROWS, device='cuda').flip(0)[:, None] // 20000, 7)
    xs = gather_rows(x, order)
    at = order.sorted_copy.long()
    assert torch.equal(xs[LAST], x[at[LAST]]) and torch.equal(xs[:10], x[at[:10]])
    weights = torch.full((ROWS, 1), 2.0, device='cuda')
    y = combine_rows(xs, weights, order)
    assert torch.equal(y[LAST], 2 * x[LAST])
    del y
    leaves = xs.requires_grad_(), weights.requires_grad_()
    dxs, dweights = torch.autograd.grad(combine_rows(*leaves, order), leaves, x)
    assert torch.equal(dxs[LAST], 2 * x[at[LAST]])
    want = (x[LAST].double() ** 2).sum(1)                   # whole numbers, sums below 2^24
    assert torch.equal(dweights[LAST, 0].double(), want)


def test_fp8_products():
    from msccl.ops import check_gemm_errors, gemm_fp8_block, grouped_gemm_fp8_block
    gen = torch.Generator(device='cuda').manual_seed(1)
    f8, k = torch.float8_e4m3fn, 128
    a = torch.randint(-3, 4, (ROWS, k), device='cuda', generator=gen).to(f8)
    w = torch.randint(-3, 4, (2, COLUMNS, k), device='cuda', generator=gen).to(f8)
    sa, sw = torch.ones(ROWS, 1, device='cuda'), torch.ones(2, COLUMNS // 128, 1, device='cuda')
    want = (a[LAST].float() @ w[1].float().t()).bfloat16()
    y = gemm_fp8_block(a, sa, w[1], sw[1])
    check_gemm_errors()
    assert torch.equal(y[LAST], want)
    del y
    y = grouped_gemm_fp8_block(a, sa, w, sw, torch.tensor([0, 70001, ROWS - 100], dtype=torch.int32, device='cuda'))
    check_gemm_errors()
    assert torch.equal(y[ROWS - 300:ROWS - 100], want[:200]) and torch.all(y[ROWS - 100:] == 0)


def test_weights():
    from msccl.ops import check_gemm_errors, grouped_gemm_wgrad, quantize_fp8_block_weight
    gen = torch.Generator(device='cuda').manual_seed(2)
    experts, n, k = 9, COLUMNS, COLUMNS
    dy = torch.randint(-3, 4, (experts * 10, n), device='cuda', generator=gen).bfloat16()
    x = torch.randint(-3, 4, (experts * 10, k), device='cuda', generator=gen).bfloat16()
    dw = grouped_gemm_wgrad(dy, x, torch.arange(0, 91, 10, dtype=torch.int32, device='cuda'))
    check_gemm_errors()
    assert torch.equal(dw[8], (dy[80:].float().t() @ x[80:].float()).bfloat16())
    q, s = quantize_fp8_block_weight(dw)
    want_q, want_s = quantize_fp8_block_weight(dw[8])
    assert torch.equal(q[8].view(torch.uint8), want_q.view(torch.uint8)) and torch.equal(s[8], want_s)
