"""The expert-layer operators together, as ``GroupedMoE`` and ``FlatGradients`` run them: forward, backward, clipping, fp8, graphs."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _reference(layer, x, experts, weights):
    """The layer in 64 bits for given routing, intermediates rounded where the layer stores them."""
    def stored(t):
        # the value that the layer stores, the gradient of the exact one
        return t + (t.to(x.dtype).double() - t).detach()
    w_gu, w_d = layer.w_gate_up, layer.w_down
    y = torch.zeros(x.shape[0], layer.hidden, dtype=torch.float64, device=x.device)
    for e in range(layer.num_experts):
        token, j = torch.where(experts == e)
        if token.numel():
            gu = stored(x[token].double() @ w_gu[e].double().t())
            gate, up = gu.split(layer.ffn, 1)
            ys = stored(stored(stored(torch.nn.functional.silu(gate)) * up) @ w_d[e].double().t())
            y = y.index_add(0, token, ys * weights[token, j][:, None].double())
    return y


def _rel(a, b):
    return float((a.detach().double() - b.detach()).norm() / b.detach().norm())


@pytest.mark.parametrize('tokens,hidden,ffn,experts,topk,dtype', [(1, 64, 128, 4, 2, torch.bfloat16), (100, 136, 72, 8, 3, torch.bfloat16),
                                                                  (1000, 512, 768, 16, 2, torch.bfloat16), (333, 256, 264, 5, 1, torch.float16)])
def test_layer_and_gradients(tokens, hidden, ffn, experts, topk, dtype):
    from msccl.ops import check_gemm_errors
    from msccl.ops.moe import route_top_k
    from msccl.parallel import GroupedMoE
    gen = torch.Generator(device='cuda').manual_seed(tokens)
    layer = GroupedMoE(hidden, ffn, experts, topk, dtype=dtype, std=0.1)
    x = torch.randn(tokens, hidden, device='cuda', generator=gen).to(dtype).requires_grad_()
    dy = torch.randn(tokens, hidden, device='cuda', generator=gen).to(dtype)
    leaves = [x, layer.w_router, layer.w_gate_up, layer.w_down]
    y = layer(x)
    got = torch.autograd.grad(y, leaves, dy)
    check_gemm_errors()
    chosen, weights = route_top_k(x @ layer.w_router.t(), topk)
    want_y = _reference(layer, x, chosen, weights)
    want = torch.autograd.grad(want_y, leaves, dy.double(), allow_unused=True)
    # Each tensor that the layer stores is off by at most half a step of its type, at most half of that in the norm.  Between a result
    # and its inputs lie up to three products in a row (the result itself and at most six stored tensors: gate | up, silu, h, ys and
    # their gradients); errors of independent roundings add up in the square.
    step = torch.finfo(dtype).eps / 2
    bound = step * 7 ** 0.5
    assert _rel(y, want_y) <= bound
    for name, g, w in zip(('x', 'w_router', 'w_gate_up', 'w_down'), got, want):
        if name == 'w_router' and topk == 1:
            # the weight of a single copy is 1 whatever the logits
            assert float(g.double().norm()) <= 1e-6 * float(want[0].norm()) * tokens
            continue
        assert _rel(g, w) <= bound, name
    # experts without tokens get a gradient of zero
    idle = torch.bincount(chosen.reshape(-1), minlength=experts) == 0
    assert torch.all(got[2][idle] == 0) and torch.all(got[3][idle] == 0)


def test_training_step_with_flat_gradients_and_clipping():
    from msccl.ops import check_gemm_errors
    from msccl.parallel import FlatGradients, GroupedMoE
    layer = GroupedMoE(128, 96, 4, 2)
    flat = FlatGradients(layer.parameters(), lambda n, d: torch.empty(n, dtype=d, device='cuda'), bucket_bytes=1 << 16)
    assert len(flat.buckets) > 1
    gen = torch.Generator(device='cuda').manual_seed(0)
    for step in range(2):
        flat.zero()
        for _ in range(2):                                 # gradients accumulate over two batches
            x = torch.randn(50, 128, device='cuda', generator=gen).bfloat16()
            layer(x).float().square().sum().backward()
        flat.all_reduce_gradients(lambda t: t.mul_(2), 2)  # two ranks with the same gradients
        before = [p.grad.double().clone() for p in layer.parameters()]
        want = torch.sqrt(sum((g * g).sum() for g in before))
        norm = flat.clip_grad_norm(float(want) / 3)
        assert abs(float(norm) - float(want)) <= 6 * 2.0 ** -24 * float(want)
        for p, b in zip(layer.parameters(), before):
            assert torch.all((p.grad.double() - b / 3).abs() <= (2.0 ** -8 + 2.0 ** -18) * b.abs() / 3 + 1e-38)
        flat.all_reduce_gradients(lambda t: None, 1)       # the views are still in place
    check_gemm_errors()


def test_fp8_forward():
    from msccl.ops import check_gemm_errors
    from msccl.parallel import GroupedMoE
    layer = GroupedMoE(256, 320, 8, 2, std=0.1)
    x = torch.randn(77, 256, device='cuda', generator=torch.Generator(device='cuda').manual_seed(1)).bfloat16()
    with pytest.raises(RuntimeError):
        layer(x, precision='fp8')
    with pytest.raises(ValueError):
        layer(x, precision='fp4')
    with pytest.raises(ValueError):
        GroupedMoE(64, 64, 2, dtype=torch.float16).quantize()
    layer.quantize()
    y8, y = layer(x, precision='fp8'), layer(x)
    check_gemm_errors()
    assert not y8.requires_grad
    # e4m3 keeps a value within 2^-4, its rounding is about uniform: 2^-4 / sqrt(3) in the norm at the coarsest, for each of the four
    # quantised operands (and their bf16 intermediates, far below)
    assert _rel(y8, y.double()) <= 2 * 2.0 ** -4 / 3 ** 0.5


def test_captured_forward_with_other_routing():
    from msccl.ops import check_gemm_errors
    from msccl.parallel import GroupedMoE
    layer = GroupedMoE(128, 128, 8, 2, std=0.1).quantize()
    gen = torch.Generator(device='cuda').manual_seed(2)
    x = torch.randn(40, 128, device='cuda', generator=gen).bfloat16()
    with torch.no_grad():
        for precision in (None, 'fp8'):
            layer(x, precision=precision)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results = [layer(x, precision=p) for p in (None, 'fp8')]
        for scale in (1.0, -1.0):
            x.copy_(torch.randn(40, 128, device='cuda', generator=gen) * scale)
            graph.replay()
            assert torch.equal(results[0], layer(x)) and torch.equal(results[1], layer(x, precision='fp8'))
    check_gemm_errors()


def test_captured_training_step():
    """Forward, backward and clipping in one graph, equal to the eager step bit for bit."""
    import os
    import subprocess
    import sys
    code = """
import torch
from msccl.ops import check_gemm_errors
from msccl.parallel import FlatGradients, GroupedMoE
layer = GroupedMoE(128, 96, 4, 2, std=0.1)
flat = FlatGradients(layer.parameters(), lambda n, d: torch.empty(n, dtype=d, device='cuda'))
x = torch.randn(60, 128, device='cuda').bfloat16()
def step():
    flat.zero()
    layer(x).float().square().sum().backward()
    return flat.clip_grad_norm(1.0)
side = torch.cuda.Stream()
side.wait_stream(torch.cuda.current_stream())
with torch.cuda.stream(side):
    step()
torch.cuda.current_stream().wait_stream(side)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    norm = step()
for _ in range(2):
    x.copy_(torch.randn(60, 128, device='cuda'))
    graph.replay()
    got = [p.grad.clone() for p in layer.parameters()], float(norm)
    want_norm = float(step())
    want = [p.grad.clone() for p in layer.parameters()]
    assert all(torch.equal(a, b) for a, b in zip(got[0], want)) and got[1] == want_norm
check_gemm_errors()
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, '-c', code], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stdout + done.stderr
