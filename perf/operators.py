"""The operators of a trained or served expert layer, as timed cases on one GPU.

* ``grouped`` / ``grouped_train`` - matrix products of the token copies of each expert with that expert's weights
  (``msccl.ops.grouped``): the forward product, and the forward product with both gradients.
* ``fp8`` / ``fp8_grouped`` - products in 8-bit floating point with one fp32 scale per 128 values of an activation row and per
  128 x 128 block of a weight (``msccl.ops.fp8_block``), the activations quantised on the way.
* ``clip`` - the global norm of a list of gradients and their clipping (``msccl.ops.grad_norm``).
* ``rows`` - token copies sorted by expert, their rows gathered, the experts' results combined with the router's weights, and
  the gradients of both (``msccl.ops.moe_rows``).

``run`` takes the elementary torch operations while ``own`` is false and the framework's entry points while it is true.
"""
import math

import torch

own = False

DTYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
HIDDEN, FFN = 4096, 14336
MOST_FLOPS = 2 * 8192 * FFN * HIDDEN            # of the largest listed product
MOST_WEIGHTS = 8 * FFN * HIDDEN
MOST_GRADIENTS = 256 << 20


def listed():
    return [
        # gate projection of the benchmark's MoE layer: 4096 tokens, top-2 of 8 experts, one of them without tokens
        dict(name='grouped_prefill', kind='grouped', rows=8192, padding=0, experts=8, empty=1, n=FFN, k=HIDDEN, dtype='bf16'),
        # the same projection for a decode batch of 16 tokens: the weights are read for a few rows each
        dict(name='grouped_decode', kind='grouped', rows=32, padding=0, experts=8, empty=0, n=FFN, k=HIDDEN, dtype='bf16'),
        # many small experts, one token with eight copies: the latency of a call
        dict(name='grouped_one_token', kind='grouped', rows=8, padding=0, experts=64, empty=0, n=1024, k=2048, dtype='bf16'),
        # training step of a projection: result, gradient of the rows, gradient of the weights
        dict(name='grouped_train', kind='grouped_train', rows=8192, padding=0, experts=8, empty=0, n=HIDDEN, k=HIDDEN, dtype='bf16'),
        # odd everything: fp16, ragged sizes that fill no tile, empty experts, padded rows behind the last expert's
        dict(name='grouped_train_odd', kind='grouped_train', rows=1777, padding=47, experts=13, empty=3, n=1000, k=1416, dtype='f16'),
        # down projection of the Llama-3-8B MLP of the benchmark in fp8, 8192 tokens
        dict(name='fp8_prefill', kind='fp8', m=8192, n=HIDDEN, k=FFN),
        # the same weights for a decode batch
        dict(name='fp8_decode', kind='fp8', m=16, n=HIDDEN, k=FFN),
        # expert layer in fp8: 2048 tokens, top-2 of 8
        dict(name='fp8_grouped', kind='fp8_grouped', rows=4096, padding=0, experts=8, empty=0, n=HIDDEN, k=HIDDEN),
        # a flat bf16 gradient bucket of 512 MB clipped into the optimizer's fp32 copy
        dict(name='clip_bucket', kind='clip', tensors=1, elements=MOST_GRADIENTS, dtype='bf16', out='f32', clipping=True),
        # the gradients of a model of some hundred parameters, in place, on a step that needs no clipping
        dict(name='clip_many', kind='clip', tensors=291, elements=8 << 20, dtype='f32', out='', clipping=False),
        # exchange of rows around the experts of the benchmark's MoE layer, in training
        dict(name='rows_train', kind='rows', tokens=4096, topk=2, experts=8, hidden=HIDDEN, dropped=False, gradients=True),
        # ... and for a decode batch
        dict(name='rows_decode', kind='rows', tokens=16, topk=2, experts=8, hidden=HIDDEN, dropped=False, gradients=False),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _size(rng, low, high, step):
    return max(low, _log(rng, low, high) // step * step)


def draw(rng):
    kind = rng.choice(('grouped', 'grouped_train', 'fp8', 'fp8_grouped', 'clip', 'rows'))
    if kind in ('grouped', 'grouped_train', 'fp8_grouped'):
        step = 16 if kind == 'fp8_grouped' else 8
        experts = _log(rng, 1, 128)
        n, k = _size(rng, 64, FFN, step), _size(rng, 64, FFN, step)
        while experts * n * k > MOST_WEIGHTS:
            experts = max(1, experts // 2)
        most = MOST_FLOPS // (2 * n * k * (3 if kind == 'grouped_train' else 1))
        case = dict(kind=kind, rows=_log(rng, 1, max(1, min(16384, most))), padding=rng.choice((0, 0, rng.randint(1, 300))),
                    experts=experts, empty=rng.randint(0, experts - 1) if rng.random() < 0.4 else 0, n=n, k=k)
        return case if kind == 'fp8_grouped' else dict(case, dtype=rng.choice(('bf16', 'bf16', 'f16')))
    if kind == 'fp8':
        n, k = _size(rng, 64, FFN, 16), _size(rng, 64, FFN, 16)
        return dict(kind=kind, m=_log(rng, 1, min(16384, MOST_FLOPS // (2 * n * k))), n=n, k=k)
    if kind == 'clip':
        tensors = _log(rng, 1, 1000)
        dtype = rng.choice(('f32', 'bf16', 'f16'))
        return dict(kind=kind, tensors=tensors, elements=_log(rng, 1000 * tensors, MOST_GRADIENTS // 2), dtype=dtype,
                    out=rng.choice(('f32', dtype)) if rng.random() < 0.5 else '', clipping=False) if rng.random() < 0.5 else \
            dict(kind=kind, tensors=tensors, elements=_log(rng, 1000 * tensors, MOST_GRADIENTS // 2), dtype=dtype,
                 out=rng.choice(('f32', dtype)), clipping=True)
    return dict(kind=kind, tokens=_log(rng, 1, 4096), topk=rng.randint(1, 8), experts=rng.randint(8, 256), hidden=_size(rng, 64, HIDDEN, 8),
                dropped=rng.random() < 0.3, gradients=rng.random() < 0.6)


# ------------------------------------------------------------------------------------------------ what a program has in hand
def _normal(gen, *shape, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, device='cuda', generator=gen) * std).to(dtype)


def _group_sizes(case, seed):
    """Rows of each expert: every expert but ``empty`` of them has one at least, the rest follows a skewed router."""
    gen = torch.Generator().manual_seed(seed)
    experts = case['experts']
    active = min(experts - case['empty'], case['rows'])
    chosen = torch.randperm(experts, generator=gen)[:active]
    popularity = torch.exp(0.5 * torch.randn(active, generator=gen))
    extra = torch.zeros(active, dtype=torch.int64)
    if case['rows'] > active:
        extra = torch.bincount(torch.multinomial(popularity, case['rows'] - active, replacement=True, generator=gen), minlength=active)
    sizes = torch.zeros(experts, dtype=torch.int64)
    sizes[chosen] = 1 + extra
    return sizes.tolist()


def _starts(sizes):
    starts = [0]
    for s in sizes:
        starts.append(starts[-1] + s)
    return starts


def _plain_quantize(x):
    """e4m3 values and one fp32 scale, largest magnitude / 448, for each 128 values of a row (the last ones may be fewer)."""
    rows, k = x.shape
    blocks = torch.nn.functional.pad(x.float(), (0, -k % 128)).view(rows, -1, 128)
    largest = blocks.abs().amax(-1).clamp_min(2.0 ** -100)
    scales = largest / torch.full_like(largest, 448.0)             # by a tensor: a number would become a product with 1 / 448
    return (blocks / scales[:, :, None]).to(torch.float8_e4m3fn).view(rows, -1)[:, :k], scales


def _quantize_weight(w):
    """The same with one scale for each block of 128 x 128 of every [n, k] matrix in ``w``."""
    n, k = w.shape[-2:]
    padded = torch.nn.functional.pad(w.float(), (0, -k % 128, 0, -n % 128))
    blocks = padded.view(*w.shape[:-2], padded.shape[-2] // 128, 128, padded.shape[-1] // 128, 128)
    largest = blocks.abs().amax((-3, -1)).clamp_min(2.0 ** -100)
    scales = largest / torch.full_like(largest, 448.0)
    q = (blocks / scales[..., :, None, :, None]).to(torch.float8_e4m3fn).view(padded.shape)
    return q[..., :n, :k].contiguous(), scales


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    kind = case['kind']
    state = dict(case)
    if kind in ('grouped', 'grouped_train', 'fp8_grouped'):
        rows, dtype = case['rows'] + case['padding'], DTYPES[case.get('dtype', 'bf16')]
        state['starts'] = _starts(_group_sizes(case, seed))
        state['offsets'] = torch.tensor(state['starts'], dtype=torch.int32, device='cuda')
        state['x'] = _normal(gen, rows, case['k'], dtype=dtype)
        w = _normal(gen, case['experts'], case['n'], case['k'], std=0.02, dtype=dtype)
        if kind == 'fp8_grouped':
            state['w'], state['w_scales'] = _quantize_weight(w)
        else:
            state['w'] = w
        if kind == 'grouped_train':
            state['dy'] = _normal(gen, rows, case['n'], std=0.1, dtype=dtype)
            state['x'].requires_grad_()
            state['w'].requires_grad_()
    elif kind == 'fp8':
        state['x'] = _normal(gen, case['m'], case['k'])
        state['w'], state['w_scales'] = _quantize_weight(_normal(gen, case['n'], case['k'], std=0.02))
    elif kind == 'clip':
        cpu = torch.Generator().manual_seed(case['tensors'])        # the model's sizes do not depend on the seed
        weights = torch.exp(1.5 * torch.randn(case['tensors'], generator=cpu, dtype=torch.float64))
        sizes = (weights / weights.sum() * case['elements']).long().clamp_min(1).tolist()
        starts = _starts([-(-s // 8) * 8 for s in sizes])           # every parameter starts on a 16-byte boundary
        cut = lambda flat: [flat[at:at + s] for at, s in zip(starts, sizes)]                            # noqa: E731
        drawn = _normal(gen, starts[-1], std=1e-2, dtype=DTYPES[case['dtype']])
        state['flat'] = torch.zeros_like(drawn)
        state['gradients'] = cut(state['flat'])
        for g, d in zip(state['gradients'], cut(drawn)):
            g.copy_(d)
        expected = 1e-2 * math.sqrt(sum(sizes))
        state['max_norm'] = 0.3 * expected if case['clipping'] else 10 * expected + 1
        state['flat_out'] = torch.zeros(starts[-1], dtype=DTYPES[case['out']], device='cuda') if case['out'] else state['flat']
        state['out'] = cut(state['flat_out']) if case['out'] else None
    else:
        tokens, topk, hidden = case['tokens'], case['topk'], case['hidden']
        logits = torch.randn(tokens, case['experts'], device='cuda', generator=gen)
        top, experts = torch.topk(logits, topk, dim=-1)
        state['chosen'] = experts.to(torch.int32)
        if case['dropped']:                             # padded tokens: no expert takes their copies
            state['chosen'][torch.rand(tokens, device='cuda', generator=gen) < 0.2] = -1
        state['weights'] = torch.softmax(top, -1)
        state['x'] = _normal(gen, tokens, hidden)
        state['ys'] = _normal(gen, tokens * topk, hidden)
        if case['gradients']:
            state['dxs'], state['dy'] = _normal(gen, tokens * topk, hidden), _normal(gen, tokens, hidden)
            for name in ('x', 'ys', 'weights'):
                state[name].requires_grad_()
    return state


# ---------------------------------------------------------------------------------------------------------------- one pass
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(state):
    from msccl.ops.fp8_block import gemm_fp8_block, grouped_gemm_fp8_block, quantize_fp8_block
    from msccl.ops.grad_norm import clip_grad_norm
    from msccl.ops.grouped import grouped_gemm
    from msccl.ops.moe_rows import combine_rows, gather_rows, sort_copies
    kind = state['kind']
    if kind == 'grouped':
        return grouped_gemm(state['x'], state['w'], state['offsets'])
    if kind == 'grouped_train':
        y = grouped_gemm(state['x'], state['w'], state['offsets'])
        dx, dw = torch.autograd.grad(y, (state['x'], state['w']), state['dy'])
        return y.detach(), dx, dw
    if kind == 'fp8':
        q, scales = quantize_fp8_block(state['x'])
        return gemm_fp8_block(q, scales, state['w'], state['w_scales'])
    if kind == 'fp8_grouped':
        q, scales = quantize_fp8_block(state['x'])
        return grouped_gemm_fp8_block(q, scales, state['w'], state['w_scales'], state['offsets'])
    if kind == 'clip':
        norm = clip_grad_norm(state['gradients'], state['max_norm'], out=state['out'])
        return norm, state['flat_out']
    order = sort_copies(state['chosen'], state['experts'])
    xs = gather_rows(state['x'], order)
    y = combine_rows(state['ys'], state['weights'], order)
    result = [order.sorted_copy, order.offsets, xs.detach(), y.detach()]
    if state['gradients']:
        result += torch.autograd.grad((xs, y), (state['x'], state['ys'], state['weights']), (state['dxs'], state['dy']))
    return result


def _plain_dequantized(x):
    q, scales = _plain_quantize(x)
    return q.float() * scales.repeat_interleave(128, 1)[:, :x.shape[1]]


def _plain_weight(w, scales):
    n, k = w.shape
    return w.float() * scales.repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]


def _run_plain(state):
    kind = state['kind']
    if kind in ('grouped', 'grouped_train'):
        x, w, starts = state['x'].detach().float(), state['w'].detach(), state['starts']
        y = torch.zeros(x.shape[0], w.shape[1], dtype=w.dtype, device='cuda')
        train = kind == 'grouped_train'
        if train:
            dy, dx, dw = state['dy'].float(), torch.zeros_like(x, dtype=w.dtype), torch.zeros_like(w)
        for e, (lo, hi) in enumerate(zip(starts, starts[1:])):
            if hi > lo:
                we = w[e].float()
                y[lo:hi] = x[lo:hi] @ we.t()
                if train:
                    dx[lo:hi] = dy[lo:hi] @ we
                    dw[e] = dy[lo:hi].t() @ x[lo:hi]
        return (y, dx, dw) if train else y
    if kind == 'fp8':
        return (_plain_dequantized(state['x']) @ _plain_weight(state['w'], state['w_scales']).t()).bfloat16()
    if kind == 'fp8_grouped':
        x, starts = _plain_dequantized(state['x']), state['starts']
        y = torch.zeros(x.shape[0], state['n'], dtype=torch.bfloat16, device='cuda')
        for e, (lo, hi) in enumerate(zip(starts, starts[1:])):
            if hi > lo:
                y[lo:hi] = x[lo:hi] @ _plain_weight(state['w'][e], state['w_scales'][e]).t()
        return y
    if kind == 'clip':
        gradients, out = state['gradients'], state['out'] or state['gradients']
        norm = torch.stack([(g.float() * g.float()).sum(dtype=torch.float64) for g in gradients]).sum().sqrt()
        factor = (state['max_norm'] / (norm + 1e-6)).clamp_max(1.0).float()
        for g, o in zip(gradients, out):
            o.copy_(g.float() * factor)
        return norm.float(), state['flat_out']
    chosen, weights, topk = state['chosen'].reshape(-1), state['weights'].detach(), state['topk']
    experts = state['experts']
    key = torch.where((chosen >= 0) & (chosen < experts), chosen, experts).long()
    order = torch.argsort(key, stable=True)
    offsets = torch.cumsum(torch.bincount(key, minlength=experts + 1), 0)[:experts]
    offsets = torch.cat([offsets.new_zeros(1), offsets]).to(torch.int32)
    kept = (key[order] < experts)[:, None].float()
    token = order // topk
    xs = (state['x'].detach().float()[token] * kept).bfloat16()
    position = torch.empty_like(order)
    position[order] = torch.arange(order.numel(), device='cuda')
    back = position.view(-1, topk)
    taken = (key < experts).view(-1, topk, 1).float()
    ys = state['ys'].detach().float()
    y = (ys[back] * taken * weights[:, :, None]).sum(1).bfloat16()
    result = [order.to(torch.int32), offsets, xs, y]
    if state['gradients']:
        dy = state['dy'].float()
        dx = (state['dxs'].float()[back] * taken).sum(1).bfloat16()
        dys = (dy[token] * kept * weights.reshape(-1)[order][:, None]).bfloat16()
        dw = (ys[back] * taken * dy[:, None, :]).sum(-1)
        result += [dx, dys, dw]
    return result


# ------------------------------------------------------------------------------------------------------- work and definition
def work(case):
    """Every input and weight read once, every result written once; FLOPs of the contractions (of the sums elsewhere)."""
    kind = case['kind']
    if kind in ('grouped', 'grouped_train'):
        rows, n, k = case['rows'], case['n'], case['k']
        active = min(case['experts'] - case['empty'], rows)
        if kind == 'grouped':
            return {'bytes': 2 * (rows * k + active * n * k + rows * n), 'flops': 2 * rows * n * k}
        return {'bytes': 2 * (2 * rows * k + 2 * rows * n + (active + case['experts']) * n * k), 'flops': 6 * rows * n * k}
    if kind == 'fp8':
        m, n, k = case['m'], case['n'], case['k']
        return {'bytes': 2 * m * k + n * k + 4 * -(-n // 128) * -(-k // 128) + 2 * m * n, 'flops': 2 * m * n * k}
    if kind == 'fp8_grouped':
        rows, n, k = case['rows'], case['n'], case['k']
        active = min(case['experts'] - case['empty'], rows)
        return {'bytes': 2 * rows * k + active * (n * k + 4 * -(-n // 128) * -(-k // 128)) + 2 * rows * n, 'flops': 2 * rows * n * k}
    if kind == 'clip':
        written = DTYPES[case['out']].itemsize if case['out'] else DTYPES[case['dtype']].itemsize if case['clipping'] else 0
        return {'bytes': case['elements'] * (DTYPES[case['dtype']].itemsize + written), 'flops': 3 * case['elements']}
    tokens, copies, hidden = case['tokens'], case['tokens'] * case['topk'], case['hidden']
    forward = 2 * hidden * (tokens + copies) * 2 + copies * 12
    if not case['gradients']:
        return {'bytes': forward, 'flops': 2 * copies * hidden}
    # back: dxs -> dx, and dy, ys -> dys, dw
    return {'bytes': forward + 2 * hidden * (copies + tokens + tokens + 2 * copies) + 4 * copies, 'flops': 7 * copies * hidden}


def _exact_e4m3(v):
    """The nearest e4m3 number, ties to even: three mantissa bits, exponents from -6 up, nothing above 448."""
    exponent = torch.frexp(v)[1].clamp_min(-5) - 1
    step = torch.ldexp(torch.ones_like(v), exponent - 3)
    return (torch.round(v / step) * step).clamp(-448.0, 448.0)


def _exact_activation(x):
    out = torch.empty(x.shape, dtype=torch.float64, device='cuda')
    for lo in range(0, x.shape[1], 128):
        part = x[:, lo:lo + 128].double()
        scale = (part.abs().max(1, keepdim=True).values.clamp_min(2.0 ** -100) / 448.0).float().double()
        out[:, lo:lo + 128] = _exact_e4m3((part / scale).float().double()) * scale      # the quotient is a 32-bit number
    return out


def _exact_weight(q, scales):
    w = q.to(torch.float32).double()
    for i in range(scales.shape[0]):
        for j in range(scales.shape[1]):
            w[128 * i:128 * i + 128, 128 * j:128 * j + 128] *= scales[i, j].double()
    return w


def exact(case, seed):
    state = prepare(case, seed)
    kind = case['kind']
    with torch.no_grad():
        if kind in ('grouped', 'grouped_train', 'fp8_grouped'):
            x = _exact_activation(state['x']) if kind == 'fp8_grouped' else state['x'].double()
            y = x.new_zeros(x.shape[0], case['n'])
            dx, dw = (torch.zeros_like(x), x.new_zeros(state['w'].shape)) if kind == 'grouped_train' else (None, None)
            for e in range(case['experts']):
                rows = slice(state['starts'][e], state['starts'][e + 1])
                if rows.start == rows.stop:
                    continue
                w = _exact_weight(state['w'][e], state['w_scales'][e]) if kind == 'fp8_grouped' else state['w'][e].double()
                y[rows] = torch.einsum('tk,nk->tn', x[rows], w)
                if dx is not None:
                    dy = state['dy'][rows].double()
                    dx[rows] = torch.einsum('tn,nk->tk', dy, w)
                    dw[e] = torch.einsum('tn,tk->nk', dy, x[rows])
            return y if dx is None else (y, dx, dw)
        if kind == 'fp8':
            return torch.einsum('mk,nk->mn', _exact_activation(state['x']), _exact_weight(state['w'], state['w_scales']))
        if kind == 'clip':
            flat = state['flat'].double()                   # zero between the parameters
            norm = torch.linalg.vector_norm(flat)
            return norm, flat * min(1.0, state['max_norm'] / (float(norm) + 1e-6))
        topk, experts = case['topk'], case['experts']
        chosen = state['chosen'].reshape(-1).tolist()
        buckets = [[] for _ in range(experts + 1)]
        for copy, e in enumerate(chosen):
            buckets[e if 0 <= e < experts else experts].append(copy)
        starts = _starts([len(b) for b in buckets[:experts]])
        order = torch.tensor([c for b in buckets for c in b], device='cuda')
        kept = order[:starts[-1]]
        x, ys, weights = state['x'].double(), state['ys'].double(), state['weights'].double().reshape(-1)
        xs = torch.zeros_like(ys)
        xs[:kept.numel()] = x[kept // topk]
        copies = torch.zeros_like(ys)                   # the experts' results in the order of the copies
        copies[kept] = ys[:kept.numel()]
        y = (copies * weights[:, None]).view(-1, topk, copies.shape[1]).sum(1)
        result = [order, torch.tensor(starts, device='cuda'), xs, y]
        if case['gradients']:
            dy = state['dy'].double()
            back = torch.zeros_like(ys)
            back[kept] = state['dxs'].double()[:kept.numel()]
            dys = torch.zeros_like(ys)
            dys[:kept.numel()] = dy[kept // topk] * weights[kept][:, None]
            result += [back.view(-1, topk, back.shape[1]).sum(1), dys,
                       (copies.view(-1, topk, copies.shape[1]) * dy[:, None, :]).sum(-1)]
        return result
