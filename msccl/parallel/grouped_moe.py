"""Mixture-of-experts layer on one GPU without a capacity, trained or served: every token copy reaches its expert, whatever the
router does.  ``ExpertParallelMoE`` shards experts over GPUs and is forward only; this layer holds all of its experts and is the one
to train data-parallel (``FlatGradients`` takes its parameters, sums and clips their gradients).
"""
import torch

from msccl.ops.fp8_block import grouped_gemm_fp8_block, quantize_fp8_block, quantize_fp8_block_weight
from msccl.ops.grouped import grouped_gemm
from msccl.ops.moe import route_top_k
from msccl.ops.moe_rows import MAX_EXPERTS, MAX_TOPK, combine_rows, gather_rows, sort_copies


class GroupedMoE(torch.nn.Module):
    """``y[t] = sum_j p[t, j] * down_e(silu(gate_e(x[t])) * up_e(x[t]))`` over the ``topk`` experts ``e`` of token ``t``, ``p`` the softmax
    over their router logits.

    ``forward`` takes any number of tokens (one at least, at most 2 ** 22 copies of them), [tokens, hidden] in the layer's dtype, and is differentiable in ``x``, the
    router and the experts.  ``quantize()`` makes the fp8 form of the experts (of a bf16 layer); ``forward(x, precision='fp8')`` then runs
    on it, without gradients; the default runs in the layer's own type.  The fp8 form moves with the layer to another device; loading a state
    or changing the layer's type ends it, until the next ``quantize()``.  hidden and ffn: multiples of 8 (16 for fp8)."""

    def __init__(self, hidden, ffn, num_experts, topk=2, device='cuda', dtype=torch.bfloat16, std=0.02, seed=0):
        super().__init__()
        if not 1 <= num_experts <= MAX_EXPERTS:
            raise ValueError(f'between 1 and {MAX_EXPERTS} experts are supported (got {num_experts})')
        if not 1 <= topk <= min(MAX_TOPK, num_experts):
            raise ValueError(f'topk must be within 1 and {min(MAX_TOPK, num_experts)} with {num_experts} experts (got {topk})')
        for name, size in (('hidden', hidden), ('ffn', ffn)):
            if size < 8 or size % 8:
                raise ValueError(f'{name} must be a positive multiple of 8 (got {size})')
        self.hidden, self.ffn, self.num_experts, self.topk = hidden, ffn, num_experts, topk
        gen = torch.Generator(device=device).manual_seed(seed)

        def mk(*shape):
            return torch.nn.Parameter((torch.randn(*shape, device=device, generator=gen) * std).to(dtype))
        self.w_router = mk(num_experts, hidden)
        self.w_gate_up = mk(num_experts, 2 * ffn, hidden)        # the gate's rows, then the up projection's
        self.w_down = mk(num_experts, hidden, ffn)
        self._fp8 = None

    def quantize(self):
        """Quantise the experts as they are now (blocks of 128 x 128, ``msccl.ops.fp8_block``).  Training goes on with the others."""
        if self.w_down.dtype != torch.bfloat16:
            raise ValueError(f'the fp8 products give bf16, the layer is {self.w_down.dtype}')
        self._fp8 = quantize_fp8_block_weight(self.w_gate_up.detach()) + quantize_fp8_block_weight(self.w_down.detach())
        return self

    def _apply(self, fn, recurse=True):
        super()._apply(fn, recurse)
        if self._fp8 is not None:
            # fn moves tensors and converts floating-point ones: as integers these keep their bits
            moved = [(fn(t.view(bits)), bits, t.dtype) for t, bits in zip(self._fp8, (torch.uint8, torch.int32) * 2)]
            kept = self.w_down.dtype == torch.bfloat16 and all(m.dtype == bits for m, bits, _ in moved)
            self._fp8 = tuple(m.view(dtype) for m, _, dtype in moved) if kept else None
        return self

    def _load_from_state_dict(self, state_dict, prefix, *args, **kwargs):
        if prefix + 'w_gate_up' in state_dict or prefix + 'w_down' in state_dict:
            self._fp8 = None                                 # of the weights that were there before
        super()._load_from_state_dict(state_dict, prefix, *args, **kwargs)

    def _experts(self, xs, offsets):
        gate, up = grouped_gemm(xs, self.w_gate_up, offsets).split(self.ffn, 1)
        return grouped_gemm(torch.nn.functional.silu(gate) * up, self.w_down, offsets)

    def _experts_fp8(self, xs, offsets):
        w_gate_up, s_gate_up, w_down, s_down = self._fp8
        gate, up = grouped_gemm_fp8_block(*quantize_fp8_block(xs), w_gate_up, s_gate_up, offsets).split(self.ffn, 1)
        return grouped_gemm_fp8_block(*quantize_fp8_block(torch.nn.functional.silu(gate) * up), w_down, s_down, offsets)

    def forward(self, x, gate_logits=None, precision=None):
        if precision not in (None, 'fp8'):
            raise ValueError(f"precision is None (the layer's own) or 'fp8' (got {precision!r})")
        if precision == 'fp8':
            if self._fp8 is None:
                raise RuntimeError('call quantize() before a forward pass in fp8')
            with torch.no_grad():
                return self._forward(x, gate_logits, self._experts_fp8)
        return self._forward(x, gate_logits, self._experts)

    def _forward(self, x, gate_logits, run_experts):
        if gate_logits is None:
            gate_logits = x @ self.w_router.t()
        experts, weights = route_top_k(gate_logits, self.topk)
        order = sort_copies(experts, self.num_experts)
        return combine_rows(run_experts(gather_rows(x, order), order.offsets), weights, order)
