"""Layers on 8-bit block-scaled weights: a linear and a mixture of experts.

Weights are e4m3 with a float32 scale for each block of 128 x 128 (`.q_weight` / `.q_scale`, as the group-quantized
layers name theirs); activations stay in the model dtype outside and are quantised in groups of 128 on the way into a
product.  As in MixtralMoE the router's logits come from the caller.
"""

from __future__ import annotations

from typing import Optional

import torch
from torch import nn

from .. import ops


def _weight(*shape, device=None) -> nn.Parameter:
    # rows a multiple of 16 bytes apart, which the kernels' loads need
    k = shape[-1]
    return nn.Parameter(torch.empty((*shape[:-1], -(-k // 16) * 16), dtype=torch.float8_e4m3fn, device=device)[..., :k], requires_grad=False)


def _rows_apart(t: torch.Tensor) -> torch.Tensor:
    """t, or where its rows are e4m3 and do not lie as _weight's do a copy that does."""
    k = t.shape[-1] if t.dim() > 1 else 0
    if t.dtype != torch.float8_e4m3fn or k % 16 == 0:
        return t
    like = _weight(*t.shape, device="meta")
    if t.stride() == like.stride() and t.untyped_storage().nbytes() - t.storage_offset() >= like.untyped_storage().nbytes():
        return t
    return _weight(*t.shape, device=t.device).data.copy_(t)


def _scale(*shape, device=None) -> nn.Parameter:
    blocks = (*shape[:-2], -(-shape[-2] // ops.FP8_BLOCK), -(-shape[-1] // ops.FP8_BLOCK))
    return nn.Parameter(torch.empty(blocks, dtype=torch.float32, device=device), requires_grad=False)


def _kept(fn, *fixed):
    """fn of a module's _apply, which moves tensors and casts them: the `fixed` ones move and keep their type, which the kernels go by."""

    def apply(t):
        y = fn(t)
        return _rows_apart(t.to(y.device) if y.dtype != t.dtype and any(t is f for f in fixed) else y)

    return apply


class _Fp8Weight(nn.Module):
    """q_weight and q_scale of a linear or a stack of experts, whose types no cast of a model (.half(), .to(dtype)) changes.  A row that is no multiple
    of 16 bytes long stands in a wider one, as a view that torch makes dense where it copies or moves a module; the rows are put apart again there."""

    def __init__(self, *shape, device=None):
        super().__init__()
        self.q_weight = _weight(*shape, device=device)
        self.q_scale = _scale(*shape, device=device)

    def _apply(self, fn, recurse=True):  # .to, .cuda, .to_empty, ...
        return super()._apply(_kept(fn, self.q_weight, self.q_scale), recurse)

    def __setstate__(self, state):  # copy.deepcopy, pickle
        super().__setstate__(state)
        self.q_weight.data = _rows_apart(self.q_weight.data)

    def _load_from_state_dict(self, *args, **kwargs):  # (assign=True takes the given tensors)
        super()._load_from_state_dict(*args, **kwargs)
        self.q_weight.data = _rows_apart(self.q_weight.data)


class Fp8Linear(_Fp8Weight):
    """y = x . W^T (+ bias) (+ residual) with W in e4m3; out_dtype as in ops.fp8_linear."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True, dtype: torch.dtype = torch.float16,
                 out_dtype: Optional[torch.dtype] = None, device=None):
        super().__init__(out_features, in_features, device=device)
        self.in_features = in_features
        self.out_features = out_features
        self.out_dtype = out_dtype
        self.bias = nn.Parameter(torch.empty((out_features,), dtype=dtype, device=device), requires_grad=False) if bias else None

    @staticmethod
    def from_linear(src: nn.Linear, out_dtype: Optional[torch.dtype] = None) -> "Fp8Linear":
        """The layer with src's weight, quantised on its GPU."""
        n, k = src.weight.shape
        layer = Fp8Linear(k, n, src.bias is not None, src.weight.dtype, out_dtype, src.weight.device)
        q, scale = ops.fp8_quantize_weight(src.weight.detach().contiguous())
        layer.q_weight.data, layer.q_scale.data = q, scale
        if src.bias is not None:
            layer.bias.data = src.bias.detach().clone()
        return layer

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        return ops.fp8_linear(x, self.q_weight, self.q_scale, bias=self.bias, out_dtype=self.out_dtype, residual=residual)


class Fp8MoE(nn.Module):
    """Experts silu(x W1^T) * (x W3^T) . W2^T in e4m3 behind a softmax or sigmoid router, its choice limited to the best groups of
    experts where num_groups says so.

    e1_e3 holds gate rows, then up rows, of each expert; score_bias (float32) moves the choice and not the weights."""

    def __init__(self, hidden_size: int, intermediate_size: int, num_local_experts: int, num_experts_per_tok: int,
                 scoring: str = "softmax", score_bias: bool = False, num_groups: int = 1, top_groups: int = 1, renormalize: bool = True,
                 routed_scale: float = 1.0, device=None):
        super().__init__()
        self.num_experts_per_tok = num_experts_per_tok
        self.num_local_experts = num_local_experts
        self.routing = {"scoring": scoring, "num_groups": num_groups, "top_groups": top_groups, "renormalize": renormalize,
                        "scale": routed_scale}
        self.e1_e3 = _Fp8Weight(num_local_experts, 2 * intermediate_size, hidden_size, device=device)
        self.e2 = _Fp8Weight(num_local_experts, hidden_size, intermediate_size, device=device)
        self.score_bias = nn.Parameter(torch.zeros((num_local_experts,), dtype=torch.float32, device=device), requires_grad=False) \
            if score_bias else None

    def _apply(self, fn, recurse=True):
        return super()._apply(_kept(fn, self.score_bias), recurse)

    def load_experts(self, e1_e3: torch.Tensor, e2: torch.Tensor) -> None:
        """Quantise e1_e3 [experts, 2 inter, hidden] and e2 [experts, hidden, inter] (float16, bfloat16 or float32) into the layer."""
        for stack, w in ((self.e1_e3, e1_e3), (self.e2, e2)):
            if tuple(w.shape) != tuple(stack.q_weight.shape):
                raise ValueError(f"weights of {tuple(w.shape)}, expected {tuple(stack.q_weight.shape)}")
            stack.q_weight.data, stack.q_scale.data = ops.fp8_quantize_weight(w)

    def forward(self, x: torch.Tensor, gate: torch.Tensor) -> torch.Tensor:
        """x [..., hidden] float16 or bfloat16; gate [tokens, num_local_experts] router logits."""
        tokens = x.reshape(-1, x.shape[-1]).contiguous()
        y = ops.fp8_moe(tokens, gate, self.e1_e3.q_weight, self.e1_e3.q_scale, self.e2.q_weight, self.e2.q_scale,
                        self.num_experts_per_tok, bias=self.score_bias, **self.routing)
        return y.reshape(x.shape)
