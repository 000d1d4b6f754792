"""Layers on 16-bit weights (float16 or bfloat16): a linear with its activation, the gated half of an MLP and a mixture of experts.

What a quantised model leaves in 16 bits (output head, routers) and models that are not quantised.  Parameters are named as an unquantised
directory names them (`.weight`, `.bias`; `e1_e3.weight` and `e2.weight` of an expert layer).  As in MixtralMoE the router's logits come
from the caller.
"""

from __future__ import annotations

from typing import Optional

import torch
from torch import nn

from .. import ops
from ..quantization import MixtralExperts


class DenseLinear(nn.Module):
    """y = act(x . W^T (+ bias)) (+ residual); activation and out_dtype as in ops.dense_linear."""

    gated = False

    def __init__(self, in_features: int, out_features: int, bias: bool = True, activation: Optional[str] = None,
                 dtype: torch.dtype = torch.float16, out_dtype: Optional[torch.dtype] = None, device=None):
        super().__init__()
        self.in_features = in_features
        self.out_features = out_features
        self.activation = activation
        self.out_dtype = out_dtype
        rows = 2 * out_features if self.gated else out_features
        self.weight = nn.Parameter(torch.zeros((rows, in_features), dtype=dtype, device=device), requires_grad=False)
        self.bias = nn.Parameter(torch.zeros((rows,), dtype=dtype, device=device), requires_grad=False) if bias else None

    @classmethod
    def from_linear(cls, src: nn.Linear, activation: Optional[str] = None, out_dtype: Optional[torch.dtype] = None):
        """The layer on src's own parameters (of a gated one: gate rows, then up rows)."""
        rows, k = src.weight.shape
        if cls.gated and rows % 2:
            raise ValueError(f"{rows} rows cannot be split into gate and up halves")
        layer = cls(k, rows // 2 if cls.gated else rows, src.bias is not None, activation, src.weight.dtype, out_dtype, device="meta")
        layer.weight = nn.Parameter(src.weight.detach(), requires_grad=False)
        if src.bias is not None:
            layer.bias = nn.Parameter(src.bias.detach(), requires_grad=False)
        return layer

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        return ops.dense_linear(x, self.weight, self.bias, self.activation, residual, self.out_dtype)


class DenseGatedLinear(DenseLinear):
    """act(gate) * up of the halves of x . W^T (+ bias), W [2 out_features, in_features]."""

    gated = True

    def __init__(self, in_features: int, out_features: int, bias: bool = True, activation: Optional[str] = "silu",
                 dtype: torch.dtype = torch.float16, out_dtype: Optional[torch.dtype] = None, device=None):
        super().__init__(in_features, out_features, bias, activation, dtype, out_dtype, device)

    @classmethod
    def from_linear(cls, src: nn.Linear, activation: Optional[str] = "silu", out_dtype: Optional[torch.dtype] = None):
        return super().from_linear(src, activation, out_dtype)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return ops.dense_linear_gated(x, self.weight, self.bias, self.activation, self.out_dtype)


class DenseMoE(nn.Module):
    """Experts act(x W1^T) * (x W3^T) . W2^T behind a softmax or sigmoid router, its choice limited to the best groups of experts where
    num_groups says so; score_bias (float32) moves the choice and not the weights.

    The layer is one for a few tokens: more than ops.DENSE_MOE_TOKENS are taken that many at a time, each with its experts' weights read
    again."""

    def __init__(self, hidden_size: int, intermediate_size: int, num_local_experts: int, num_experts_per_tok: int,
                 activation: str = "silu", scoring: str = "softmax", score_bias: bool = False, num_groups: int = 1, top_groups: int = 1,
                 renormalize: bool = True, routed_scale: float = 1.0, dtype: torch.dtype = torch.float16, device=None):
        super().__init__()
        self.num_experts_per_tok = num_experts_per_tok
        self.num_local_experts = num_local_experts
        self.activation = activation
        self.routing = {"scoring": scoring, "num_groups": num_groups, "top_groups": top_groups, "renormalize": renormalize,
                        "scale": routed_scale}
        self.e1_e3 = MixtralExperts(num_local_experts, hidden_size, 2 * intermediate_size, device=device).to(dtype)
        self.e2 = MixtralExperts(num_local_experts, intermediate_size, hidden_size, device=device).to(dtype)
        self.score_bias = nn.Parameter(torch.zeros((num_local_experts,), dtype=torch.float32, device=device), requires_grad=False) \
            if score_bias else None

    def _apply(self, fn, recurse=True):  # a cast of the model (.half(), .to(dtype)) leaves the choice's bias in float32
        before = None if self.score_bias is None else self.score_bias.data
        super()._apply(fn, recurse)
        if before is not None and self.score_bias.dtype != before.dtype:
            self.score_bias.data = before.to(self.score_bias.device)
        return self

    def forward(self, x: torch.Tensor, gate: torch.Tensor) -> torch.Tensor:
        """x [..., hidden]; gate [tokens, num_local_experts] router logits."""
        tokens = x.reshape(-1, x.shape[-1]).contiguous()
        if isinstance(gate, torch.Tensor) and tuple(gate.shape) != (len(tokens), self.num_local_experts):  # (a run of it would hide further rows)
            raise ValueError(f"gate {tuple(gate.shape)} for {len(tokens)} tokens of {self.num_local_experts} experts")
        most = ops.DENSE_MOE_TOKENS
        parts = [(tokens[i : i + most], gate[i : i + most]) for i in range(0, max(len(tokens), 1), most)]
        out = [ops.dense_moe(t, g, self.e1_e3.weight, self.e2.weight, self.num_experts_per_tok, activation=self.activation,
                             bias=self.score_bias, **self.routing) for t, g in parts]
        return (out[0] if len(out) == 1 else torch.cat(out)).reshape(x.shape)
