"""Gated feed-forward block, in float32, bfloat16 and float16: both projections, the activation and the product in one kernel, the
projection back in another; the backward likewise, without keeping the hidden features.

``gated_feed_forward`` is the operator; ``GatedFeedForward`` holds the parameters of a layer.  The encoder takes the block in
place of its two Linears (models/indexed_latticeformer_encoder.py:884-890) where its ``activation`` is ``"swiglu"``, ``"geglu"`` or
``"reglu"``."""
from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor
from torch.nn import Linear, Module

from . import ops

#: activation of the encoder -> of the gate
GATES = {"swiglu": "silu", "geglu": "gelu", "reglu": "relu"}


class GatedFeedForwardFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, b_gate, b_up, b_down, activation: str):
        ctx.save_for_backward(x, w_gate, w_up, w_down, b_gate, b_up, b_down)
        ctx.activation = activation
        return ops.gated_ffn_fwd(x, w_gate, w_up, w_down, b_gate, b_up, b_down, activation)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gy):
        return (*ops.gated_ffn_bwd(*ctx.saved_tensors, ctx.activation, gy, ctx.needs_input_grad[:7]), None)


def gated_feed_forward(x: Tensor, w_gate: Tensor, w_up: Tensor, w_down: Tensor, b_gate: Optional[Tensor] = None, b_up: Optional[Tensor] = None,
                       b_down: Optional[Tensor] = None, activation: str = "silu") -> Tensor:
    """``(act(x w_gate^T + b_gate) * (x w_up^T + b_up)) w_down^T + b_down`` with the weights of Linears, (F,D), (F,D) and (D,F);
    x (..., D); ``activation``: "silu", "gelu" (the exact one) or "relu".  All of one type; of any sizes.  float32 has float32's
    accuracy (operands in three pieces on the tensor cores); of 16-bit types the hidden features and their gradients are rounded to
    the type once, sums are float32.  The backward computes the hidden features again instead of keeping them."""
    shape = x.shape
    if x.dim() != 2:
        x = x.reshape(-1, shape[-1]) if x.dim() > 0 else x
    leaves = (x, w_gate, w_up, w_down, b_gate, b_up, b_down)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in leaves):
        y = GatedFeedForwardFunction.apply(*leaves, activation)
    else:
        y = ops.gated_ffn_fwd(*leaves, activation)
    return y if len(shape) == 2 else y.view(shape)


class GatedFeedForward(Module):
    """The block with its parameters: Linears ``gate`` and ``up`` (dim -> hidden) and ``down`` (hidden -> dim)."""

    def __init__(self, dim: int, hidden: int, activation: str = "silu", bias: bool = True, device=None, dtype=None):
        super().__init__()
        if activation not in ops.GATE_CODES:
            raise ValueError(f"activation {activation!r} is none of {', '.join(ops.GATE_CODES)}")
        self.activation = activation
        self.gate, self.up = (Linear(dim, hidden, bias, device=device, dtype=dtype) for _ in range(2))
        self.down = Linear(hidden, dim, bias, device=device, dtype=dtype)

    def forward(self, x: Tensor) -> Tensor:
        return gated_feed_forward(x, self.gate.weight, self.up.weight, self.down.weight, self.gate.bias, self.up.bias, self.down.bias,
                                  self.activation)
