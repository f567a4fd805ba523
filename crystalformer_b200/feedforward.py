"""Gated feed-forward block, in float32, bfloat16 and float16: both projections, the activation and the product in one kernel, the
projection back in another; the backward likewise, without keeping the hidden features.

``gated_feed_forward`` is the operator; ``GatedFeedForward`` holds the parameters of a layer.  The encoder takes the block in
place of its two Linears (models/indexed_latticeformer_encoder.py:884-890) where its ``activation`` is ``"swiglu"``, ``"geglu"`` or
``"reglu"``."""
from __future__ import annotations

from typing import Optional

from torch import Tensor
from torch.nn import Linear, Module

from . import _lib, ops

#: activation of the encoder -> of the gate
GATES = {"swiglu": "silu", "geglu": "gelu", "reglu": "relu"}


def gated_feed_forward(x: Tensor, w_gate: Tensor, w_up: Tensor, w_down: Tensor, b_gate: Optional[Tensor] = None, b_up: Optional[Tensor] = None,
                       b_down: Optional[Tensor] = None, activation: str = "silu") -> Tensor:
    """``(act(x w_gate^T + b_gate) * (x w_up^T + b_up)) w_down^T + b_down`` with the weights of Linears, (F,D), (F,D) and (D,F);
    x (..., D); ``activation``: "silu", "gelu" (the exact one) or "relu".  All of one type; of any sizes.  float32 has float32's
    accuracy (operands in three pieces on the tensor cores, which hold values down to 1e-33 whole; infinities, and sums beyond the range,
    may come out as NaN where they meet values beyond 256); of 16-bit types the hidden features and their gradients are rounded to
    the type once (forward of up to eight rows: not at all, or to twice its digits), sums are float32; float16 has its range too: hidden
    features beyond 65,504 overflow (of up to eight rows: beyond 131,008 at the earliest), and hidden gradients below 6e-5 lose digits
    (scale the loss, as elsewhere in float16).  The backward computes the hidden features again instead of keeping them."""
    return _lib.torch_ops().gated(x, w_gate, w_up, w_down, b_gate, b_up, b_down, ops.gate_code(activation))


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
