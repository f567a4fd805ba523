"""Norms of the query and key heads and their rotation by positions, in one pass forward and one backward.

``normalize_rotate`` is the operator; ``QKNorm`` holds the weights and waves of a layer (``LatticeformerParams.qk_norm`` and
``qk_rotation``).  In a crystal the positions are fractional coordinates and the waves whole numbers: the rotated q_i . k_j then
depends on the difference of the fractional coordinates modulo lattice vectors, as everything in a crystal does."""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch import Tensor
from torch.nn import Module, Parameter

from . import _lib


def normalize_rotate(q: Tensor, k: Tensor, wq: Optional[Tensor] = None, wk: Optional[Tensor] = None, pos: Optional[Tensor] = None,
                     waves: Optional[Tensor] = None, eps: float = 1e-6, interleaved: bool = False) -> Tuple[Tensor, Tensor]:
    """q (N,Hq,D) and k (N,Hk,D), Hq a multiple of Hk, each head divided by its root mean square (of its D entries, ``eps``
    added to the mean), times the weights (D,) or (H,D), if given; then, with ``pos`` (N,C) and ``waves`` (1 or Hk, P, C), both
    float32, turned: pair p of a head - entries (p, P + p), ``interleaved`` (2p, 2p + 1) - by 2 pi pos . waves[h, p].  Entries from
    2 P on are not turned.  Waves count cycles per unit of position and angles keep their accuracy at any distance.  q and k may
    be strided views (of a joint projection); outputs are contiguous, of their type (float32, bfloat16 or float16).  Gradients: of
    q, k and the weights; positions and waves that ask for one are refused."""
    return _lib.torch_ops().normalize_rotate(q, k, wq, wk, pos, waves, eps, interleaved)


def shortest_waves(heads: int, pairs: int) -> Tensor:
    """(heads, pairs, 3) whole-numbered waves, all different: the shortest of the lattice, one of each {n, -n}, dealt to the heads in
    turn."""
    reach = 1
    while ((2 * reach + 1) ** 3 - 1) // 2 < heads * pairs:
        reach += 1
    reach += 1  # (the shortest lie in a ball, not in a cube)
    r = torch.arange(-reach, reach + 1)
    n = torch.cartesian_prod(r, r, r)
    first = (n[:, 0] > 0) | ((n[:, 0] == 0) & ((n[:, 1] > 0) | ((n[:, 1] == 0) & (n[:, 2] > 0))))
    n = n[first]
    n = n[torch.argsort((n * n).sum(1), stable=True)][:heads * pairs]
    return n.reshape(pairs, heads, 3).transpose(0, 1).float().contiguous()


class QKNorm(Module):
    """Weights (H, D) of the query and key norms of a layer, ones to begin with, and, with ``pairs`` > 0, its waves."""

    def __init__(self, heads: int, head_dim: int, pairs: int = 0, eps: float = 1e-6, device=None, dtype=None):
        super().__init__()
        if pairs < 0 or 2 * pairs > head_dim:
            raise ValueError(f"{pairs} pairs in heads of {head_dim}")
        self.eps = eps
        self.q_weight = Parameter(torch.ones((heads, head_dim), device=device, dtype=dtype))
        self.k_weight = Parameter(torch.ones((heads, head_dim), device=device, dtype=dtype))
        self.register_buffer("waves", shortest_waves(heads, pairs).to(device=device) if pairs > 0 else None)

    def forward(self, q: Tensor, k: Tensor, pos: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
        if self.waves is not None and pos is None:
            raise ValueError("the rotation needs positions")
        if self.waves is None:
            return normalize_rotate(q, k, self.q_weight, self.k_weight, eps=self.eps)
        # (a module that was converted holds its waves in 16 bits: small whole numbers, the same ones)
        return normalize_rotate(q, k, self.q_weight, self.k_weight, pos, self.waves.float(), self.eps)
