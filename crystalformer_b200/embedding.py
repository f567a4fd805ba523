"""Embedding of species (or any labels) by id: scaled rows of a table, with the gradient of the table from sorted ids.

The reference multiplies one-hot species by the weight of a Linear (models/latticeformer.py:224); the same rows come from a
lookup, ``embed_species(ids, linear.weight.t())``, which reads the weight where it lies.  ``Latticeformer`` calls it when
``data.x`` holds species ids instead of one-hot rows."""
from __future__ import annotations

import torch
from torch import Tensor

from . import ops


class SpeciesEmbeddingFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table: Tensor, ids: Tensor, scale: float) -> Tensor:
        ctx.save_for_backward(ids)
        ctx.how = table.shape[0], scale, table.stride(0) < table.stride(1)
        return ops.embed_fwd(ids, table, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gout: Tensor):
        V, scale, transposed = ctx.how
        (ids,) = ctx.saved_tensors
        return ops.embed_bwd(ids, gout, V, scale, transposed), None, None


def embed_species(ids: Tensor, table: Tensor, scale: float = 1.0) -> Tensor:
    """``scale * table[ids]``, (*ids.shape, D), in the table's type (float32, bfloat16 or float16; any strides).  Ids outside
    [0, V), -1 for instance, stand for padding: rows of zeros that have no part in the gradient.  The gradient of the table is
    dense, of the layout of the table (the transposed weight of a Linear gets the gradient of that weight without a copy), and the
    same bits every time."""
    if torch.is_grad_enabled() and table.requires_grad:
        return SpeciesEmbeddingFunction.apply(table, ids, float(scale))
    return ops.embed_fwd(ids, table, float(scale))
