"""Embedding of species (or any labels) by id: scaled rows of a table, with the gradient of the table from sorted ids.

The reference multiplies one-hot species by the weight of a Linear (models/latticeformer.py:224); the same rows come from a
lookup, ``embed_species(ids, linear.weight.t())``, which reads the weight where it lies.  ``Latticeformer`` calls it for a
batch that holds species ids ``data.z`` instead of one-hot rows ``data.x``."""
from __future__ import annotations

from torch import Tensor

from . import _lib


def embed_species(ids: Tensor, table: Tensor, scale: float = 1.0) -> Tensor:
    """``scale * table[ids]``, (*ids.shape, D), in the table's type (float32, bfloat16 or float16; any strides).  Ids outside
    [0, V), -1 for instance, stand for padding: rows of zeros that have no part in the gradient.  The gradient of the table is
    dense, of the layout of the table (the transposed weight of a Linear gets the gradient of that weight without a copy), and the
    same bits every time."""
    return _lib.torch_ops().embed(ids, table, scale)
