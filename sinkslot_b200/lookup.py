"""Rows of a learned table by index, and the table's gradient.

The points of a cloud (or the inputs of a model) are often rows of a table that
is trained: ``embedding_lookup(table, index, scale)`` gives them, and its
backward pass sums each row's gradients in the order of the tokens that name it,
so that training is reproducible run to run, as the rest of the package is.
"""

from __future__ import annotations

from typing import Optional

import torch

from ._lib import torch_ops


def embedding_lookup(table: torch.Tensor, index: torch.Tensor, scale: float = 1.0,
                     padding_index: Optional[int] = None) -> torch.Tensor:
    """``scale * table[index]``, differentiable in ``table``.

    ``table``: (rows, dim), float32, float16 or bfloat16; its rows may lie apart
    (a view of a wider table).  ``index``: int32 or int64, any shape; the result
    has that shape with ``dim`` behind it.  Tokens equal to ``padding_index`` are
    looked up like the others and give no gradient.  An index outside
    ``[0, rows)`` gives a row of NaN and no gradient (the values are on the
    device; checking them would wait for it).

    The gradient is dense and of the table's type: each row's sum is taken in
    float32 in token order and rounded once.
    """
    return torch_ops().embedding_lookup(table, index, scale, padding_index)
