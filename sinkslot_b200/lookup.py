"""Rows of a learned table by index, and the table's gradient.

The points of a cloud (or the inputs of a model) are often rows of a table that
is trained: ``embedding_lookup(table, index, scale)`` gives them, and its
backward pass sums each row's gradients in the order of the tokens that name it,
so that training is reproducible run to run, as the rest of the package is.
"""

from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import call, dtype_code, on_device, ptr, stream_of


def _lookup_impl(table, index, scale):
    """The body of the ``sinkslot_b200::lookup`` operator."""
    dev = table.device
    out = torch.empty((index.numel(), table.shape[1]), dtype=table.dtype, device=dev)
    with on_device(dev):
        call("sinkslot_lookup", ptr(table), dtype_code(table), table.stride(0), table.shape[0],
             table.shape[1], ptr(index), index.element_size(), index.numel(), scale, ptr(out),
             stream_of(dev))
    return out


def _lookup_grad_impl(grad_out, index, rows, scale, padding):
    """The body of the ``sinkslot_b200::lookup_grad`` operator."""
    dev = grad_out.device
    if grad_out.stride(1) != 1:
        grad_out = grad_out.contiguous()
    dim = grad_out.shape[1]
    nb = _lib.out_i64()
    call("sinkslot_lookup_grad_workspace_bytes", index.numel(), rows, dim, ctypes.byref(nb))
    ws = torch.empty(nb.value, dtype=torch.uint8, device=dev)
    out = torch.empty((rows, dim), dtype=grad_out.dtype, device=dev)
    with on_device(dev):
        call("sinkslot_lookup_grad", ptr(grad_out), dtype_code(grad_out), grad_out.stride(0),
             ptr(index), index.element_size(), index.numel(), rows, dim, scale, padding, ptr(out),
             ptr(ws), ws.numel(), stream_of(dev))
    return out


class _LookupFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, index, scale, padding):
        ctx.save_for_backward(index)
        ctx.args = (table.shape[0], scale, padding)
        return torch.ops.sinkslot_b200.lookup(table, index, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        index, = ctx.saved_tensors
        rows, scale, padding = ctx.args
        return torch.ops.sinkslot_b200.lookup_grad(g, index, rows, scale, padding), None, None, None


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
    name = "embedding_lookup"
    if table.dim() != 2 or table.shape[0] < 1 or table.shape[1] < 1:
        raise ValueError(f"{name}: table must be (rows, dim), got {tuple(table.shape)}")
    _lib.require_cuda(name, table, index)
    _lib.require_dtype(name, "table", table)
    _lib.require_index(name, "index", index)
    rows = table.shape[0]
    if rows >= 1 << 31 or index.numel() >= 1 << 31:
        raise ValueError(f"{name}: 2^31 rows or tokens and more are not supported")
    padding = -1
    if padding_index is not None:
        if not -rows <= padding_index < rows:
            raise ValueError(f"{name}: padding_index {padding_index} is outside the table of "
                             f"{rows} rows")
        padding = padding_index % rows
    if table.stride(1) != 1:
        table = table.contiguous()
    flat = index.reshape(-1).contiguous()
    out = _LookupFn.apply(table, flat, float(scale), padding)
    return out if index.dim() == 1 else out.view(*index.shape, table.shape[1])
