"""Rows of a learned node-embedding table, scaled, and the table's gradient.

The reference trains on given features only (its feature caches,
TAC_training_backend/spmm_cnic/src/core/spmm_kernel.cu:129-153); graphs
without node features learn a row per node instead.  ``embedding`` reads such
rows by index -- a sampled block's input nodes (``minibatch.embedding_rows``),
the endpoints of edges, node or edge types -- and its backward writes the dense
gradient of the table, each row the sum over its indices in ascending order of
their position, so the same call gives the same bits.

``partition.gather_rows`` packs fp32 rows for the halo exchange; here tables are
fp32, fp16 or bf16 of any width and stride, indices int32 or int64, rows scaled,
padded and differentiable.
"""
from __future__ import annotations

import torch

from . import _lib as L
from ._args import TYPES, launch, rows_of, scratch_for, tracked, type_code

_INDEX = {torch.int32: L.I32, torch.int64: L.I64}


def _index(idx: torch.Tensor, device: torch.device):
    code = _INDEX.get(idx.dtype)
    if code is None:
        raise TypeError(f"indices must be int32 or int64, not {idx.dtype}")
    if idx.device != device:
        raise ValueError("indices must be on the rows' device")
    return idx if idx.is_contiguous() else idx.contiguous(), code


def _padding(padding_idx) -> int:
    if not L.NO_PADDING < padding_idx < 1 << 63:
        raise ValueError("padding_idx must lie between -2^63 and 2^63")
    return padding_idx


def _bad_flag(bad, device):
    if bad.dtype != torch.int32 or bad.device != device or bad.numel() < 1:
        raise ValueError("bad must be an int32 tensor of one element on the rows' device")
    return bad.data_ptr()


def _flag_bad(idx, num_rows: int, padding_idx, bad) -> None:
    """What a call that launches nothing (no columns, or no rows to write) has to say of its indices."""
    if bad is None or idx.numel() == 0:
        return
    outside = (idx < 0) | (idx >= num_rows)
    if padding_idx is not None:
        outside &= idx != padding_idx
    bad.as_strided((1,), (1,)).bitwise_or_(outside.any())  # the word at its address, whatever its shape


def _lookup(table, idx, scale, padding_idx, out_dtype, bad):
    code = type_code(table, "table")
    if table.dim() != 2:
        raise ValueError("the table must be 2-D")
    num_rows, width = table.shape
    ld, col = table.stride()
    if width > 1 and col != 1:
        raise ValueError("the table must have unit column stride")
    if num_rows < 2:
        ld = max(width, 1)
    if out_dtype is None or out_dtype == table.dtype:
        out_dtype, out_code = table.dtype, code
    elif out_dtype == torch.float32:
        out_code = L.F32
    else:
        raise TypeError("out_dtype must be the table's or float32")
    device = table.device
    idx, idx_code = _index(idx, device)
    out = torch.empty((*idx.shape, width), dtype=out_dtype, device=device)
    n = idx.numel()
    padding = L.NO_PADDING if padding_idx is None else _padding(padding_idx)
    flag = None if bad is None else _bad_flag(bad, device)
    if n and width:
        launch(device, "tcc_embedding_forward", table.data_ptr(), code, ld, num_rows, idx.data_ptr(), idx_code, n,
               padding, scale, out.data_ptr(), out_code, width, width, flag)
    else:
        _flag_bad(idx, num_rows, padding_idx, bad)
    return out


def embedding_backward(grad_out: torch.Tensor, idx: torch.Tensor, num_rows: int, scale: float = 1.0,
                       padding_idx: int | None = None, dtype: torch.dtype | None = None,
                       bad: torch.Tensor | None = None) -> torch.Tensor:
    """Gradient [num_rows, F] of a table for ``embedding``'s output gradient
    ``grad_out`` [*idx.shape, F]: scale * the sum of the rows of each index.
    Not differentiable itself.
    ``dtype``: the table's type (default grad_out's); ``bad`` as in ``embedding``."""
    code = type_code(grad_out, "grad_out")
    dtype = grad_out.dtype if dtype is None else dtype
    if dtype not in TYPES or (dtype != grad_out.dtype and code != L.F32):
        raise TypeError("grad_out must have the table's type or be float32")
    if grad_out.shape[:-1] != idx.shape:
        raise ValueError("grad_out must have one row per index")
    if num_rows < 0:
        raise ValueError("num_rows must not be negative")
    device, width = grad_out.device, grad_out.shape[-1]
    idx, idx_code = _index(idx, device)
    grad_out, ld = rows_of(grad_out, width)
    out = torch.empty((num_rows, width), dtype=dtype, device=device)
    padding = L.NO_PADDING if padding_idx is None else _padding(padding_idx)
    flag = None if bad is None else _bad_flag(bad, device)
    if out.numel():
        n = idx.numel()
        nbytes = L.lib().tcc_embedding_backward_scratch_bytes(n, num_rows, width)
        hold, scratch = scratch_for(nbytes, device)
        launch(device, "tcc_embedding_backward", grad_out.data_ptr(), code, ld, idx.data_ptr(), idx_code, n,
               padding, scale, out.data_ptr(), TYPES[dtype], width, num_rows, width, scratch, nbytes, flag)
    else:
        _flag_bad(idx, num_rows, padding_idx, bad)
    return out


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, idx, scale, padding_idx, out_dtype, bad):
        ctx.save_for_backward(idx)
        ctx.args = (table.shape[0], scale, padding_idx, table.dtype)
        return _lookup(table, idx, scale, padding_idx, out_dtype, bad)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        (idx,) = ctx.saved_tensors
        num_rows, scale, padding_idx, dtype = ctx.args
        grad = embedding_backward(grad_out, idx, num_rows, scale, padding_idx, dtype)
        return grad, None, None, None, None, None


def embedding(table: torch.Tensor, idx: torch.Tensor, scale: float = 1.0, padding_idx: int | None = None,
              out_dtype: torch.dtype | None = None, bad: torch.Tensor | None = None) -> torch.Tensor:
    """scale * table[idx] ([*idx.shape, F]), differentiable in the table (in reverse mode).

    ``padding_idx`` (any value, e.g. -1 for the filled-up end of a block): its
    rows are zero and give no gradient.  ``out_dtype``: the table's type
    (default) or float32, which the aggregation takes.  An index outside the
    table gives a zero row, no gradient, and sets ``bad`` (an int32 CUDA tensor,
    optional) to 1."""
    if tracked(table):
        return _Embedding.apply(table, idx, scale, padding_idx, out_dtype, bad)
    return _lookup(table, idx, scale, padding_idx, out_dtype, bad)


class NodeEmbedding(torch.nn.Module):
    """A learned row per node (or per node or edge type), read by index; ``bad`` as in ``embedding``."""

    def __init__(self, num_rows: int, width: int, scale: float = 1.0, padding_idx: int | None = None,
                 dtype: torch.dtype | None = None, out_dtype: torch.dtype | None = None, device=None):
        super().__init__()
        self.weight = torch.nn.Parameter(torch.empty(num_rows, width, dtype=dtype, device=device))
        torch.nn.init.normal_(self.weight)
        self.scale, self.padding_idx, self.out_dtype = scale, padding_idx, out_dtype

    def forward(self, idx: torch.Tensor, bad: torch.Tensor | None = None) -> torch.Tensor:
        return embedding(self.weight, idx, self.scale, self.padding_idx, self.out_dtype, bad)
