"""Rows of a table by token, scaled, with the table's gradient: the entry of features that are categories or node numbers
(graphs without a feature matrix), which the reference's model, a Linear layer on float features
(src/SpectralTrainer.py:28-39), does not have.

The gradient sorts the tokens and sums every row's places in one fixed order, so runs repeat bit for bit and a row that
thousands of places share is no queue of atomics.  It is dense: all rows of the table, zeros included, in one pass."""
from __future__ import annotations

import torch
import torch.nn as nn
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from ._lib import lib, load_autograd
from .graph import launch, require_gpu

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}   # SPARC_F32, SPARC_BF16, SPARC_F16
_ID_DTYPES = {torch.int32: 0, torch.int64: 1}


def refuse_forward_mode(what: str, tensors) -> None:
    """Raises inside a dual level where a tensor carries a tangent: the kernels know nothing of it and it would be lost."""
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{what} has no forward-mode derivative")


def _tokens(ids: torch.Tensor, device) -> torch.Tensor:
    if not torch.is_tensor(ids) or ids.dtype not in _ID_DTYPES:
        raise ValueError("ids must be an int32 or int64 tensor")
    if ids.device != device:
        raise ValueError(f"ids are on {ids.device}, the values on {device}")
    return ids if ids.is_contiguous() else ids.contiguous()


def _rows_of(t: torch.Tensor, what: str) -> int:
    """Row stride of a matrix whose rows are contiguous."""
    if t.dtype not in DTYPES:
        raise ValueError(f"{what} must be float32, bfloat16 or float16, not {t.dtype}")
    if t.dim() == 2:
        rows, dim = t.shape
        ld, step = t.stride()
        if (ld >= dim or rows <= 1) and (step == 1 or dim <= 1):
            return ld if ld > dim else max(dim, 1)
    raise ValueError(f"{what} must be a matrix with contiguous rows that do not overlap")


def _padding(padding_idx, rows: int) -> int:
    if padding_idx is None:
        return -1
    if not 0 <= int(padding_idx) < rows:
        raise ValueError(f"padding_idx {padding_idx} is no row of a table of {rows}")
    return int(padding_idx)


def _lookup(ids: torch.Tensor, table: torch.Tensor, scale: float) -> torch.Tensor:
    dev = table.device
    if not table.is_cuda:
        require_gpu(dev)
    ids = _tokens(ids, dev)
    ld = _rows_of(table, "table")
    rows, dim = table.shape
    out = table.new_empty((*ids.shape, dim))
    n = ids.numel()
    if n and dim:
        launch("sparc_embedding_fwd", lib.sparc_embedding_fwd, dev, n, rows, dim, DTYPES[table.dtype], ids.data_ptr(),
               _ID_DTYPES[ids.dtype], table.data_ptr(), ld, scale, out.data_ptr(), dim)
    return out


def embedding_grad(ids: torch.Tensor, grad: torch.Tensor, rows: int, scale: float = 1.0, padding_idx=None) -> torch.Tensor:
    """[rows, dim], in grad's type: row v = scale times the sum of grad[i] over the places i with ids[i] = v (grad: the
    shape of ids and one more dimension, dim).  float32 sums, rounded once.  Rows without a place, and row padding_idx,
    are zero; places whose token is no row are left out.  Not differentiable: a grad that requires a gradient (where gradients
    are recorded) or carries a forward-mode tangent raises."""
    if grad.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("embedding_grad is not differentiable: detach grad, or call it under torch.no_grad()")
    refuse_forward_mode("embedding_grad", (grad,))
    dev = grad.device
    if not grad.is_cuda:
        require_gpu(dev)
    ids = _tokens(ids, dev)
    rows = int(rows)
    if rows < 0 or grad.shape[:-1] != ids.shape or grad.dim() == 0:
        raise ValueError(f"a gradient of shape {tuple(grad.shape)} does not belong to ids of shape {tuple(ids.shape)}")
    dim = grad.shape[-1]
    g = grad if grad.dim() == 2 else grad.reshape(ids.numel(), dim)
    if (dim > 1 and g.stride(1) != 1) or (g.shape[0] > 1 and g.stride(0) < dim):   # an expanded gradient
        g = g.contiguous()
    ld = _rows_of(g, "grad")
    pad = -1 if padding_idx is None else _padding(padding_idx, rows)
    out = g.new_empty((rows, dim))
    if rows and dim:
        n, code = ids.numel(), DTYPES[g.dtype]
        nbytes = lib.sparc_embedding_grad_workspace_bytes(n, rows, dim, code)
        at = None
        if nbytes:
            ws = torch.empty(nbytes + 256, dtype=torch.uint8, device=dev)   # of this call alone: streams and graphs share nothing
            at = ws.data_ptr()
            at += (-at) % 256
        launch("sparc_embedding_grad", lib.sparc_embedding_grad, dev, n, rows, dim, code, ids.data_ptr(), _ID_DTYPES[ids.dtype],
               g.data_ptr(), ld, scale, pad, out.data_ptr(), at, nbytes)
    return out


_leaf_stream = load_autograd()


def refuse_capture_beside_eager_graph(leaf: torch.Tensor) -> None:
    """Raises if a node of this leaf lives that was made on the default stream (by whatever operation): the backward that is
    to be captured would let that stream, which cannot be captured, wait for the capture, and the process would end."""
    if leaf.requires_grad and _leaf_stream(leaf) == 0:
        raise RuntimeError(f"a backward is to be captured while an earlier graph of the same parameter, of shape {tuple(leaf.shape)}, "
                           "made on the default stream, is alive. Drop what holds it (its outputs, its loss) before capturing")


class EmbeddingLookup(torch.autograd.Function):
    """Arguments ids, table, scale, padding_idx; gradient for the table."""

    @staticmethod
    def forward(ctx, ids, table, scale, padding_idx):
        out = _lookup(ids, table, scale)
        ctx.save_for_backward(ids)
        ctx.rows, ctx.scale, ctx.padding_idx = table.shape[0], scale, padding_idx
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        (ids,) = ctx.saved_tensors
        if torch.cuda.is_current_stream_capturing():
            leaf = getattr(ctx.next_functions[1][0], "variable", None)   # (None: the table is computed)
            if leaf is not None:
                refuse_capture_beside_eager_graph(leaf)
        return None, embedding_grad(ids, g, ctx.rows, ctx.scale, ctx.padding_idx), None, None


def embedding_lookup(ids: torch.Tensor, table: torch.Tensor, scale: float = 1.0, padding_idx=None) -> torch.Tensor:
    """scale * table[ids], of shape ids.shape + (dim,): ids int32 or int64 of any shape, table [rows, dim] float32, bfloat16
    or float16 with contiguous rows (any row stride).  The product is rounded once.  A token that is no row of the table
    gives a row of NaN (nothing is read, nothing synchronises) and no gradient.  padding_idx: this row is read as any
    other and gets no gradient.  Differentiable once, with respect to the table, in reverse mode; a table with a forward-mode
    tangent raises."""
    if padding_idx is not None:
        _padding(padding_idx, table.shape[0])
    refuse_forward_mode("embedding_lookup", (table,))
    if table.requires_grad and torch.is_grad_enabled():
        return EmbeddingLookup.apply(ids, table, float(scale), padding_idx)
    return _lookup(ids, table, float(scale))


class NodeTable(nn.Module):
    """A learned row per node or category: forward(ids) = embedding_lookup(ids, weight, scale, padding_idx)."""

    def __init__(self, rows: int, dim: int, scale: float = 1.0, padding_idx=None):
        super().__init__()
        if rows < 1 or dim < 1:
            raise ValueError("a table needs at least one row and one column")
        _padding(padding_idx, rows)
        self.scale, self.padding_idx = float(scale), padding_idx
        self.weight = nn.Parameter(torch.randn(rows, dim))
        if padding_idx is not None:
            with torch.no_grad():
                self.weight[padding_idx].zero_()

    def forward(self, ids: torch.Tensor) -> torch.Tensor:
        return embedding_lookup(ids, self.weight, self.scale, self.padding_idx)
