"""Embedding lookup: rows of a table by token, and the table's gradient by sorted tokens, through dg_embedding_lookup /
dg_embedding_grad (embedding.hip).  AppearanceEmbedding (dogs_amd.masks) reads a batch of views' codes with it.

    Y[i] = scale E[t_i]        dE[v] = scale sum over i with t_i = v of dY[i]

The gradient's sums run in an order that only the tokens set, in 32 bits and without atomics: the same bits every time
(torch's own backward of an index adds with atomics)."""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}     # dogs_hip.h DG_F32, DG_F16, DG_BF16
_WIDE = {torch.int64: 1, torch.int32: 0}


def _lookup(table: torch.Tensor, tokens: torch.Tensor, scale: float) -> torch.Tensor:
    v, d = table.shape
    out = table.new_empty((*tokens.shape, d))
    _lib.launch(_lib.load().dg_embedding_lookup, table.get_device(), table.data_ptr(), _DTYPES[table.dtype], v, d,
                table.stride(0), table.stride(1), tokens.data_ptr(), _WIDE[tokens.dtype], tokens.numel(), scale,
                out.data_ptr())
    return out


def _table_grad(ctx, g):
    _lib.refuse_unrecorded("embedding_lookup's gradient", (g,))
    tokens, = ctx.saved_tensors
    v, d, scale, padding = ctx.call
    if g.is_neg():
        g = g.resolve_neg()
    if not g.is_contiguous():
        g = g.contiguous()
    dtype, n = _DTYPES[g.dtype], tokens.numel()
    L = _lib.load()
    dtable = g.new_empty((v, d))
    nbytes = L.dg_embedding_grad_scratch_bytes(v, d, n, dtype) if n > 1024 else 0     # few tokens need none
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=g.device) if nbytes else None
    _lib.launch(L.dg_embedding_grad, g.get_device(), g.data_ptr(), dtype, tokens.data_ptr(), _WIDE[tokens.dtype], n, v, d,
                scale, padding, dtable.data_ptr(), scratch.data_ptr() if nbytes else None, nbytes)
    return dtable, None, None, None


class _EmbeddingLookup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, tokens, scale, padding):
        ctx.save_for_backward(tokens)
        ctx.call = (*table.shape, scale, padding)
        return _lookup(table, tokens, scale)

    @staticmethod
    def backward(ctx, g):
        if torch.is_grad_enabled():    # create_graph: a second derivative would be missing this node's
            return _table_grad_once(ctx, g)
        return _table_grad(ctx, g)


_table_grad_once = once_differentiable(_table_grad)


def embedding_lookup(table: torch.Tensor, tokens: torch.Tensor, scale: float = 1.0,
                     padding_idx: int | None = None) -> torch.Tensor:
    """scale * table[tokens] of shape [*tokens.shape, D] in table's type, differentiable (once) w.r.t. table.

    table: [V, D] float32, float16 or bfloat16 on a HIP device, any strides; tokens: int32 or int64 of any shape on the
    same device, or on the host.  Products and sums are 32-bit and round once.  padding_idx (negative: from the end) is
    a row that gets no gradient; its lookup is like any other's.

    Tokens outside [0, V) are an IndexError where tokens is on the host.  On the device reading them back would stall
    the stream: there such a token reads nothing, its row of the result is NaN, and it adds nothing to the gradient.

    Forward-mode tangents, of the table or of the result's gradient, and torch.jit.trace are refused.

    The gradient is dense, in table's type, with every row written.  Lookup and backward may be captured into a graph, the
    backward only while no graph of the same table that was built outside the capture is alive (autograd would join
    the two streams)."""
    if not table.is_cuda or table.dim() != 2 or table.dtype not in _DTYPES:
        _lib.require_device(table, "table")
        raise RuntimeError(f"embedding_lookup: table must be [V, D] float32, float16 or bfloat16, got "
                           f"{tuple(table.shape)} {table.dtype}")
    _lib.refuse_unrecorded("embedding_lookup", (table,))
    if table.is_neg():      # a view of a conjugate's imaginary part: its memory holds the other sign
        table = table.resolve_neg()
    if tokens.dtype not in _WIDE:
        raise RuntimeError(f"embedding_lookup: tokens must be int32 or int64, got {tokens.dtype}")
    if tokens.get_device() != table.get_device():
        tokens = _to_device(tokens, table)
    if not tokens.is_contiguous():
        tokens = tokens.contiguous()
    if isinstance(scale, torch.Tensor):
        raise RuntimeError("embedding_lookup: scale must be a number (it gets no gradient)")
    padding = -1
    if padding_idx is not None:
        v = table.shape[0]
        if not -v <= padding_idx < v:
            raise IndexError(f"embedding_lookup: padding_idx {padding_idx} is outside the table's {v} rows")
        padding = padding_idx % v
    if table.requires_grad and torch.is_grad_enabled():
        return _EmbeddingLookup.apply(table, tokens, float(scale), padding)
    return _lookup(table, tokens, float(scale))


def _to_device(tokens: torch.Tensor, table: torch.Tensor) -> torch.Tensor:
    v = table.shape[0]
    if tokens.device.type != "cpu":
        raise RuntimeError(f"embedding_lookup: tokens is on {tokens.device}, table on {table.device}")
    if tokens.numel() and not (int(tokens.min()) >= 0 and int(tokens.max()) < v):
        raise IndexError(f"embedding_lookup: a token is outside [0, {v})")
    return tokens.to(table.device)
