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
    out = torch.empty((*tokens.shape, d), dtype=table.dtype, device=table.device)
    with _lib.device_ctx(table.device):
        _lib.check(_lib.load().dg_embedding_lookup(table.data_ptr(), _DTYPES[table.dtype], v, d, *table.stride(),
                                                   tokens.data_ptr(), _WIDE[tokens.dtype], tokens.numel(), scale,
                                                   out.data_ptr(), _lib.stream_of(table.device)))
    return out


class _EmbeddingLookup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, tokens, scale, padding):
        ctx.save_for_backward(tokens)
        ctx.sizes, ctx.dtype, ctx.scale, ctx.padding = table.shape, table.dtype, scale, padding
        return _lookup(table, tokens, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        tokens, = ctx.saved_tensors
        (v, d), dtype, n, dev = ctx.sizes, ctx.dtype, tokens.numel(), g.device
        g = g.contiguous()
        L = _lib.load()
        dtable = torch.empty((v, d), dtype=dtype, device=dev)
        nbytes = L.dg_embedding_grad_scratch_bytes(v, d, n, _DTYPES[dtype])
        scratch = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        with _lib.device_ctx(dev):
            _lib.check(L.dg_embedding_grad(g.data_ptr(), _DTYPES[dtype], tokens.data_ptr(), _WIDE[tokens.dtype], n, v, d,
                                           ctx.scale, ctx.padding, dtable.data_ptr(), scratch.data_ptr(), nbytes,
                                           _lib.stream_of(dev)))
        return dtable, None, None, None


def embedding_lookup(table: torch.Tensor, tokens: torch.Tensor, scale: float = 1.0,
                     padding_idx: int | None = None) -> torch.Tensor:
    """scale * table[tokens] of shape [*tokens.shape, D] in table's type, differentiable (once) w.r.t. table.

    table: [V, D] float32, float16 or bfloat16 on a HIP device, any strides; tokens: int32 or int64 of any shape on the
    same device, or on the host.  Products and sums are 32-bit and round once.  padding_idx (negative: from the end) is
    a row that gets no gradient; its lookup is like any other's.

    Tokens outside [0, V) are an IndexError where tokens is on the host.  On the device reading them back would stall
    the stream: there such a token reads nothing, its row of the result is NaN, and it adds nothing to the gradient.

    The gradient is dense, in table's type, with every row written."""
    _lib.require_device(table, "table")
    if table.dim() != 2 or table.dtype not in _DTYPES:
        raise RuntimeError(f"embedding_lookup: table must be [V, D] float32, float16 or bfloat16, got "
                           f"{tuple(table.shape)} {table.dtype}")
    if tokens.dtype not in _WIDE:
        raise RuntimeError(f"embedding_lookup: tokens must be int32 or int64, got {tokens.dtype}")
    v = table.shape[0]
    if tokens.device != table.device:
        if tokens.device.type != "cpu":
            raise RuntimeError(f"embedding_lookup: tokens is on {tokens.device}, table on {table.device}")
        if tokens.numel() and not (int(tokens.min()) >= 0 and int(tokens.max()) < v):
            raise IndexError(f"embedding_lookup: a token is outside [0, {v})")
        tokens = tokens.to(table.device)
    if not tokens.is_contiguous():
        tokens = tokens.contiguous()
    padding = -1
    if padding_idx is not None:
        if not -v <= padding_idx < v:
            raise IndexError(f"embedding_lookup: padding_idx {padding_idx} is outside the table's {v} rows")
        padding = padding_idx % v
    if table.requires_grad and torch.is_grad_enabled():
        return _EmbeddingLookup.apply(table, tokens, float(scale), padding)
    return _lookup(table, tokens, float(scale))
