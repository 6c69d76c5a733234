"""The lookup of token embeddings and its gradient by sorted tokens, on the kernels of csrc/embedding.cu: EmbeddingScaled of the reference
(pratchya/_nnx_impl/_module.py:21-37) without its quantization, which the model adds."""
from __future__ import annotations

import operator
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from ._logprobs import wants_derivative
from ._nograph import run


def embedding_lookup(table: torch.Tensor, ids: torch.Tensor, scale: float = 1.0, padding_id: Optional[int] = None) -> torch.Tensor:
    """scale * table[ids], of shape [..., C] and the type of table [V, C] (f32 or bf16; the product is rounded once), for whole numbers `ids` [...].

    An id below zero counts from the table's end, as an index does.  `padding_id` (counted so, too) gives rows of zeros, an id beyond the table on either side rows of NaN; neither has
    a gradient.  Differentiable once in the table: its gradient, of its type, is scale times sums in f32 over a token's positions in an order that goes by the ids alone, so
    that it has the same bits every time; all of it is written, rows of no token with zeros."""
    scale = float(scale)
    if padding_id is not None:
        padding_id = operator.index(padding_id)
    derivative = wants_derivative(table)
    vocab = table.shape[0] if isinstance(table, torch.Tensor) and table.dim() == 2 else 0
    if padding_id is None or -vocab <= padding_id < vocab:
        padding = -1 if padding_id is None else padding_id % vocab
        out = _lib.native().embedding_lookup(table, ids, scale, padding, derivative)
        if out is not None:
            return out
    table, ids, padding = _checked(table, ids, padding_id)          # what has to be converted first, or refused
    return run(_EmbeddingFn, table, ids, scale, padding) if derivative else _forward(table, ids, scale, padding)


def _checked(table, ids, padding_id):
    if not isinstance(table, torch.Tensor) or not isinstance(ids, torch.Tensor) or not table.is_cuda:
        raise RuntimeError("embedding_lookup needs CUDA tensors: pratchya_b200 has no CPU path")
    if ids.device != table.device:
        raise RuntimeError("embedding_lookup: ids must be on the table's device")
    if table.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"embedding_lookup: the table is {table.dtype}; float32 and bfloat16 are taken")
    if table.dim() != 2 or table.numel() == 0:
        raise ValueError(f"embedding_lookup: table {tuple(table.shape)}")
    if ids.dtype is not torch.int64:
        if ids.dtype not in (torch.int32, torch.int16, torch.int8, torch.uint8):
            raise TypeError(f"embedding_lookup: ids are {ids.dtype}, not whole numbers")
        ids = ids.to(torch.int64)
    vocab = table.shape[0]
    if padding_id is not None and not -vocab <= padding_id < vocab:
        raise ValueError(f"embedding_lookup: padding_id {padding_id} of a table of {vocab}")
    if torch.jit.is_tracing():          # a trace would hold the result as a constant
        raise RuntimeError("embedding_lookup cannot be traced")
    return table.contiguous(), ids.contiguous(), -1 if padding_id is None else padding_id % vocab


def _forward(table, ids, scale, padding):
    out = torch.empty((*ids.shape, table.shape[1]), dtype=table.dtype, device=table.device)
    _lib.native().pb_embedding_lookup(table, _type(table), *table.shape, ids, ids.numel(), scale, padding, out)
    return out


def _type(x):
    return _lib.PB_F32 if x.dtype is torch.float32 else _lib.PB_BF16


class _EmbeddingFn(torch.autograd.Function):
    """What the extension's own function does, for calls that a dispatch mode watches."""
    @staticmethod
    def forward(ctx, table, ids, scale, padding):
        ctx.save_for_backward(ids)
        ctx.scale, ctx.padding, ctx.shape = scale, padding, table.shape
        return _forward(table, ids, scale, padding)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        (ids,) = ctx.saved_tensors
        nat, g = _lib.native(), g.contiguous()
        d = torch.empty(ctx.shape, dtype=g.dtype, device=g.device)
        size = nat.pb_embedding_lookup_bwd_workspace_size(ids.numel(), *ctx.shape)
        workspace = torch.empty(max(size, 256), dtype=torch.uint8, device=g.device)
        nat.pb_embedding_lookup_bwd(g, _type(g), ids, ids.numel(), *ctx.shape, ctx.scale, ctx.padding, d, workspace, size)
        return d, None, None, None
