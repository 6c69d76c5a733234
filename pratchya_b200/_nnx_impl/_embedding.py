"""The lookup of token embeddings and its gradient by sorted tokens, on the kernels of csrc/embedding.cu: EmbeddingScaled of the reference
(pratchya/_nnx_impl/_module.py:21-37) without its quantization, which the model adds."""
from __future__ import annotations

import operator
from typing import Optional

import torch

from .. import _lib
from ._logprobs import wants_derivative


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
    out = _lib.native().embedding_lookup(table, ids, scale, padding, derivative)
    if out is None:
        raise RuntimeError("embedding_lookup takes plain CUDA tensors only")
    return out


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
