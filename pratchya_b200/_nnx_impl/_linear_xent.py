"""The training loss behind a vocabulary's weight without the logits, on the kernels of csrc/linear_xent.cu: what lm_head and compute_loss of the reference
(pratchya/_nnx_impl/_model.py:77, _utils.py:7-13) compute, for a weight in bf16 and one loss for each position."""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from ._logprobs import wants_derivative


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, smoothing: float = 0.0) -> torch.Tensor:
    """Losses (f32, of `targets`' shape [...]) of hidden states x [..., C] against `weight` [C, V], both bf16: with z = x W

        lse(z) - (1 - smoothing) z[target] - smoothing mean(z),

    cross entropy against one-hot targets smoothed as in `smoothed_cross_entropy`.  Products have f32 sums; no logits are written: forward keeps a
    maximum and two sums of each 128 of a position, backward makes them again, a piece of the vocabulary at a time (256 MB).

    A negative target is none: loss 0, no gradient, and nothing of the position's x (a NaN neither) reaches anything; such positions cost next to nothing.  One beyond the
    vocabulary has loss NaN and no gradient.  x may be a strided view such as x[:, :-1], and weight the transpose of a [V, C] table: both are read in
    place (a weight whose rows do not lie 16 bytes apart is copied).  Differentiable once in x and weight; gradients are bf16 and weight's lies as weight does."""
    smoothing = float(smoothing)
    x, weight, targets = _checked(x, weight, targets, smoothing)
    if wants_derivative(x) or wants_derivative(weight):
        return _LinearXentFn.apply(x, weight, targets, smoothing)
    return _forward(x, weight, targets, smoothing)[0]


def _checked(x, weight, targets, smoothing):
    if not (isinstance(x, torch.Tensor) and isinstance(weight, torch.Tensor) and isinstance(targets, torch.Tensor) and x.is_cuda):
        raise RuntimeError("linear_cross_entropy needs CUDA tensors: pratchya_b200 has no CPU path")
    if weight.device != x.device or targets.device != x.device:
        raise RuntimeError("linear_cross_entropy: x, weight and targets must be on one device")
    if x.dtype is not torch.bfloat16 or weight.dtype is not torch.bfloat16:
        raise TypeError(f"linear_cross_entropy: x is {x.dtype} and weight {weight.dtype}; bfloat16 is taken (the products run on its tensor cores)")
    if weight.dim() != 2 or x.dim() < 1 or weight.shape[0] != x.shape[-1] or weight.numel() == 0 or targets.shape != x.shape[:-1]:
        raise ValueError(f"linear_cross_entropy: x {tuple(x.shape)}, weight {tuple(weight.shape)}, targets {tuple(targets.shape)}")
    if not 0.0 <= smoothing <= 1.0:
        raise ValueError(f"linear_cross_entropy: smoothing {smoothing}")
    if targets.dtype is not torch.int64:
        if targets.dtype not in (torch.int32, torch.int16, torch.int8, torch.uint8):
            raise TypeError(f"linear_cross_entropy: targets are {targets.dtype}, not whole numbers")
        targets = targets.to(torch.int64)
    if torch.jit.is_tracing():          # a trace would hold the results as constants
        raise RuntimeError("linear_cross_entropy cannot be traced")
    return x if _lib.native().rows_at_two_strides(x) else x.contiguous(), weight, targets.contiguous()


def _lies(weight):
    """(weight, elements from row to row, whether a row is a word's): the weight as the library reads it, [C, V] or [V, C] rows."""
    (depth, vocab), (by_depth, by_vocab) = weight.shape, weight.stride()
    if (by_vocab == 1 or vocab == 1) and (by_depth >= vocab or depth == 1):
        return weight, by_depth if depth > 1 else vocab, 0
    if (by_depth == 1 or depth == 1) and (by_vocab >= depth or vocab == 1):
        return weight, by_vocab if vocab > 1 else depth, 1
    return weight.contiguous(), vocab, 0


def _workspace(x, weight, targets, ld, by_word, backward):
    nat = _lib.native()
    size = nat.pb_linear_xent_workspace_size(targets.numel(), x.shape[-1], weight, ld, by_word, weight.shape[1], backward)
    return torch.empty(max(size, 256), dtype=torch.uint8, device=x.device), size


def _forward(x, weight, targets, smoothing):
    weight, ld, by_word = _lies(weight)
    nat = _lib.native()
    loss, lse = (torch.empty(targets.shape, dtype=torch.float32, device=x.device) for _ in range(2))
    with _lib.on_device(x.device):
        workspace, size = _workspace(x, weight, targets, ld, by_word, 0)
        outer, inner, stride_outer, stride_inner = nat.strides_of_rows(x)
        nat.pb_linear_xent(x, outer, inner if x.numel() else 0, stride_outer, stride_inner, x.shape[-1], weight, ld, by_word, weight.shape[1], targets, smoothing, loss, lse, workspace, size)
    return loss, lse


class _LinearXentFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, targets, smoothing):
        loss, lse = _forward(x, weight, targets, smoothing)
        ctx.save_for_backward(x, weight, targets, lse)
        ctx.smoothing = smoothing
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        x, weight, targets, lse = ctx.saved_tensors
        weight, ld, by_word = _lies(weight)
        nat, (depth, vocab) = _lib.native(), weight.shape
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if ctx.needs_input_grad[0] else None
        dw = torch.empty((vocab, depth) if by_word else (depth, vocab), dtype=weight.dtype, device=x.device) if ctx.needs_input_grad[1] else None
        g = g.to(torch.float32).contiguous()
        with _lib.on_device(x.device):
            workspace, size = _workspace(x, weight, targets, ld, by_word, 1)
            outer, inner, stride_outer, stride_inner = nat.strides_of_rows(x)
            nat.pb_linear_xent_bwd(x, outer, inner if x.numel() else 0, stride_outer, stride_inner, depth, weight, ld, by_word, vocab, targets, ctx.smoothing, lse, g, dx, dw, workspace, size)
        return dx, dw.t() if by_word and dw is not None else dw, None, None
