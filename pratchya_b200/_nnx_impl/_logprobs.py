"""From logits to scores and answers: log probabilities of given tokens, the entropy, and the best alternatives of every position, on
the kernels of csrc/logprobs.cu.  Stands next to the training loss (pratchya/_nnx_impl/_utils.py:7-13), which gives one
smoothed number for a whole batch."""
from __future__ import annotations

import operator
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

from .. import _lib
from ._nograph import no_graph

MAX_TOKENS, MAX_TOP = 128, 128


class TokenLogprobs(NamedTuple):
    """All f32 but for top_tokens (int64).  With logits [..., V]: `logprobs` of the shape of the given tokens (None without any),
    `entropy` [...], `top_logprobs` and `top_tokens` [..., top]."""
    logprobs: Optional[torch.Tensor]
    entropy: torch.Tensor
    top_logprobs: torch.Tensor
    top_tokens: torch.Tensor


def token_logprobs(logits, tokens=None, top: int = 0) -> TokenLogprobs:
    """Scores of f32 or bf16 `logits` [..., V], in one pass over them:

    * `logprobs`: log softmax(logits) at `tokens`, one per position ([...]) or several ([..., n], n <= 128; a teacher's alternatives, say).  A
      negative token is none: 0, and no gradient.  A token beyond the vocabulary: NaN.
    * `entropy` of the softmax (natural logarithm).
    * `top_logprobs`, `top_tokens`: the `top` largest logits (top <= 128, top <= V), equal ones in the order of their indices.

    -inf masks a token out.  A position where nothing is left has log probabilities of -inf, an entropy of 0 and no gradient; one with a
    NaN or +inf has NaN throughout (its top_tokens are valid indices).  Logits may be a strided view such as logits[:, :-1]: it is read in place.
    Differentiable in the logits through all three; the gradient has the logits' type."""
    derivative = wants_derivative(logits)
    out = _lib.native().token_logprobs(logits, tokens, top, derivative)
    if out is None:          # what has to be converted first, or refused
        if torch.jit.is_tracing():          # a trace would hold the results as constants
            raise RuntimeError("token_logprobs cannot be traced")
        logits, tokens, top = _checked(logits, tokens, top)
        out = _lib.native().token_logprobs(logits, tokens, top, derivative)
        if out is None:
            raise RuntimeError("token_logprobs takes plain CUDA tensors only")
    return TokenLogprobs(*out)


def wants_derivative(x) -> bool:
    """Whether anything can ask for a derivative of an op on x: a graph that x is in, or forward-mode differentiation or a function transform under way (which the
    op's autograd.Function then refuses).  Torch has no public name for the level of the former; where its own is gone, the answer is yes."""
    if torch.is_grad_enabled():
        return (isinstance(x, torch.Tensor) and x.requires_grad) or getattr(forward_ad, "_current_level", 0) >= 0
    return not no_graph()


def _checked(logits, tokens, top):
    if not isinstance(logits, torch.Tensor) or not logits.is_cuda:
        raise RuntimeError("token_logprobs needs CUDA tensors: pratchya_b200 has no CPU path")
    if logits.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"token_logprobs: logits are {logits.dtype}; float32 and bfloat16 are taken")
    if logits.dim() == 0 or logits.shape[-1] == 0:
        raise ValueError(f"token_logprobs: logits {tuple(logits.shape)}")
    lead, top = logits.shape[:-1], operator.index(top)
    if not 0 <= top <= min(MAX_TOP, logits.shape[-1]):
        raise ValueError(f"token_logprobs: {top} alternatives of {logits.shape[-1]} (at most {MAX_TOP})")
    if tokens is not None:
        if not isinstance(tokens, torch.Tensor) or tokens.device != logits.device:
            raise RuntimeError("token_logprobs: tokens must be on the logits' device")
        if tokens.dtype is not torch.int64:
            if tokens.dtype not in (torch.int32, torch.int16, torch.int8, torch.uint8):
                raise TypeError(f"token_logprobs: tokens are {tokens.dtype}, not whole numbers")
            tokens = tokens.to(torch.int64)
        if tokens.shape != lead and (tokens.shape[:-1] != lead or tokens.dim() != logits.dim()):
            raise ValueError(f"token_logprobs: tokens {tuple(tokens.shape)} for logits {tuple(logits.shape)}")
        if tokens.shape != lead and tokens.shape[-1] > MAX_TOKENS:
            raise ValueError(f"token_logprobs: {tokens.shape[-1]} tokens of a position (at most {MAX_TOKENS})")
        tokens = tokens.contiguous()
    return logits if _lib.native().rows_at_two_strides(logits) else logits.contiguous(), tokens, top
