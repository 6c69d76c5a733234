"""Answers and scores of a PratchyaCausalLM: the loop around `advance` that a program would write, on token_logprobs."""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from ._logprobs import TokenLogprobs, token_logprobs


class Answer(NamedTuple):
    """`tokens` [B, n] and of each the log probability and the entropy of the position it was chosen at; `top_logprobs` and `top_tokens` [B, n, top]."""
    tokens: torch.Tensor
    logprobs: torch.Tensor
    entropy: torch.Tensor
    top_logprobs: torch.Tensor
    top_tokens: torch.Tensor


@torch.no_grad()
def generate(model, prompt, steps: int, top: int = 1, uniform: Optional[torch.Tensor] = None) -> Answer:
    """`steps` tokens after `prompt` [B, T].  The next token is the best of the `top` alternatives, or, with `uniform` [B, steps] of numbers in [0, 1), the one
    where the sum of their probabilities (as shares of the alternatives') passes that number.

    The log probabilities are those of a text read token by token behind its prompt.  `score` reads it at once and has others: the norm over a block's heads runs
    over the tokens of a call (see `advance`).  Importance ratios want both sides from the same of the two.

    A prompt with a token beyond the vocabulary is not refused: its answer's log probabilities are NaN, and its tokens say nothing."""
    if prompt.dim() != 2 or prompt.shape[1] == 0 or steps < 1 or top < 1:
        raise ValueError(f"generate: prompt {tuple(prompt.shape)}, {steps} steps, {top} alternatives")
    if uniform is not None and tuple(uniform.shape) != (prompt.shape[0], steps):
        raise ValueError(f"generate: uniform {tuple(uniform.shape)} for {prompt.shape[0]} answers of {steps}")
    state, ids, taken = None, prompt, []
    for i in range(steps):
        logits, state = model.advance(ids, state, last=True)
        scores = token_logprobs(logits[:, -1], top=top)
        pick = torch.zeros_like(scores.top_tokens[:, :1])
        if uniform is not None:
            share = torch.softmax(scores.top_logprobs, -1).cumsum(-1)
            last = (share < share[:, -1:]).sum(-1, keepdim=True)          # behind it is what has no probability; a sum of shares may round to less than the number
            pick = torch.minimum((share <= uniform[:, i:i + 1]).sum(-1, keepdim=True), last)
        ids = scores.top_tokens.gather(-1, pick)
        taken.append((ids[:, 0], scores.top_logprobs.gather(-1, pick)[:, 0], scores.entropy, scores.top_logprobs, scores.top_tokens))
    return Answer(*(torch.stack(part, dim=1) for part in zip(*taken)))


def score(model, ids, top: int = 0) -> TokenLogprobs:
    """How the model takes a text `ids` [B, T]: of each token but the first its log probability behind the ones before it, with the entropy there and the
    best alternatives [B, T-1, ..].  Differentiable in the model's parameters where gradients are on.  Not what `generate` found for the same tokens: there they are
    read one by one."""
    logits, _ = model(ids)
    return token_logprobs(logits[:, :-1], ids[:, 1:], top=top)
