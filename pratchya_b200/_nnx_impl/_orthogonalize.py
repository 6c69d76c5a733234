"""The orthogonalised update of a weight, by Newton-Schulz products on the kernels of csrc/orthogonalize.cu: what the Muon branch of the reference's
optimizer does with the momentum blend `c` (newton_schulz, pratchya/_nnx_impl/_optimizer.py:11-29; :136-142 for a stack of layers, :208)."""
from __future__ import annotations

import array
import math
import operator

import torch

from .. import _lib
from ._logprobs import wants_derivative

#: a, b, c of the odd polynomial a s + b s^3 + c s^5: steepest at zero of those that keep [0, 1] near 1 in five steps
COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def orthogonalize(update: torch.Tensor, steps: int = 5, coefficients=COEFFICIENTS, eps: float = 1e-7) -> torch.Tensor:
    """`update` [..., m, n] (f32 or bf16; a stack of layers is one call) with its singular values drawn to about 1: X = update / (|update| + eps) and `steps`
    times X = a X + (b A + c A A) X with A = X X^T, from the side with the smaller A.  Returns bf16 of update's shape.

    `coefficients`: (a, b, c), or `steps` triples of them; refused where they take a singular value beyond 4.  X is carried with 22 bits from step to step and the products'
    operands have 11, so that the result is within some 3e-3 of the exact polynomial's in the 2-norm (half of that is bf16's own rounding) for updates of
    any rank (more where the update's norm is 10^-5 of eps and less: X's numbers are held to 2^-37).  An update with an infinity or a NaN becomes NaN throughout, one of zeros
    stays zero (eps > 0; else 0 / 0).  Has no derivative."""
    if not isinstance(update, torch.Tensor) or not update.is_cuda:
        raise RuntimeError("orthogonalize needs a CUDA tensor: pratchya_b200 has no CPU path")
    if update.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"orthogonalize: update is {update.dtype}; float32 and bfloat16 are taken")
    if update.dim() < 2:
        raise ValueError(f"orthogonalize: update {tuple(update.shape)} is no matrix")
    if torch.jit.is_tracing():          # a trace would hold the result as a constant
        raise RuntimeError("orthogonalize cannot be traced")
    if wants_derivative(update):
        raise RuntimeError("orthogonalize has no derivative: call it under torch.no_grad() or with update.detach()")
    steps, eps = operator.index(steps), float(eps)
    if not 1 <= steps <= 64 or not (eps >= 0.0 and math.isfinite(eps)):
        raise ValueError(f"orthogonalize: {steps} steps (1 to 64), eps {eps}")
    triples = [t for t in coefficients]
    if not any(hasattr(t, "__len__") for t in triples):
        triples = [triples] * steps
    if len(triples) != steps or not all(hasattr(t, "__len__") and len(t) == 3 for t in triples):
        raise ValueError(f"orthogonalize: coefficients are three numbers or {steps} times three")
    flat = [float(v) for t in triples for v in t]
    out = torch.empty(update.shape, dtype=torch.bfloat16, device=update.device)
    if update.numel() == 0:
        return out
    rows, cols = update.shape[-2:]
    batch, update, nat = update.numel() // (rows * cols), update.contiguous(), _lib.native()
    dtype, element = (_lib.PB_F32, 4) if update.dtype is torch.float32 else (_lib.PB_BF16, 2)
    most = 65535          # matrices a call of the library takes
    with _lib.on_device(update.device):
        size = nat.pb_orthogonalize_workspace_size(min(batch, most), rows, cols)
        workspace = torch.empty(max(size, 256), dtype=torch.uint8, device=update.device)
        for first in range(0, batch, most):
            nat.pb_orthogonalize(update.data_ptr() + first * rows * cols * element, dtype, min(most, batch - first), rows, cols, steps, array.array("f", flat), eps,
                                 out.data_ptr() + first * rows * cols * 2, workspace, size, _lib.current_stream(update.device))
    return out
