"""Linear layers whose weight is held in 4 bits, for a model that answers: the kernel of pratchya/_nnx_impl/_module.py:39-50 quantized once on
groups along fan_in, and products of the activations as they are with it (no fp8 rounding of the input or the output)."""
from __future__ import annotations

import torch

from .._qualia._int4 import dequantize_int4_impl, int4_matmul_impl, quantize_int4_impl


class Int4Linear(torch.nn.Module):
    """y = x W for few rows of x, f32 or bf16, W [fan_in, fan_out] in groups of 32, 64 or 128 values, with zero points or without.  It has no gradient:
    neither in x nor in the weight.  The weight is read once for every eight rows of an f32 x, and every 32 of a bf16 one."""

    def __init__(self, kernel: torch.Tensor, group: int = 128, zero_points: bool = False):
        super().__init__()
        q, scale, zero = quantize_int4_impl(kernel, group, zero_points)
        self.fan_in, self.fan_out = kernel.shape
        self.register_buffer("q", q)
        self.register_buffer("scale", scale)
        self.register_buffer("zero", zero)

    def _apply(self, fn, recurse=True):
        """Moves the weight's parts with the module, but a cast of the module is none of theirs."""
        parts = {name: self._buffers[name] for name in ("q", "scale", "zero")}
        super()._apply(fn, recurse)
        for name, t in parts.items():
            if t is not None and self._buffers[name].dtype is not t.dtype:
                self._buffers[name] = t.to(self._buffers[name].device)
        return self

    def forward(self, x, raw=False):
        """`raw` is for callers of a Linear that re-quantizes its product: this one never does."""
        return int4_matmul_impl(x, self.q, self.scale, self.zero, self.fan_out)

    def weight(self, dtype=torch.float32):
        """The values [fan_in, fan_out] that the layer multiplies by."""
        return dequantize_int4_impl(self.q, self.scale, self.zero, (self.fan_in, self.fan_out), dtype)
