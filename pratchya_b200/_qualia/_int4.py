"""Weights in 4 bits with a scale (and where wanted a zero point) for each group of values along the contraction, for models that answer
one token at a time: such a product is bound by the weights' bytes, and these are half of fp8's.  Functional like the rest of
this package: the parts of a weight are plain tensors.

    w[k][n] = scale[n][k / group] * (u[k][n] - zero[n][k / group])          u in 0..15; zero is 8 where none is stored

With A = ceil(N / 16) and B = ceil(K / 128): q uint8 [A, B, 1024], scale bf16 [A, B, 16, 128 / group], zero uint8 the same.  1024 bytes hold
16 columns and 128 values of k in the order in which the product's matrix instructions take them (include/pratchya_b200.h gives it)."""
from __future__ import annotations

import operator

import torch
from torch.autograd import forward_ad

from .. import _lib
from ._ops import _require_cuda

GROUPS = (32, 64, 128)


def _no_derivative(what, *tensors):
    """Refuses where a derivative could be asked for that the op does not have, or a trace would hold its result as a constant (the extension leaves such calls alone)."""
    if torch.jit.is_tracing():
        raise RuntimeError(f"{what} cannot be traced")
    for t in tensors:
        if not isinstance(t, torch.Tensor):
            continue
        if t.requires_grad and torch.is_grad_enabled():
            raise RuntimeError(f"{what} has no backward pass: call it under torch.no_grad(), or with detached tensors")
        if getattr(forward_ad, "_current_level", 0) >= 0 and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{what} has no forward-mode derivative")


def _int4_parts(q, scale, zero, depth, cols, what):
    for t, name in ((q, "q"), (scale, "scale"), *(((zero, "zero"),) if zero is not None else ())):
        _require_cuda(t, f"{what}: {name}")
        if t.device != q.device:
            raise RuntimeError(f"{what}: {name} is on {t.device}, q on {q.device}")
    tiles = (-(-cols // 16), -(-depth // 128))
    if depth <= 0 or cols <= 0 or q.dtype is not torch.uint8 or tuple(q.shape) != (*tiles, 1024):
        raise ValueError(f"{what}: q {q.dtype} {tuple(q.shape)} is no weight of [{depth}, {cols}], which is uint8 {(*tiles, 1024)}")
    if scale.dtype is not torch.bfloat16 or scale.dim() != 4 or tuple(scale.shape[:3]) != (*tiles, 16) or scale.shape[3] not in (1, 2, 4):
        raise ValueError(f"{what}: scale {scale.dtype} {tuple(scale.shape)} for a weight of [{depth}, {cols}], which has bfloat16 {(*tiles, 16, '128 / group')}")
    if zero is not None and (zero.dtype is not torch.uint8 or zero.shape != scale.shape):
        raise ValueError(f"{what}: zero {zero.dtype} {tuple(zero.shape)} beside scale {tuple(scale.shape)}")
    groups = scale.shape[3]
    return _at(q, 16), _at(scale, 2 * groups), _at(zero, groups) if zero is not None else None


def _at(t, align):
    """t as it is where the kernels can read it there, contiguous from a multiple of `align` bytes; else a copy."""
    t = t.contiguous()
    return t if t.data_ptr() % align == 0 else t.clone()


def quantize_int4_impl(w: torch.Tensor, group: int = 128, zero_points: bool = False):
    """(q, scale, zero or None) of w [K, N]; K and N may be any sizes.  scale = bf16(max|w| / 7) of a group and u = rint(w / scale) + 8; with
    zero points scale = bf16((max(w, 0) - min(w, 0)) / 15), zero = rint(-min / scale) and u = rint(w / scale) + zero.  The codes are the nearest
    ones for the scale as stored.  Like the other quantizers of this package it takes w's values: no graph leads back to w."""
    _require_cuda(w, "quantize_int4_impl input")
    if w.dim() != 2 or w.numel() == 0:
        raise ValueError(f"quantize_int4_impl: a weight of {tuple(w.shape)} is no [K, N]")
    if group not in GROUPS:
        raise ValueError(f"quantize_int4_impl: groups of {group}; {GROUPS} are built")
    if w.dtype not in (torch.float32, torch.bfloat16):
        w = w.to(torch.float32)
    out = _lib.native().quantize_int4(w.detach().contiguous(), group, bool(zero_points))
    if out is None:
        _no_derivative("quantize_int4_impl")
        raise RuntimeError("quantize_int4_impl takes plain CUDA tensors only")
    return out


def dequantize_int4_impl(q, scale, zero, shape, dtype=torch.float32):
    """The values [K, N] that the parts of a weight of that shape stand for.  Not differentiable in the scale."""
    depth, cols = (operator.index(n) for n in shape)
    if dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"dequantize_int4_impl: {dtype}; float32 and bfloat16 are built")
    out = _lib.native().dequantize_int4(q, scale, zero, depth, cols, dtype)
    if out is None:
        _no_derivative("dequantize_int4_impl", scale)
        out = _lib.native().dequantize_int4(*_int4_parts(q, scale, zero, depth, cols, "dequantize_int4_impl"), depth, cols, dtype)
        if out is None:
            raise RuntimeError("dequantize_int4_impl takes plain CUDA tensors only")
    return out


def int4_matmul_impl(x, q, scale, zero, cols: int, dtype=None):
    """x [..., K] times a weight of [K, cols] in its parts, in x's type or `dtype`.  Sums are f32; x keeps its bits but for what is far below its
    neighbours (of 128 the largest has 2^30 steps above zero where x is f32, 2^22 at least where it is bf16, and the others the same steps).  A row of x with an
    infinity or a NaN has no finite products.  Made for few rows: the weight is read once for every 32 of a bf16 x and every eight of an f32 one.
    Not differentiable: an x or a scale that asks for a gradient or carries a tangent is refused, and so is tracing."""
    out = _lib.native().int4_product(x, q, scale, zero, cols, dtype)
    if out is not None:
        return out
    _no_derivative("int4_matmul_impl", x, scale)
    _require_cuda(x, "int4_matmul_impl input")
    if x.dim() == 0:
        raise ValueError("int4_matmul_impl: x has no dimension")
    if x.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"int4_matmul_impl: x is {x.dtype}; float32 and bfloat16 are taken")
    if dtype not in (None, torch.float32, torch.bfloat16):
        raise TypeError(f"int4_matmul_impl: {dtype}; float32 and bfloat16 are built")
    cols = operator.index(cols)
    parts = _int4_parts(q, scale, zero, x.shape[-1], cols, "int4_matmul_impl")
    if x.device != q.device:
        raise RuntimeError(f"int4_matmul_impl: x is on {x.device}, the weight on {q.device}")
    out = _lib.native().int4_product(x.contiguous(), *parts, cols, dtype)
    if out is None:
        raise RuntimeError("int4_matmul_impl takes plain CUDA tensors only")
    return out
