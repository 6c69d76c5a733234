"""Weights in 4 bits: the quantizer's bits and their order in memory against the rule as plain operations, its inverse, and products of few rows against 64 bits, at
sizes around tiles, blocks, warps and CTAs, with one group size each and zero points or none."""
import math

import pytest
import torch
from torch.autograd import forward_ad

from pratchya_b200._qualia import dequantize_int4_impl, int4_matmul_impl, quantize_int4_impl

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
PLACES = (0, 4, 1, 5, 2, 6, 3, 7)          # the nibble of k = 8 w + i in its word


def _rule(w, group, zero_points):
    """(codes [K, N], scale [K/g, N], zero [K/g, N]) by the formulas, in 32-bit operations that round as the kernel's do (a quotient by a tensor:
    torch takes one by a number as a product with its reciprocal)."""
    k, n = w.shape
    steps = torch.full((1,), 15.0 if zero_points else 7.0, device=w.device)
    w = torch.nn.functional.pad(w.float(), (0, 0, 0, -k % 128)).view(-1, group, n)
    if zero_points:
        low, high = w.amin(1).clamp(max=0), w.amax(1).clamp(min=0)
        s = ((high - low) / steps).bfloat16().float()
        z = torch.where(s > 0, torch.round(-low / s).clamp(0, 15), 0.0)
        u = torch.where((s > 0).unsqueeze(1), (torch.round(w / s.unsqueeze(1)) + z.unsqueeze(1)).clamp(0, 15), 0.0)
    else:
        s = (w.abs().amax(1) / steps).bfloat16().float()
        z = torch.full_like(s, 8.0)
        u = torch.where((s > 0).unsqueeze(1), torch.round(w / s.unsqueeze(1)).clamp(-8, 7), 0.0) + 8
    return u.reshape(-1, n)[:k], s, z


def _codes(q, depth, cols):
    """[K, N] codes read out of q by the order that the header gives."""
    k, n = torch.arange(depth, device=q.device)[:, None], torch.arange(cols, device=q.device)[None, :]
    place = torch.tensor(PLACES, device=q.device)[k % 8]
    byte = n % 16 // 8 * 512 + (n % 8 * 4 + k % 32 // 8) * 16 + k % 128 // 32 * 4 + place // 2
    return q[n // 16, k // 128, byte].long() >> 4 * (place % 2) & 15


def _parts(t, depth, cols, group):
    """[K/g, N] of a scale's or zero point's array."""
    g, n = torch.arange(-(-depth // group), device=t.device)[:, None], torch.arange(cols, device=t.device)[None, :]
    per = 128 // group
    return t[n // 16, g // per, n % 16, g % per]


def _weight(depth, cols, dtype, seed, scale=0.05):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = torch.randn(depth, cols, generator=g, device="cuda") * scale
    w[:, cols // 2] = 0.0                              # a column of zeros
    w[: depth // 2, 0] = w[: depth // 2, 0].abs() + 0.1        # groups of one sign
    w[-1, -1] = 3.0
    return w.to(DTYPES[dtype])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("zero_points", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("depth,cols", [(1, 1), (128, 16), (127, 15), (129, 17), (33, 100), (1000, 777), (2048, 128)])
def test_quantizer_bits(built_lib, depth, cols, group, zero_points, dtype):
    w = _weight(depth, cols, dtype, depth + cols)
    q, scale, zero = quantize_int4_impl(w, group, zero_points)
    tiles = (-(-cols // 16), -(-depth // 128))
    assert q.shape == (*tiles, 1024) and scale.shape == (*tiles, 16, 128 // group) and (zero is not None) == zero_points
    u, s, z = _rule(w, group, zero_points)
    assert torch.equal(_codes(q, depth, cols), u.long())
    groups = -(-depth // group)
    assert torch.equal(_parts(scale, depth, cols, group).float(), s[:groups])
    if zero_points:
        assert torch.equal(_parts(zero, depth, cols, group).float(), z[:groups])
    # what pads the tiles stands for zero
    full = dequantize_int4_impl(q, scale, zero, (tiles[1] * 128, tiles[0] * 16))
    assert (full[depth:] == 0).all() and (full[:, cols:] == 0).all()
    want = (u - z.repeat_interleave(group, 0)[:depth]) * s.repeat_interleave(group, 0)[:depth]
    assert torch.equal(full[:depth, :cols], want)
    assert torch.equal(dequantize_int4_impl(q, scale, zero, (depth, cols), torch.bfloat16), want.bfloat16())
    # the nearest of sixteen values: half a step away at most, and where the scale's rounding takes the ends out of reach, 2^-8 of 7 or 15 steps more
    assert ((want - w.float()).abs() <= (0.5 + (15 if zero_points else 7) * 2.0 ** -8 + (0.5 if zero_points else 0.0)) * s.repeat_interleave(group, 0)[:depth] * (1 + 2.0 ** -20)).all()


def test_quantizer_of_groups_that_are_no_numbers(built_lib):
    w = _weight(256, 40, "f32", 3)
    clean = dequantize_int4_impl(*quantize_int4_impl(w, 64, True), (256, 40))
    w[70, 5] = math.nan
    w[10, 6] = math.inf
    for zero_points in (False, True):
        back = dequantize_int4_impl(*quantize_int4_impl(w, 64, zero_points), (256, 40))
        assert not torch.isfinite(back[64:128, 5]).any() and not torch.isfinite(back[:64, 6]).any()
        bad = torch.zeros(256, 40, dtype=torch.bool, device="cuda")
        bad[64:128, 5] = True
        bad[:64, 6] = True
        assert torch.isfinite(back[~bad]).all()
        if zero_points:
            assert torch.equal(back[~bad], clean[~bad])


@pytest.mark.parametrize("zero_points", [False, True])
def test_every_scale(built_lib, zero_points):
    """scale * (code - zero) to the bit for all 65536 bit patterns of a scale, the smallest and those that are no numbers among them."""
    g = torch.Generator(device="cuda").manual_seed(11)
    depth, cols = 128, 65536
    q = torch.randint(0, 256, (cols // 16, 1, 1024), generator=g, device="cuda", dtype=torch.uint8)
    scale = torch.arange(cols, device="cuda").to(torch.int16).view(torch.bfloat16).view(cols // 16, 1, 16, 1)
    zero = torch.randint(0, 16, (cols // 16, 1, 16, 1), generator=g, device="cuda", dtype=torch.uint8) if zero_points else None
    less = zero.view(1, cols).float() if zero_points else 8.0
    want = (_codes(q, depth, cols).float() - less) * scale.view(1, cols).float()
    got = dequantize_int4_impl(q, scale, zero, (depth, cols))
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0.0, math.inf, -math.inf), want.nan_to_num(0.0, math.inf, -math.inf))
    low = dequantize_int4_impl(q, scale, zero, (depth, cols), torch.bfloat16)
    assert torch.equal(low.float().nan_to_num(0.0, math.inf, -math.inf), want.bfloat16().float().nan_to_num(0.0, math.inf, -math.inf))


def _check_product(x, parts, depth, cols, dtype=None, warps=8):
    y = int4_matmul_impl(x, *parts, cols, dtype)
    assert y.shape == (*x.shape[:-1], cols) and y.dtype is (dtype or x.dtype)
    w = dequantize_int4_impl(*parts, (depth, cols)).double()
    want = x.double() @ w
    size = x.double().abs() @ w.abs()
    # a group's sum: eight instructions of sixteen products, each rounded or cut to two units of 2^-23 of what it has summed; then the groups of a warp, the warps, the
    # CTAs of a cluster and the three terms of an f32, at 2^-24 each
    by = (8 * 2.0 ** -22 + (depth / 32 / warps + 8 + 8 + 3) * 2.0 ** -24) * size
    if y.dtype is torch.bfloat16:
        by = by + 2.0 ** -8 * (want.abs() + by)
    else:
        by = by + 2.0 ** -23 * want.abs()
    assert ((y.double() - want).abs() <= by + 1e-37).all(), ((y.double() - want).abs() / (by + 1e-37)).max()
    return y


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("zero_points", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows,depth,cols", [(1, 1, 1), (1, 128, 16), (2, 127, 33), (3, 1000, 100), (5, 1024, 128), (8, 2048, 272), (9, 1100, 64), (16, 640, 31), (17, 384, 48), (32, 2048, 64), (33, 300, 20), (70, 512, 40)])
def test_products(built_lib, rows, depth, cols, group, zero_points, dtype):
    g = torch.Generator(device="cuda").manual_seed(rows)
    parts = quantize_int4_impl(_weight(depth, cols, "f32", depth), group, zero_points)
    x = torch.randn(rows, depth, generator=g, device="cuda")
    x[:, :: max(1, depth // 3)] *= 100.0
    _check_product(x.to(DTYPES[dtype]), parts, depth, cols)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,depth,cols", [(32, 8192, 48), (1, 16384, 2048), (8, 8192, 4096), (3, 40000, 17), (1, 300, 70000), (20, 5000, 9000)])
def test_long_contractions_and_many_columns(built_lib, rows, depth, cols, dtype):
    """x in several CTAs' shared memory, fewer rows a pass than instructions have columns, more tiles than CTAs."""
    parts = quantize_int4_impl(_weight(depth, cols, "bf16", 1), 64, True)
    x = torch.randn(rows, depth, device="cuda").to(DTYPES[dtype])
    _check_product(x, parts, depth, cols)


def test_every_code_and_place(built_lib):
    """Rows of the identity pick single weights out: every code at every place of a tile, exactly."""
    codes = torch.arange(128 * 16, device="cuda").view(128, 16) * 7 % 16
    for zero_points in (False, True):
        w = (codes.float() - 8).clamp(-7, 7) * 0.5
        parts = quantize_int4_impl(w, 128, zero_points)
        want = dequantize_int4_impl(*parts, (128, 16))
        for dtype in (torch.float32, torch.bfloat16):
            eye = torch.eye(128, device="cuda", dtype=dtype)
            for at in range(0, 128, 8):
                assert torch.equal(int4_matmul_impl(eye[at:at + 8], *parts, 16, torch.float32), want[at:at + 8])
    # all sixteen zero points
    lows = -torch.arange(16, device="cuda").float()
    w = torch.stack([lows, lows + 15]).repeat(64, 1)
    parts = quantize_int4_impl(w, 32, True)
    assert sorted(set(parts[2].flatten().tolist())) == list(range(16))
    assert torch.equal(int4_matmul_impl(torch.eye(128, device="cuda")[:3], *parts, 16), w[:3])


def test_an_f32_x_is_taken_whole(built_lib):
    """Values whose bf16 neighbours are far: with one weight of 1, y is x to the last bit, whatever its size."""
    w = torch.zeros(128, 16, device="cuda")
    w[5, 3] = 7.0
    parts = quantize_int4_impl(w, 128)
    x = torch.zeros(6, 128, device="cuda")
    x[:, 5] = torch.tensor([1.0 + 2.0 ** -23, -math.pi, 3.0e38, 1.0e-30, 16777215.0, 1.0 / 3.0], device="cuda")
    assert torch.equal(int4_matmul_impl(x / 7.0, *parts, 16)[:, 3], (x / 7.0)[:, 5] * 7.0) or ((int4_matmul_impl(x / 7.0, *parts, 16)[:, 3] - x[:, 5]).abs() <= 2.0 ** -23 * x[:, 5].abs()).all()


def test_x_that_is_no_number(built_lib):
    parts = quantize_int4_impl(_weight(256, 64, "f32", 2, 1.0).abs() + 0.5, 128)
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.ones(4, 256, device="cuda", dtype=dtype)
        x[1, 7] = math.inf
        x[2, 200] = math.nan
        y = int4_matmul_impl(x, *parts, 64)
        assert torch.isfinite(y[0]).all() and torch.isfinite(y[3]).all() and torch.isnan(y[2]).all() and not torch.isfinite(y[1]).any()


def test_views_shapes_types_and_streams(built_lib):
    parts = quantize_int4_impl(_weight(640, 96, "f32", 2), 64, True)
    big = torch.randn(6, 4, 700, device="cuda")
    for dtype in (torch.float32, torch.bfloat16):
        x = big.to(dtype)
        whole = int4_matmul_impl(x[:, :, :640].contiguous(), *parts, 96)
        assert whole.shape == (6, 4, 96)
        assert torch.equal(int4_matmul_impl(x[:, :, :640], *parts, 96), whole)                # rows at a stride
        assert torch.equal(int4_matmul_impl(x[:, 1:3, :640], *parts, 96), whole[:, 1:3])      # ... at two
        off = int4_matmul_impl(x[:, :, 3:643], *parts, 96)                                    # ... off 16 bytes
        assert torch.equal(off, int4_matmul_impl(x[:, :, 3:643].contiguous(), *parts, 96))
        assert torch.equal(int4_matmul_impl(x[2, 1, :640], *parts, 96), int4_matmul_impl(x[2, 1:2, :640], *parts, 96)[0])
        assert int4_matmul_impl(x[:0, :, :640], *parts, 96).shape == (0, 4, 96)
        assert torch.equal(int4_matmul_impl(x[0, :1, :640].expand(5, -1), *parts, 96), int4_matmul_impl(x[0, :1, :640].expand(5, -1).contiguous(), *parts, 96))
        for out in (torch.float32, torch.bfloat16):
            _check_product(x[0, :, :640].contiguous(), parts, 640, 96, out)
    x = big[0, :, :640].contiguous()
    want = int4_matmul_impl(x, *parts, 96)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = int4_matmul_impl(x, *parts, 96)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = int4_matmul_impl(x, *parts, 96)
    x.mul_(2.0)
    graph.replay()
    assert torch.equal(held, want * 2)


def test_refusals(built_lib):
    w = _weight(256, 32, "f32", 1)
    parts = q, scale, zero = quantize_int4_impl(w, 64, True)
    x = torch.randn(2, 256, device="cuda")
    with pytest.raises(RuntimeError):
        quantize_int4_impl(w.cpu())
    for bad in (0, 16, 48, 256):
        with pytest.raises(ValueError):
            quantize_int4_impl(w, bad)
    with pytest.raises(ValueError):
        quantize_int4_impl(w[0])
    with pytest.raises(ValueError):
        quantize_int4_impl(w[:0])
    with pytest.raises(RuntimeError):
        int4_matmul_impl(x.cpu(), *parts, 32)
    with pytest.raises(RuntimeError):
        int4_matmul_impl(x, q.cpu(), scale, zero, 32)
    with pytest.raises(TypeError):
        int4_matmul_impl(x.half(), *parts, 32)
    with pytest.raises(TypeError):
        int4_matmul_impl(x, *parts, 32, torch.float16)
    with pytest.raises(ValueError):
        int4_matmul_impl(x[:, :100], *parts, 32)
    with pytest.raises(ValueError):
        int4_matmul_impl(x, *parts, 33)
    with pytest.raises(ValueError):
        int4_matmul_impl(x, q, scale[..., :1].expand(-1, -1, -1, 3).contiguous(), None, 32)
    with pytest.raises(ValueError):
        int4_matmul_impl(x, q, scale, zero[..., :1].contiguous(), 32)
    with pytest.raises(ValueError):
        int4_matmul_impl(x, q, scale.float(), zero, 32)
    with pytest.raises(RuntimeError):
        int4_matmul_impl(x.clone().requires_grad_(True), *parts, 32)
    with pytest.raises(ValueError):
        dequantize_int4_impl(*parts, (300, 32))
    with pytest.raises(TypeError):
        dequantize_int4_impl(*parts, (256, 32), torch.float16)
    # the same parts, strided: taken by way of a copy
    assert torch.equal(int4_matmul_impl(x, q, scale.repeat(1, 1, 1, 2)[..., :2], zero, 32), int4_matmul_impl(x, *parts, 32))


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_parts_that_lie_anywhere_in_a_flat_buffer(built_lib, group, dtype):
    """A model's buffers may be views of one: scales at any multiple of their two bytes, codes and zero points at any byte."""
    g = torch.Generator(device="cuda").manual_seed(group)
    w, x = torch.randn(260, 40, generator=g, device="cuda"), torch.randn(3, 260, generator=g, device="cuda").to(DTYPES[dtype])
    parts = quantize_int4_impl(w, group, True)
    want, back = int4_matmul_impl(x, *parts, 40), dequantize_int4_impl(*parts, (260, 40))
    for ahead in (1, 2, 3, 4):
        moved = []
        for t in parts:
            flat = torch.empty(t.numel() + ahead, dtype=t.dtype, device="cuda")
            moved.append(flat[ahead:].view(t.shape).copy_(t))
            assert moved[-1].is_contiguous() and moved[-1].data_ptr() % 512 == ahead * t.element_size()
        assert torch.equal(int4_matmul_impl(x, *moved, 40), want) and torch.equal(dequantize_int4_impl(*moved, (260, 40)), back)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("zero_points", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantizer_of_the_smallest_numbers(built_lib, group, zero_points, dtype):
    """Groups whose largest value is 1 to 50 of bf16's smallest step: a scale is a few such steps there, up to a third off the quotient, and the codes of the ends lie beyond 0..15 but
    for the clamp."""
    g = torch.Generator(device="cuda").manual_seed(group)
    depth, cols = 256, 50
    most = torch.arange(1, cols + 1, device="cuda").float()
    w = (torch.rand(depth, cols, generator=g, device="cuda") * (2 * most + 1)).floor() - most
    w[::32], w[1::32] = most, -most                    # both ends in every group
    w[:, 1::3] = w[:, 1::3].abs()
    w[:, 2::3] = -w[:, 2::3].abs()
    w = (w * 2.0 ** -133).to(DTYPES[dtype])
    q, scale, zero = quantize_int4_impl(w, group, zero_points)
    u, s, z = _rule(w, group, zero_points)
    assert torch.equal(_codes(q, depth, cols), u.long())
    assert torch.equal(_parts(scale, depth, cols, group).float(), s)
    if zero_points:
        assert torch.equal(_parts(zero, depth, cols, group).float(), z)
    want = (u - z.repeat_interleave(group, 0)) * s.repeat_interleave(group, 0)
    assert torch.equal(dequantize_int4_impl(q, scale, zero, (depth, cols)), want)


def test_quantizer_of_groups_whose_span_is_beyond_f32(built_lib):
    """Finite weights of both signs whose largest less smallest is no f32: the scale is a fifteenth of it all the same, and the weights read back finite."""
    g = torch.Generator(device="cuda").manual_seed(5)
    w = (torch.randint(-12, 13, (256, 40), generator=g, device="cuda").double() * 2.0 ** 124).float()
    w[::32], w[1::32] = -1.5 * 2.0 ** 127, 1.25 * 2.0 ** 127
    w[:, 7] = -w[:, 7].abs()                           # of one sign: no more than the type holds
    for dtype in (torch.float32, torch.bfloat16):
        x = w.to(dtype)
        q, scale, zero = quantize_int4_impl(x, 64, True)
        v = x.double().view(4, 64, 40)
        low, high = v.amin(1).clamp(max=0), v.amax(1).clamp(min=0)
        s = ((high - low) / 15).float().bfloat16()
        z = torch.round(-low / s.double()).clamp(0, 15)
        u = (torch.round(v / s.double().unsqueeze(1)) + z.unsqueeze(1)).clamp(0, 15).view(256, 40)
        assert torch.equal(_parts(scale, 256, 40, 64), s) and torch.isfinite(s).all()
        assert torch.equal(_parts(zero, 256, 40, 64).double(), z) and torch.equal(_codes(q, 256, 40), u.long())
        want = ((u - z.repeat_interleave(64, 0)) * s.double().repeat_interleave(64, 0)).float()
        assert torch.equal(dequantize_int4_impl(q, scale, zero, (256, 40)), want) and torch.isfinite(want).all()


def test_no_derivative_is_dropped_without_a_word(built_lib):
    parts = q, scale, zero = quantize_int4_impl(_weight(256, 32, "f32", 1), 64, True)
    x = torch.randn(2, 256, device="cuda")
    want = int4_matmul_impl(x, *parts, 32)
    learned = scale.clone().requires_grad_(True)
    for f in (lambda: int4_matmul_impl(x.clone().requires_grad_(True), *parts, 32), lambda: int4_matmul_impl(x, q, learned, zero, 32),
              lambda: dequantize_int4_impl(q, learned, zero, (256, 32))):
        with pytest.raises(RuntimeError, match="backward"):
            f()
        with torch.no_grad():
            f()
    for grads in (True, False):
        with torch.set_grad_enabled(grads), forward_ad.dual_level():
            dual, scales = forward_ad.make_dual(x, torch.ones_like(x)), forward_ad.make_dual(scale, torch.ones_like(scale))
            for f in (lambda: int4_matmul_impl(dual, *parts, 32), lambda: int4_matmul_impl(x, q, scales, zero, 32), lambda: dequantize_int4_impl(q, scales, zero, (256, 32))):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    f()
            assert torch.equal(int4_matmul_impl(x, *parts, 32), want)          # nobody's tangent
        with torch.set_grad_enabled(grads):
            for f in (lambda t: int4_matmul_impl(t, *parts, 32), lambda t: quantize_int4_impl(t, 64)[0], lambda t: dequantize_int4_impl(*parts, (256, 32)) + t.sum()):
                with pytest.raises(RuntimeError, match="traced"):
                    torch.jit.trace(f, x, check_trace=False)


# ---- what x keeps in digits --------------------------------------------------------------------------------------------

def _picked(depth, cols, zero_points):
    """A weight of zeros, but for one of exactly 1 in each column at k = 5 (and a 7, or 14, at k = 6 that sets the scale to 1)."""
    w = torch.zeros(depth, cols, device="cuda")
    w[5], w[6] = 1.0, 14.0 if zero_points else 7.0
    w[7] = -1.0 if zero_points else 0.0
    parts = quantize_int4_impl(w, 128, zero_points)
    assert torch.equal(dequantize_int4_impl(*parts, (depth, cols)), w)
    return parts


@pytest.mark.parametrize("zero_points", [False, True])
@pytest.mark.parametrize("dtype,rows,depth,cols", [("f32", 1, 128, 16), ("f32", 8, 300, 40), ("bf16", 2, 512, 65536), ("bf16", 6, 128, 16)])
def test_a_weight_of_one_gives_x_to_the_bit(built_lib, dtype, rows, depth, cols, zero_points):
    """Alone in its block of 128, whatever its size: f32 in four digits, bf16 in three (two rows and many columns) and as it is."""
    parts = _picked(depth, cols, zero_points)
    values = torch.tensor([1.0 + 2.0 ** -23, -math.pi, 3.0e38, 1.0e-30, 16777215.0, 1.0 / 3.0, -1.0e-20, 255.0], device="cuda").to(DTYPES[dtype])
    for at in range(0, 8, rows):
        x = torch.zeros(min(rows, 8 - at), depth, device="cuda", dtype=DTYPES[dtype])
        x[:, 5] = values[at:at + rows]
        assert (int4_matmul_impl(x, *parts, cols, torch.float32) == x[:, 5:6].float()).all()


@pytest.mark.parametrize("zero_points", [False, True])
@pytest.mark.parametrize("dtype,rows,depth,cols,exact,step", [("f32", 1, 128, 16, 6, 30), ("f32", 8, 300, 40, 6, 30), ("bf16", 2, 512, 65536, 14, 22), ("bf16", 8, 128, 16, 126, 126)])
def test_small_numbers_beside_a_large_one(built_lib, dtype, rows, depth, cols, exact, step, zero_points):
    """The large one meets weights of zero, so that what is lost of the small one is all that y is off: nothing from 2^-6 (2^-14) of the large one on, and no more than 2^-30 (2^-22) of it
    below.  A bf16 x that is taken as it is loses nothing."""
    parts = _picked(depth, cols, zero_points)
    g = torch.Generator(device="cuda").manual_seed(rows)
    for power in range(0, 40):
        for large in (1.0, 1.99, 3.0e5):
            x = torch.zeros(rows, depth, device="cuda", dtype=DTYPES[dtype])
            x[:, 100] = large
            x[:, 5] = ((torch.rand(rows, generator=g, device="cuda") + 1.0) * 0.5 * large * 2.0 ** -power).to(x.dtype)
            x[-1, 5] = -x[-1, 5]
            of = float(x[0, 100])
            off = (int4_matmul_impl(x, *parts, cols, torch.float32).double() - x[:, 5:6].double()).abs()
            inside = (x[:, 5].double().abs() >= of * 2.0 ** -exact).unsqueeze(-1)
            assert (off[inside.expand_as(off)] == 0).all() and (off <= of * 2.0 ** -step).all(), (power, large)


def test_a_number_of_columns_is_whole(built_lib):
    parts = quantize_int4_impl(_weight(256, 32, "f32", 1), 64, True)
    x = torch.randn(2, 256, device="cuda")
    for bad in (32.5, 32.0, "32"):
        with pytest.raises(TypeError):
            int4_matmul_impl(x, *parts, bad)
        with pytest.raises(TypeError):
            dequantize_int4_impl(*parts, (256, bad))
    assert torch.equal(int4_matmul_impl(x, *parts, torch.tensor(32)), int4_matmul_impl(x, *parts, 32))
