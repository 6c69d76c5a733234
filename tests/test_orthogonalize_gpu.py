"""The orthogonalised update against its polynomial in 64 bits: matrices of any extent, of any rank, stacks, scales from subnormal to beyond f32's squares.

Errors are 2-norms against the exact result's.  A step rounds four numbers to fp16 (half a step is h = 2^-11; over many elements the root mean square is
0.42 h): X's first term, which A takes twice and the last product once, A, and B.  By the derivatives of a s + b s^3 + c s^5 at s = 1 they weigh 2b + 4c + b + c, b + 2c and
b + c, in all sqrt(2.74^2 + 1.4^2 + 0.7^2 + 2.74^2) = 4.2 of them, 8.6e-4 a step, and |p'| <= 1.6 where the values have settled hands on that much of the steps
before: sqrt(1 + 1.6^2 + 1.6^4) = 3.2 times, 2.7e-3, with the output's own rounding 0.42 * 2^-8 = 1.7e-3 in all 3.2e-3.  Few numbers may all be rounded the worst way: 7.6 h a step, 5.2
times that over the steps, and 2^-8."""
import math

import pytest
import torch

from pratchya_b200 import _lib
from pratchya_b200._nnx_impl import orthogonalize

pytestmark = pytest.mark.gpu

MANY, FEW = 5e-3, 7.6 * 2.0 ** -11 * 5.2 + 2.0 ** -8
COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _exact(g, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    x = g.double()
    x = x / (x.norm(dim=(-2, -1), keepdim=True) + eps)
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    for k in range(steps):
        a, b, c = coefficients if not hasattr(coefficients[0], "__len__") else coefficients[k]
        p = x @ x.mT
        x = a * x + (b * p + c * p @ p) @ x
    return x.mT if tall else x


def _off(got, want):
    assert got.dtype == torch.bfloat16 and got.shape == want.shape
    return ((got.double() - want).norm(dim=(-2, -1)) / want.norm(dim=(-2, -1))).max().item()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1, 1), (1, 2), (3, 2), (7, 5), (1, 5000), (777, 1), (16, 16), (31, 33), (64, 200), (127, 129), (128, 128), (129, 127), (255, 257), (100, 4099), (4099, 100), (128, 2048),
                                   (2048, 128), (513, 511), (1000, 777), (1025, 2050), (2048, 2048), (5, 64, 32), (3, 2, 40, 72), (2, 300, 900), (17, 130, 40)])
def test_any_extent(built_lib, shape, dtype):
    g = (torch.randn(shape, generator=_gen(sum(shape)), device="cuda") * 1e-3).to(dtype)
    got = orthogonalize(g)
    assert _lib.load().pb_gemm_check(torch.cuda.current_stream().cuda_stream) == 0
    assert _off(got, _exact(g)) <= (MANY if min(shape[-2:]) >= 16 else FEW)
    assert torch.equal(got, orthogonalize(g))                     # the same bits again


@pytest.mark.parametrize("shape", [(300, 300), (128, 1000), (1000, 128), (700, 1500)])
@pytest.mark.parametrize("rank", [1, 3, 40])
def test_updates_of_low_rank(built_lib, shape, rank):
    """Where the update has no direction, nothing grows over the steps: 3.44^5 = 485 times what rounding leaves there."""
    m, n = shape
    g = torch.randn(m, rank, generator=_gen(m), device="cuda") @ torch.randn(rank, n, generator=_gen(n), device="cuda")
    assert _off(orthogonalize(g), _exact(g)) <= (MANY if rank >= 16 else FEW)
    one = torch.zeros(shape, device="cuda")
    one[m // 2, n // 3] = -1e-5                                  # a single number
    assert _off(orthogonalize(one), _exact(one)) <= FEW and (orthogonalize(one) != 0).sum() == 1


def test_singular_values_that_fall_steeply(built_lib):
    u, _ = torch.linalg.qr(torch.randn(256, 256, generator=_gen(1), device="cuda", dtype=torch.float64))
    v, _ = torch.linalg.qr(torch.randn(512, 256, generator=_gen(2), device="cuda", dtype=torch.float64))
    for ratio in (1e-1, 1e-3, 1e-6):
        s = torch.logspace(0, math.log10(ratio), 256, device="cuda", dtype=torch.float64)
        g = (u * s @ v.T).float()
        assert _off(orthogonalize(g), _exact(g)) <= MANY, ratio


@pytest.mark.parametrize("scale", [1e-42, 1e-30, 1e-12, 1.0, 1e15, 1e30, 1e37])
def test_any_scale(built_lib, scale):
    """Squares of these leave f32 on either side; the norm is taken in 64 bits."""
    g = (torch.randn(96, 160, generator=_gen(3), device="cuda", dtype=torch.float64) * scale).float()
    assert _off(orthogonalize(g, eps=0.0), _exact(g, eps=0.0)) <= MANY
    assert _off(orthogonalize(g, eps=scale * 100), _exact(g, eps=scale * 100)) <= MANY          # an eps beside the norm


def test_nothing_and_no_numbers(built_lib):
    zero = torch.zeros(3, 40, 50, device="cuda")
    assert not orthogonalize(zero).any()
    g = torch.randn(4, 40, 50, generator=_gen(4), device="cuda")
    clean = orthogonalize(g)
    g[0, 3, 4], g[2, 0, 0] = math.nan, -math.inf
    got = orthogonalize(g)
    assert got[0].isnan().all() and got[2].isnan().all() and torch.equal(got[1], clean[1]) and torch.equal(got[3], clean[3])
    assert orthogonalize(zero, eps=0.0).isnan().all()             # 0 / 0, as the formula has it
    for shape in ((0, 4, 4), (3, 0, 5), (3, 5, 0)):
        assert orthogonalize(torch.empty(shape, device="cuda")).shape == shape


def test_views_steps_and_coefficients(built_lib):
    base = torch.randn(3, 100, 140, generator=_gen(5), device="cuda")
    for g in (base.mT, base[:, 1:, 3:], base[::2], base[0, :, ::2], base.to(torch.bfloat16)[:, 1:, 1:], base.flatten()[1:100 * 139 + 1].view(100, 139)):
        assert _off(orthogonalize(g), _exact(g)) <= MANY
        assert torch.equal(orthogonalize(g), orthogonalize(g.contiguous().clone()))
    for steps in (1, 2, 3, 9):
        assert _off(orthogonalize(base, steps=steps), _exact(base, steps)) <= 2 * MANY        # nine steps hand on more of the ones before: 1.6^2 each two
    mild = [(1.5, -0.5, 0.0), (1.875, -1.25, 0.375), (1.5, -0.5, 0.0)]
    assert _off(orthogonalize(base, 3, mild), _exact(base, 3, mild)) <= MANY
    assert torch.equal(orthogonalize(base, 2, (mild[1], mild[1])), orthogonalize(base, 2, mild[1]))


def test_refusals(built_lib):
    g = torch.randn(8, 8, device="cuda")
    for bad, error in (((g.cpu(),), RuntimeError), ((g.half(),), TypeError), ((g[0],), ValueError), ((g, 0), ValueError), ((g, 65), ValueError), ((g, 2.5), TypeError), ((g, 5, (1.0, 2.0)), ValueError),
                       ((g, 5, [(1.0, 0.0, 0.0)] * 4), ValueError), ((g, 5, (1.0, 0.0, 0.0), -1.0), ValueError), ((g, 5, (1.0, 0.0, 0.0), math.nan), ValueError)):
        with pytest.raises(error):
            orthogonalize(*bad)
    for far in ((9.0, 0.0, 0.0), (3.0, 40.0, -40.0), (math.nan, 0.0, 0.0), (2.5, 0.0, 0.0)):          # the last leaves by its second step
        with pytest.raises(_lib.PbError):
            orthogonalize(g, 5, far)
    with pytest.raises(RuntimeError):
        orthogonalize(g.requires_grad_(True))
    with torch.no_grad():
        assert orthogonalize(g).shape == g.shape


def test_captured_and_on_another_stream(built_lib):
    g = torch.randn(200, 300, generator=_gen(6), device="cuda")
    want = orthogonalize(g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = orthogonalize(g)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = orthogonalize(g)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(there, want)
    g.mul_(-2.0)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, -want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(256, 128), (257, 128), (512, 127), (513, 1), (1024, 65), (1025, 64), (2049, 128), (4096, 128), (128, 4096), (3000, 120), (99, 3001), (4097, 128), (20, 2048, 128), (3, 128, 300),
                                   (129, 6000), (6000, 129), (300, 8000), (500, 2100), (2, 260, 5000), (700, 700), (3, 900, 520), (1280, 1024)])
def test_every_form(built_lib, shape, dtype):
    """One launch for all steps by one to sixteen CTAs a matrix, A in whole tiles of three sizes, and cut along its contraction."""
    g = (torch.randn(shape, generator=_gen(sum(shape)), device="cuda") * 30).to(dtype)
    got = orthogonalize(g)
    assert _lib.load().pb_gemm_check(torch.cuda.current_stream().cuda_stream) == 0
    assert _off(got, _exact(g)) <= (MANY if min(shape[-2:]) >= 16 else FEW)
    assert torch.equal(got, orthogonalize(g))
    if len(shape) == 3:
        assert torch.equal(got[-1], orthogonalize(g[-1])) or _off(got[-1], _exact(g[-1])) <= MANY          # alone, it may be cut otherwise
