"""Cross entropy against a vocabulary's weight without logits, and its gradients, against the definition in 64 bits: every edge of tiles, parts and pieces, both
orders of the weight, rows that TMA cannot read in place, positions without a target, values that are no numbers.

Bounds.  A logit's sum of C products in f32 by the tensor core, whose additions do not round to nearest: each term and each of the C / 16 + 1 sums within 2^-22 of the sum of magnitudes.  A
loss: that of lse's exponentials (weighted by the softmax) and of the target's logit, and 2^-20 of the numbers that meet.  A gradient: dz is rounded to bf16, the softmax
within the logit's error and 2^-20; the sums of the second product as those of the first; the result rounded to bf16.  x times g over the largest g is rounded to bf16 for dW (two numbers that are both half a step off:
2^-8 + 2^-8).  A probability, a product and a sum below f32's
normal numbers may each be 0: 2^-126, times g where it is a probability."""
import math

import pytest
import torch

from pratchya_b200 import _lib
from pratchya_b200._nnx_impl import linear_cross_entropy
from pratchya_b200._nnx_impl import _linear_xent

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _inputs(lead, depth, vocab, tied, seed=0, sharp=2.0, ignored=0.0):
    g = _gen(seed + depth + vocab)
    lead = (lead,) if isinstance(lead, int) else lead
    x = torch.randn(*lead, depth, generator=g, device="cuda").to(torch.bfloat16)
    w = (torch.randn(vocab, depth, generator=g, device="cuda") * (sharp / math.sqrt(depth))).to(torch.bfloat16)
    t = torch.randint(0, vocab, lead, generator=g, device="cuda")
    t = torch.where(torch.rand(lead, generator=g, device="cuda") < ignored, -1 - t, t)
    return x, w.t() if tied else w.t().contiguous(), t, torch.randn(lead, generator=g, device="cuda") / max(1, t.numel())


def _definition(x, w, t, a, g):
    """(loss, dx, dw) in 64 bits and the bounds of their errors."""
    c, v = w.shape
    x, w, tt, g = x.detach().reshape(-1, c).double(), w.detach().double(), t.reshape(-1), g.reshape(-1, 1).double()
    some = ((tt >= 0) & (tt < v)).unsqueeze(-1)
    x = torch.where(some, x, 0.0)
    z, size = x @ w, x.abs() @ w.abs()
    logp = torch.log_softmax(z, -1)
    hot = torch.zeros_like(z).scatter_(-1, tt.clamp(0, v - 1).unsqueeze(-1), 1.0)
    q = (1 - a) * hot + a / v
    loss = torch.where(some, -(q * logp).sum(-1, keepdim=True), 0.0)
    p = logp.exp()
    dz = torch.where(some, g * (p - q), 0.0)
    ez = size * 2.0 ** -22 * 2
    el = (p * ez).sum(-1, keepdim=True) + (q * ez).sum(-1, keepdim=True) + 2.0 ** -20 * (1.0 + torch.logsumexp(z, -1, keepdim=True).abs() + (q * z.abs()).sum(-1, keepdim=True))
    edz = torch.where(some, g.abs() * p * (ez + (p * ez).sum(-1, keepdim=True) + 2.0 ** -20 * (1 + z.abs())) + (2.0 ** -8 + 2.0 ** -20) * dz.abs() + (1 + g.abs()) * 2.0 ** -126, 0.0)
    more = lambda m, n: m * 2.0 ** -21 + n.abs() * 2.0 ** -8 + 2.0 ** -126
    dx, dw = dz @ w.t(), x.t() @ dz
    edx = edz @ w.abs().t() + more(dz.abs() @ w.abs().t(), dx)
    edw = x.abs().t() @ edz * (1 + 2.0 ** -8) + 2.0 ** -8 * (x.abs().t() @ dz.abs()) + more(x.abs().t() @ dz.abs(), dw)
    shape = t.shape
    return (loss.view(shape), dx.view(*shape, c), dw), (el.view(shape), edx.view(*shape, c), edw)


def _check(x, w, t, a, g, equal=False):
    x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = linear_cross_entropy(x, w, t, a)
    dx, dw = torch.autograd.grad(loss, (x, w), g)
    assert _lib.load().pb_gemm_check(torch.cuda.current_stream().cuda_stream) == 0
    assert loss.dtype == torch.float32 and loss.shape == t.shape and dx.dtype == dw.dtype == torch.bfloat16 and dx.shape == x.shape and dw.shape == w.shape
    want, bounds = _definition(x, w, t, a, g)
    for name, got, exact, bound in zip(("loss", "dx", "dw"), (loss.detach(), dx, dw), want, bounds):
        off = (got.double() - exact).abs()
        assert (off <= bound).all(), f"{name}: {(off / bound).max().item():.3g} of the bound"
        if name != "loss" and exact.norm() > 0 and not equal:      # (equal logits round alike, and what adds up is the bound above) bf16's roundings of dz, of x times g and of the result, 0.42 * 2^-8 each as a root mean square, and half as much for what cancels
            assert (got.double() - exact).norm() <= 1.5 * 0.73 * 2.0 ** -8 * exact.norm() or exact.numel() < 1000, name
    with torch.no_grad():
        assert torch.equal(linear_cross_entropy(x, w, t, a), loss)
    return loss.detach(), dx, dw


@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("rows,depth,vocab", [(1, 1, 1), (1, 8, 2), (2, 3, 7), (1, 64, 256), (3, 63, 255), (31, 65, 257), (128, 128, 129), (129, 72, 512), (255, 16, 1000), (256, 256, 768), (257, 136, 1001), (300, 777, 4099),
                                              (513, 200, 2048), (1000, 1000, 3001), (64, 2048, 20000)])
def test_any_extent(built_lib, rows, depth, vocab, tied):
    for a in (0.0, 0.1):
        _check(*_inputs(rows, depth, vocab, tied)[:3], a, _inputs(rows, depth, vocab, tied)[3])


@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("ignored", [0.05, 0.5, 0.97, 1.0])
def test_positions_without_a_target(built_lib, ignored, tied):
    x, w, t, g = _inputs((3, 211), 120, 1500, tied, ignored=ignored)
    loss, dx, dw = _check(x, w, t, 0.1, g)
    none = t < 0
    assert not loss[none].any() and not dx[none].any()
    x[none] = math.nan                                       # what lies in a padded position reaches nothing
    g[none] = math.inf
    again = _check(x.nan_to_num(0.0) if ignored == 1.0 else x, w, t, 0.1, torch.where(none, 0.0, g))
    got = linear_cross_entropy(x, w, t, 0.1)
    assert torch.equal(got, loss) and torch.equal(again[1], dx) and torch.equal(again[2], dw)
    if ignored == 1.0:
        assert not dw.any()


def test_pieces_of_the_vocabulary(built_lib):
    """More of dz than is held at a time: dx is added up over the pieces.  16384 rows make pieces of 8192 columns."""
    for tied in (False, True):
        x, w, t, g = _inputs(16300, 64, 20001, tied, ignored=0.1)
        _check(x, w, t, 0.0, g)


def test_views(built_lib):
    x, w, t, g = _inputs((3, 40), 96, 600, False)
    for view in (x[:, :-1], x[:, 1:], x.transpose(0, 1), x[0], x[0, 0], x[..., 1:], x[..., ::2], x[:1].expand(5, -1, -1), x.reshape(3, 8, 5, 96).permute(2, 0, 1, 3), x.flatten()[1:1 + 7 * 96].view(7, 96)):
        lead, depth = view.shape[:-1], view.shape[-1]
        tt = torch.randint(-1, 600, lead, generator=_gen(3), device="cuda")
        gg = torch.randn(lead, generator=_gen(4), device="cuda")
        one = _check(view, w[:depth], tt, 0.1, gg)
        same = _check(view.contiguous().clone(), w[:depth].clone(), tt, 0.1, gg)
        assert all(torch.equal(p, q) for p, q in zip(one, same))
    for weight in (w[:, :599], w[:, 1:], w[1:, :], w[:, ::2], w.t().contiguous().t()[:, 3:], w[:, :1].expand(-1, 50), torch.cat([w, w])[::2][:48]):
        depth = weight.shape[0]
        tt = t.clamp(max=weight.shape[1] - 1)
        xx = x[..., :depth]
        equal = weight.stride(1) == 0
        loss, dx, dw = _check(xx, weight, tt, 0.0, g, equal)
        assert all(torch.equal(p, q) for p, q in zip(_check(xx, weight.contiguous().clone(), tt, 0.0, g, equal)[:1], (loss,)))


def test_far_logits(built_lib):
    """Logits of hundreds, of 1e30, equal ones, a target without a chance, and a softmax that is all the target's."""
    x, w, t, g = _inputs(300, 64, 3000, True, sharp=200.0)
    _check(x, w, t, 0.0, g)
    _check(x * 0, w, t, 0.1, g, equal=True)                   # every logit is zero
    assert (linear_cross_entropy(x * 0, w, t) - math.log(3000)).abs().max() <= 2.0 ** -20 * 9
    z = (x.double() @ w.double())
    _check(x, w, z.argmax(-1), 0.0, g)
    _check(x, w, z.argmin(-1), 0.0, g)
    huge = torch.full_like(x, 1e15)
    loss = linear_cross_entropy(huge, torch.full_like(w, 1e15), t)      # 6.4e31 each
    assert (loss - math.log(3000)).abs().max() <= 2.0 ** -22 * 6.4e31


def test_not_a_number(built_lib):
    x, w, t, g = _inputs(300, 72, 900, False)
    clean = linear_cross_entropy(x, w, t)
    x[7, 3], x[100], x[250, 0] = math.nan, math.inf, -math.inf
    loss = linear_cross_entropy(x, w, t)
    bad = torch.zeros(300, dtype=torch.bool, device="cuda")
    bad[[7, 100, 250]] = True
    assert loss[bad].isnan().all() and torch.equal(loss[~bad], clean[~bad])
    far = t.clone()
    far[[5, 9]] = torch.tensor([900, 1 << 40], device="cuda")
    x, w, _, _ = _inputs(300, 72, 900, False)
    X, W = x.requires_grad_(True), w.requires_grad_(True)
    loss = linear_cross_entropy(X, W, far)
    assert loss[[5, 9]].isnan().all() and not loss.isnan().sum() > 2
    dx, dw = torch.autograd.grad(loss, (X, W), g)
    none = torch.where((far >= 900), -1, far)
    want = torch.autograd.grad(linear_cross_entropy(X, W, none), (X, W), g)
    assert not dx[[5, 9]].any() and torch.equal(dx, want[0]) and torch.equal(dw, want[1])


def test_gradient_by_differences(built_lib):
    """Losses in f32 of moved inputs: the directional derivative, with steps that bf16 holds exactly."""
    x, w, t, _ = _inputs(40, 64, 500, True)
    g = torch.rand(40, generator=_gen(8), device="cuda")
    X, W = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    dx, dw = torch.autograd.grad(linear_cross_entropy(X, W, t, 0.1), (X, W), g)
    for leaf, d in ((0, dx), (1, dw)):
        at = [x.double(), w.double()]
        step = torch.randn(at[leaf].shape, generator=_gen(9), device="cuda") * 0.02
        up, down = [v.clone() for v in (x, w)], [v.clone() for v in (x, w)]
        up[leaf], down[leaf] = (up[leaf].float() + step).bfloat16(), (down[leaf].float() - step).bfloat16()
        moved = up[leaf].double() - down[leaf].double()
        want = ((linear_cross_entropy(up[0], up[1], t, 0.1).double() - linear_cross_entropy(down[0], down[1], t, 0.1).double()) * g).sum()
        # the sum is linear but for the third derivative, 0.02^2 of it; losses of 6 within 2^-20 of themselves
        assert ((d.double() * moved).sum() - want).abs() <= 2e-2 * (d.double().norm() * moved.norm()) / math.sqrt(500) + 40 * 6 * 2.0 ** -20


def test_one_gradient_alone_types_and_empty_calls(built_lib):
    x, w, t, g = _inputs((2, 30), 48, 333, True)
    both = _check(x, w, t, 0.0, g)
    X, W = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(X, w, t), X, g)[0], both[1])
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(x, W, t), W, g)[0], both[2])
    for kind in (torch.int32, torch.int16):
        assert torch.equal(linear_cross_entropy(x, w, t.to(kind)), both[0])
    assert both[2].stride() == w.stride()
    shared = x.detach().requires_grad_(True)                  # broadcast positions: their gradients meet
    d = torch.autograd.grad(linear_cross_entropy(shared[:1].expand(3, -1, -1), w, t[:1].expand(3, -1)).sum(), shared)[0]
    assert d.shape == x.shape and not d[1].any()
    for lead in ((0,), (3, 0), (0, 4)):
        e = torch.empty(*lead, 48, device="cuda", dtype=torch.bfloat16).requires_grad_(True)
        loss = linear_cross_entropy(e, W, torch.empty(lead, device="cuda", dtype=torch.int64))
        de, dW = torch.autograd.grad(loss.sum(), (e, W))
        assert loss.shape == lead and de.shape == e.shape and not dW.any()


def test_refusals(built_lib):
    x, w, t, g = _inputs(6, 16, 20, False)
    for bad, error in (((x.cpu(), w, t), RuntimeError), ((x, w.cpu(), t), RuntimeError), ((x, w, t.cpu()), RuntimeError), ((x.float(), w, t), TypeError), ((x, w.float(), t), TypeError), ((x.half(), w.half(), t), TypeError),
                       ((x, w[:8], t), ValueError), ((x, w, t[:5]), ValueError), ((x, w[0], t), ValueError), ((x, w[:, :0], t), ValueError), ((x, w, t.float()), TypeError), ((x, w, t, 1.5), ValueError),
                       ((x, w, t, -0.1), ValueError), ((x, w, t, math.nan), ValueError)):
        with pytest.raises(error):
            linear_cross_entropy(*bad)
    X = x.detach().requires_grad_(True)
    (d,) = torch.autograd.grad(linear_cross_entropy(X, w, t).sum(), X, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(d.float().sum(), X)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda y: linear_cross_entropy(y, w, t[:1]))(x.view(6, 1, 16))


def test_captured_with_an_eager_graph_alive(built_lib):
    x, w, t, g = _inputs(200, 64, 700, False, ignored=0.3)
    X, W = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    eager = linear_cross_entropy(X, W, t)
    want = torch.autograd.grad(eager, (X, W), g, retain_graph=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        Y, Z = X.detach().requires_grad_(True), W.detach().requires_grad_(True)      # the same memory; torch binds a leaf's own node to the stream it was first used on
        torch.autograd.grad(linear_cross_entropy(Y, Z, t), (Y, Z), g)
        graphs = []
        for _ in range(2):                                   # two graphs, each with a workspace of its own
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                loss = linear_cross_entropy(Y, Z, t)
                grads = torch.autograd.grad(loss, (Y, Z), g)
            graphs.append((graph, loss, grads))
    torch.cuda.current_stream().wait_stream(side)
    with torch.no_grad():
        X.copy_(X.flip(0)); t.copy_(t.flip(0)); g.copy_(g.flip(0))
    for graph, loss, grads in graphs:
        graph.replay()
        graph.replay()
    torch.cuda.synchronize()
    for graph, loss, grads in graphs:
        assert torch.equal(loss.detach().flip(0), eager.detach()) and torch.equal(grads[0].flip(0), want[0])
        assert (grads[1].double() - want[1].double()).norm() <= 2.0 ** -8 * want[1].double().norm()      # other sums' order


@pytest.mark.parametrize("tied", (False, True))
@pytest.mark.parametrize("offset", range(9))
def test_weights_that_are_copied_first_give_the_same_bits(built_lib, tied, offset):
    """Columns of a wider array, from any element on: what TMA cannot read is moved, and nothing else changes; the last row ends with the array."""
    g = torch.Generator(device="cuda").manual_seed(70 + offset)
    inner, outer = 328, 137
    wide = torch.randn(outer, inner + offset, generator=g, device="cuda").bfloat16()
    view = wide[:, offset:]
    weight, whole = (view.t(), view.clone().t()) if tied else (view, view.clone())
    x = torch.randn(70, weight.shape[0], generator=g, device="cuda").bfloat16()
    t = torch.randint(0, weight.shape[1], (70,), generator=g, device="cuda")
    up = torch.rand(70, generator=g, device="cuda")
    got, want = [], []
    for w, to in ((weight, got), (whole, want)):
        a, b = x.clone().requires_grad_(True), w.detach().requires_grad_(True)
        loss = linear_cross_entropy(a, b, t, smoothing=0.1)
        to += [loss, *torch.autograd.grad(loss, (a, b), up)]
    assert all(torch.equal(a, b) for a, b in zip(got, want))
