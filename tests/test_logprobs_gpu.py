"""Log probabilities of given tokens, entropy and best alternatives, and their gradient, against the definition in 64 bits: vocabularies
around every edge of the row's split into threads, vectors and CTAs, rows at any alignment and stride, masks that leave little or nothing,
ties, and rows whose best logits crowd into a few threads."""
import math

import pytest
import torch
from torch.autograd import forward_ad

from pratchya_b200._nnx_impl import token_logprobs

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _definition(z, tokens, top):
    """Everything in 64 bits: (logprobs, entropy, top values, top tokens, logp, p, dead rows)."""
    z = z.double()
    dead = (z == -math.inf).all(-1, keepdim=True)
    logp = torch.where(dead, -math.inf, torch.log_softmax(torch.where(dead, 0.0, z), -1))
    p = logp.exp()
    entropy = -torch.where(p > 0, p * logp, 0.0).sum(-1)
    picked = None
    if tokens is not None:
        t = tokens.reshape(*z.shape[:-1], -1)
        picked = torch.where(t < 0, 0.0, logp.gather(-1, t.clamp(min=0))).reshape(tokens.shape)
    order = torch.sort(z + 0.0, dim=-1, descending=True, stable=True).indices[..., :top]
    return picked, entropy, logp.gather(-1, order), order, logp, p, dead


def _errors(z, logp, p, dead):
    """Bounds on the errors of log S, of a row's entropy and of log p.  An exponential's argument is a difference rounded to 2^-24 of it and again
    where it is scaled to base 2, the instruction is within 2^-22; a thread adds at most vocab / 256 terms and ten more where threads meet; a
    logarithm and two differences round to 2^-24 of what they are."""
    vocab = z.shape[-1]
    z64 = z.double()
    m = torch.where(dead, 0.0, z64.amax(-1, keepdim=True))
    d = torch.where(p > 0, (z64 - m).abs(), 0.0)
    far = (p * d).sum(-1)
    adds = (vocab / 256 + 20) * 2.0 ** -24
    log_s = (-torch.where(p > 0, logp - (z64 - m), 0.0)).abs().amax(-1)
    e_log_s = far * 2.0 ** -22 + 2.0 ** -22 + adds + 2.0 ** -23 * log_s
    e_entropy = e_log_s + (p * d * (d * 2.0 ** -22)).sum(-1) + far * (2.0 ** -21 + 2 * adds + e_log_s) + 2.0 ** -22 * (log_s + far)
    return log_s, e_log_s, e_entropy


def _check(z, tokens, top):
    out = token_logprobs(z, tokens, top)
    picked, entropy, tops, order, logp, p, dead = _definition(z, tokens, top)
    log_s, e_log_s, e_entropy = _errors(z, logp, p, dead)
    lead = z.shape[:-1]
    assert out.entropy.shape == lead and out.top_tokens.shape == (*lead, top) and out.top_logprobs.shape == (*lead, top)
    assert torch.equal(out.top_tokens, order)
    assert ((out.entropy.double() - entropy).abs() <= e_entropy).all(), ((out.entropy.double() - entropy).abs() / e_entropy).max()

    def close(got, want, what):
        fine = torch.isfinite(want)
        assert torch.equal(fine, torch.isfinite(got)) and torch.equal(got[~fine].double(), want[~fine]), what
        by = e_log_s.unsqueeze(-1) + 2.0 ** -23 * (want.abs() + log_s.unsqueeze(-1))
        assert ((got.double() - want).abs()[fine] <= by.expand_as(want)[fine]).all(), what

    close(out.top_logprobs, tops, "alternatives")
    if tokens is None:
        assert out.logprobs is None
    else:
        assert out.logprobs.shape == tokens.shape
        close(out.logprobs.reshape(*lead, -1), picked.reshape(*lead, -1), "given tokens")
    return out


def _case(rows, vocab, dtype, seed, n=1, sharp=3.0):
    g = _gen(seed)
    z = (torch.randn(rows, vocab, generator=g, device="cuda") * sharp).to(DTYPES[dtype])
    tokens = torch.randint(-1, vocab, (rows, n) if n > 1 else (rows,), generator=g, device="cuda")
    return z, tokens


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (2, 2, 2), (3, 7, 7), (1, 31, 5), (5, 100, 100), (3, 255, 64), (3, 1000, 128), (2, 1023, 1), (2, 4096, 20), (3, 4099, 0),
                                            (1, 32003, 5), (2, 65536, 64), (1, 131072, 128), (400, 1025, 3), (320, 8200, 17), (300, 32003, 128)])
def test_rows_of_any_length(built_lib, rows, vocab, top, dtype):
    z, tokens = _case(rows, vocab, dtype, rows * 7 + vocab)
    z[0] -= 50.0                                       # a row far from zero
    z[-1, -1] = 40.0                                   # its maximum is the last logit
    _check(z, tokens, top)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape,top", [((3, 5, 1001), 4), ((2, 301, 515), 9), ((2, 3, 65536), 6)])
def test_views_are_read_in_place(built_lib, shape, top, dtype):
    bsz, steps, vocab = shape
    z, _ = _case(bsz * (steps + 1), vocab, dtype, vocab)
    z = z.reshape(bsz, steps + 1, vocab)
    tokens = torch.randint(0, vocab, (bsz, steps), generator=_gen(3), device="cuda")
    whole = _check(z[:, :-1], tokens, top)
    again = token_logprobs(z[:, :-1].contiguous(), tokens, top)
    # the same values; the last bits may go by where a row lies among 16 bytes, since its first logits go to other threads
    assert torch.equal(whole.top_tokens, again.top_tokens) and (whole.entropy - again.entropy).abs().max() <= 1e-4
    _check(z[:, 1:], tokens, top)
    _check(z.transpose(0, 1), torch.randint(0, vocab, (steps + 1, bsz), device="cuda"), top)
    _check(z[..., 1:], None, top)                      # rows that begin off 16 bytes
    _check(z[0, 0], tokens[0, 0], top)                 # one row without a leading dimension
    _check(z[:1].expand(4, -1, -1)[:, :2], torch.randint(0, vocab, (4, 2), device="cuda"), top)
    _check(z.reshape(1, bsz, steps + 1, vocab)[:, :, 1:], tokens.reshape(1, bsz, steps), top)
    _check(z.permute(2, 1, 0)[: steps, :, :], None, 1)            # no row lies together: a copy is made


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [6, 330])
def test_masks(built_lib, rows, dtype):
    z, tokens = _case(rows, 9001, dtype, 5, n=3)
    low = torch.finfo(z.dtype).min
    z[0] = -math.inf                                   # nothing left
    z[1] = -math.inf
    z[1, 8000] = 1.5                                   # one left
    z[2, :8900] = -math.inf
    z[3, 1:9000] = low                                 # the type's lowest value weighs nothing, but is finite
    z[4] = low                                         # ... and alone it is all there is: uniform
    z[5] = low
    z[5, 17] = -math.inf
    tokens[:, 0] = 8000
    out = _check(z, tokens, 40)
    assert out.entropy[0] == 0 and out.top_tokens[0].tolist() == list(range(40)) and (out.top_logprobs[0] == -math.inf).all()
    assert out.entropy[1] == 0 and out.top_tokens[1, :3].tolist() == [8000, 0, 1] and out.logprobs[1, 0] == 0


def test_not_a_number(built_lib):
    for rows in (4, 300):
        z, tokens = _case(rows, 5000, "f32", 9)
        tokens = tokens.clamp(min=0)
        clean = token_logprobs(z, tokens, 8)
        z[1, 77] = math.nan
        z[2, 4000] = math.inf
        z[3] = math.nan
        out = token_logprobs(z, tokens, 8)
        for i in (1, 2, 3):
            assert torch.isnan(out.entropy[i]) and torch.isnan(out.logprobs[i]) and torch.isnan(out.top_logprobs[i]).all()
            assert (0 <= out.top_tokens[i]).all() and (out.top_tokens[i] < 5000).all()
        assert out.top_tokens[2, 0] == 4000 and out.top_tokens[3].tolist() == list(range(8))
        keep = [i for i in range(rows) if i not in (1, 2, 3)]
        assert all(torch.equal(a[keep], b[keep]) for a, b in zip(out, clean))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab", [(5, 2000), (5, 70001), (310, 9001)])
def test_many_alternatives_where_logits_are_no_numbers(built_lib, rows, vocab, dtype):
    z, tokens = _case(rows, vocab, dtype, 19)
    tokens = tokens.clamp(min=0)
    z[1, 5::3] = math.nan
    z[2, 40:1900] = math.inf
    z[3] = math.nan
    z[4, 3:] = math.nan                                # three numbers, then the first of what is none
    out = token_logprobs(z, tokens, 128)
    want = torch.sort(torch.where(z.isnan(), -math.inf, z.float()) + 0.0, dim=-1, descending=True, stable=True).indices[:, :128]
    assert torch.equal(out.top_tokens, want)
    assert torch.isnan(out.top_logprobs[1:5]).all() and torch.isnan(out.entropy[1:5]).all()
    keep = [i for i in range(rows) if not 1 <= i < 5]
    _check(z[keep], tokens[keep], 128)


def test_tokens_that_are_none_or_beyond(built_lib):
    z, _ = _case(5, 1000, "f32", 1)
    tokens = torch.tensor([0, -1, 999, 1000, -100], device="cuda")
    out = token_logprobs(z, tokens)
    assert out.logprobs[1] == 0 and out.logprobs[4] == 0 and torch.isnan(out.logprobs[3]) and torch.isfinite(out.logprobs[[0, 2]]).all()
    assert torch.equal(out.logprobs[[0, 2]], token_logprobs(z, tokens.clamp(0, 999).to(torch.int32)).logprobs[[0, 2]])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [2, 320])
def test_ties_go_to_the_lowest_index(built_lib, rows, dtype):
    g = _gen(rows)
    z = torch.randint(-3, 3, (rows, 20000), generator=g, device="cuda").to(DTYPES[dtype])
    z[0] = 2.0                                         # all equal
    z[1, ::2] = 0.0
    z[1, 1::2] = -0.0                                  # -0 is 0
    _check(z, None, 128)
    assert token_logprobs(z, None, 128).top_tokens[0].tolist() == list(range(128))


@pytest.mark.parametrize("rows", [1, 310])
@pytest.mark.parametrize("period", [4, 1024, 1536])
def test_best_logits_that_crowd_together(built_lib, rows, period):
    """Large logits in every period-th place's neighbours, in rising order: whichever threads have them have far more than their share."""
    vocab = 131072
    z, _ = _case(rows, vocab, "f32", period, sharp=1.0)
    place = torch.arange(vocab, device="cuda")
    z = torch.where(place % period < 16, 20.0 + place / 1e5, z)
    _check(z, None, 16)
    _check(z.flip(-1).contiguous(), None, 128)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("top", [3, 17, 60, 128])
@pytest.mark.parametrize("rows,vocab", [(2, 300), (3, 1000), (160, 1001), (2, 2051), (300, 4096), (2, 9001), (310, 9001), (2, 65536), (160, 65535)])
def test_few_values(built_lib, rows, vocab, top, dtype):
    """Rows of one, two, five, fifty and some thousand different values, a row of which two thirds are -inf, and one of -inf but for five: the bound's value is
    many logits', and the number of alternatives ends inside a vector."""
    g = _gen(vocab + top)
    levels = torch.tensor([1, 2, 5, 50, 5000], device="cuda")[torch.arange(rows, device="cuda") % 5].unsqueeze(1)
    z = ((torch.rand(rows, vocab, generator=g, device="cuda") * levels).floor() * 0.125 - 3.0).to(DTYPES[dtype])
    z[1, torch.rand(vocab, generator=g, device="cuda") < 0.67] = -math.inf
    if rows > 2:
        z[2, 5:] = -math.inf
    _check(z, None, top)
    _check(z[:, 1:], None, min(top, vocab - 1))        # off 16 bytes


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("top", [5, 40, 128])
@pytest.mark.parametrize("rows,vocab", [(6, 131073), (6, 3000), (300, 20000)])
def test_rows_with_less_left_than_is_wanted(built_lib, rows, vocab, top, dtype):
    """Nothing, five, a hundred and thirty-nine logits above -inf, at a row's start, end and all over it, and rows of the type's lowest value but for as many:
    what fills the alternatives up are the first of the others, of a row's several CTAs, too."""
    g = _gen(vocab + top)
    z, _ = _case(rows, vocab, dtype, vocab)
    low = torch.finfo(z.dtype).min
    keep = torch.zeros(rows, vocab, dtype=torch.bool, device="cuda")
    keep[1, -5:] = True
    keep[2, torch.randperm(vocab, generator=g, device="cuda")[:100]] = True
    keep[3, :39] = True
    keep[4, torch.randperm(vocab, generator=g, device="cuda")[:39]] = True
    keep[5, vocab // 2:vocab // 2 + 100] = True
    z[:6] = torch.where(keep[:6], z[:6], -math.inf)
    if rows > 12:
        z[6:12] = torch.where(keep[:6], z[6:12], low)
    _check(z, None, top)
    z[:6] = torch.where(z[:6] == -math.inf, low, z[:6])
    z[0, 7::9] = -math.inf
    _check(z, None, top)


def test_another_stream_and_a_graph(built_lib):
    z, tokens = _case(3, 32003, "bf16", 4)
    want = token_logprobs(z, tokens, 5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = token_logprobs(z, tokens, 5)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = token_logprobs(z, tokens, 5)
    z.copy_(z.flip(0))
    graph.replay()
    assert torch.equal(held.top_tokens, want.top_tokens.flip(0))
    want = token_logprobs(z, tokens, 5)                # a row's last bits go by where it lies among 16 bytes
    assert all(torch.equal(a, b) for a, b in zip(held, want))


# ---- the gradient ------------------------------------------------------------------------------------------------------

def _check_gradient(z, tokens, top, seed, use=(True, True, True)):
    g = _gen(seed)
    zz = z.detach().requires_grad_(True)
    out = token_logprobs(zz, tokens, top)
    picked, entropy, tops, order, logp, p, dead = _definition(z, tokens, top)
    lead = z.shape[:-1]
    gl, ge, gt = (torch.randn(s, generator=g, device="cuda") for s in (tokens.shape, lead, (*lead, top)))
    outs = [(o, c) for o, c, u in zip((out.logprobs, out.entropy, out.top_logprobs), (gl, ge, gt), use) if u]
    (dz,) = torch.autograd.grad([o for o, _ in outs], zz, [c for _, c in outs])
    assert dz.dtype is z.dtype and dz.shape == z.shape
    t = tokens.reshape(*lead, -1)
    gl, ge, gt = (c.double() * u for c, u in zip((gl, ge, gt), use))
    gl = torch.where(t < 0, 0.0, gl.reshape(t.shape))
    total = (gl.sum(-1) + gt.sum(-1)).unsqueeze(-1)
    inner = torch.where(p > 0, logp + entropy.unsqueeze(-1), 0.0)
    want = -p * (total + ge.unsqueeze(-1) * inner)
    hot, size = torch.zeros_like(want), torch.zeros_like(want)
    for index, value in ((t.clamp(min=0), torch.where(dead, 0.0, gl)), (order, torch.where(dead, 0.0, gt))):
        hot.scatter_add_(-1, index, value)
        size.scatter_add_(-1, index, value.abs())
    want = want + hot
    log_s, e_log_s, e_entropy = _errors(z, logp, p, dead)
    x = torch.where(p > 0, logp.abs(), 0.0)
    e_x = e_log_s.unsqueeze(-1) + 2.0 ** -23 * (x + log_s.unsqueeze(-1))
    g_sum = (gl.abs().sum(-1) + gt.abs().sum(-1)).unsqueeze(-1)
    ge = ge.abs().unsqueeze(-1)
    # p by its exponential's argument, the sums of cotangents (of up to 256 terms in 32 lanes) and the entropy's terms by theirs
    by = p * ((e_x + x * 2.0 ** -23 + 2.0 ** -21) * (total.abs() + ge * inner.abs()) + g_sum * 13 * 2.0 ** -24 + ge * (e_x + e_entropy.unsqueeze(-1) + 2.0 ** -22 * (x + inner.abs())))
    by = by + size * 2.0 ** -20 + 2.0 ** -23 * want.abs()
    if z.dtype is torch.bfloat16:
        by = by + 2.0 ** -8 * (want.abs() + by)
    assert ((dz.double() - want).abs() <= by + 1e-37).all(), ((dz.double() - want).abs() / (by + 1e-37)).max()
    return dz


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab,n,top", [(1, 1, 1, 1), (2, 3, 1, 0), (3, 100, 4, 100), (2, 1000, 128, 128), (3, 4099, 1, 5), (2, 65536, 16, 64), (300, 2049, 1, 0), (310, 4096, 3, 2)])
def test_gradient(built_lib, rows, vocab, n, top, dtype):
    z, tokens = _case(rows, vocab, dtype, vocab + n, n=n)
    _check_gradient(z, tokens, top, 11)


@pytest.mark.parametrize("use", [(True, False, False), (False, True, False), (False, False, True)])
def test_gradient_of_one_output(built_lib, use):
    z, tokens = _case(4, 3001, "f32", 2, n=5)
    _check_gradient(z, tokens, 7, 3, use)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_gradient_of_views_masks_and_repeated_tokens(built_lib, dtype):
    z, _ = _case(4 * 6, 1003, dtype, 8)
    z = z.reshape(4, 6, 1003)
    z[0, 0] = -math.inf
    z[1, 1, :1000] = -math.inf
    z[1, 2, 5:] = torch.finfo(z.dtype).min
    tokens = torch.randint(0, 1003, (4, 5, 6), generator=_gen(1), device="cuda")
    tokens[..., 3] = tokens[..., 0]                    # a token given twice, and one that is among the best as well
    tokens[..., 4] = z[:, :-1].argmax(-1)
    tokens[2, 2] = -1
    dz = _check_gradient(z[:, :-1], tokens, 9, 4)
    assert (dz[0, 0] == 0).all()
    full = z.detach().requires_grad_(True)             # through the view: the last position's gradient is zero
    token_logprobs(full[:, :-1], tokens).logprobs[1:].sum().backward()
    assert (full.grad[:, -1] == 0).all() and (full.grad[2, 2] == 0).all() and full.grad[1, 0].abs().sum() > 0
    shared = z[:1, :1].detach().requires_grad_(True)   # one row read by many positions: its gradients add up
    t = torch.tensor([[1], [2], [2]], device="cuda")
    token_logprobs(shared.expand(3, 1, -1), t).logprobs.sum()


def test_gradient_of_a_shared_row(built_lib):
    z, _ = _case(1, 501, "f32", 21)
    z.requires_grad_(True)
    t = torch.tensor([[7, 9], [9, -1], [500, 9]], device="cuda")
    token_logprobs(z.expand(3, -1), t).logprobs.sum().backward()
    p = torch.softmax(z.detach().double(), -1)[0]
    want = -5 * p
    want[7] += 1; want[9] += 3; want[500] += 1
    assert (z.grad[0].double() - want).abs().max() <= 5 * 2.0 ** -20


def test_gradient_without_tokens_and_without_use(built_lib):
    z, _ = _case(3, 1001, "f32", 31)
    z.requires_grad_(True)
    out = token_logprobs(z)
    assert out.logprobs is None and out.top_logprobs.shape == (3, 0)
    out.entropy.sum().backward()
    z64 = z.detach().double().requires_grad_(True)
    logp = torch.log_softmax(z64, -1)
    (-(logp.exp() * logp).sum()).backward()
    assert (z.grad.double() - z64.grad).abs().max() <= 2.0 ** -19
    with torch.no_grad():
        assert not token_logprobs(z).entropy.requires_grad
    assert not token_logprobs(z, None, 3).top_tokens.requires_grad
    best = token_logprobs(z, None, 2)
    (g,) = torch.autograd.grad(best.top_logprobs[:, 0].sum(), z)
    assert (g.sum(-1).abs() <= 2.0 ** -18).all() and (g.gather(1, best.top_tokens[:, :1]) > 0).all()


def test_gradient_against_differences(built_lib):
    """A step h along a direction v of unit size: (f(z + h v) - f(z - h v)) / 2h is v . grad f up to h^2 / 6 of a third derivative and 2^-22 of |f| / h.  f is a sum
    of log probabilities and entropies of three rows; a third derivative of either along a unit vector is below 8 (1 + entropy)."""
    z, tokens = _case(3, 700, "f32", 6, n=2, sharp=1.0)
    tokens = tokens.clamp(min=0)

    def f(x):
        r = token_logprobs(x, tokens, 4)
        return (r.logprobs.double() * 0.5).sum() + r.entropy.double().sum() + 0.25 * r.top_logprobs.double().sum()

    x = z.clone().requires_grad_(True)
    f(x).backward()
    h = 2.0 ** -5
    for seed in range(4):
        v = torch.randn(z.shape, generator=_gen(seed), device="cuda")
        if seed % 2:
            v = x.grad.clone()
        v = v / v.norm()
        slope = float((f(z + h * v) - f(z - h * v)) / (2 * h))
        size = float(f(z).abs()) + 40
        assert abs(slope - float((x.grad.double() * v.double()).sum())) <= h * h / 6 * 8 * 8 * 3 + 2.0 ** -22 * size / h


def test_refusals(built_lib):
    z, tokens = _case(4, 1000, "f32", 0)
    with pytest.raises(RuntimeError):
        token_logprobs(z.cpu())
    with pytest.raises(TypeError):
        token_logprobs(z.half())
    with pytest.raises(TypeError):
        token_logprobs(z, tokens.float())
    with pytest.raises(RuntimeError):
        token_logprobs(z, tokens.cpu())
    for bad in (-1, 129, 1001):
        with pytest.raises(ValueError):
            token_logprobs(z, tokens, bad)
    with pytest.raises(ValueError):
        token_logprobs(z[:, :5], None, 6)
    with pytest.raises(ValueError):
        token_logprobs(z, tokens[:3])
    with pytest.raises(ValueError):
        token_logprobs(z, torch.zeros(4, 129, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError):
        token_logprobs(z[:, :0])
    with pytest.raises(RuntimeError):                  # no second derivative
        x = z.clone().requires_grad_(True)
        (g,) = torch.autograd.grad(token_logprobs(x, tokens.clamp(min=0)).logprobs.sum(), x, create_graph=True)
        g.sum().backward()
    none = token_logprobs(z[:0], tokens[:0], 3)
    assert none.logprobs.shape == (0,) and none.top_tokens.shape == (0, 3)
    empty = z[:0].clone().requires_grad_(True)
    token_logprobs(empty, tokens[:0], 3).entropy.sum().backward()
    assert empty.grad.shape == (0, 1000)


@pytest.mark.parametrize("ctas", [2, 4, 8])
@pytest.mark.parametrize("vocab,top", [(1, 1), (40, 20), (4099, 0), (4099, 5), (4099, 128)])
def test_rows_so_short_that_a_cluster_has_hardly_begun(built_lib, diag_lib, monkeypatch, ctas, vocab, top):
    """The diagnostics build gives a row to as many CTAs as it is told: of a short row most have nothing, and hand that to the first one at once."""
    monkeypatch.setenv("PB_LP_CTAS", str(ctas))
    rows = 301
    z, tokens = _case(rows, vocab, "f32", ctas + vocab)
    tokens = tokens.clamp(min=0)
    f32 = lambda *shape: torch.full(shape, math.nan, device="cuda")
    logprobs, entropy, tops, best = f32(rows), f32(rows), f32(rows, top), torch.full((rows, top), -1, device="cuda")
    assert diag_lib.pb_token_logprobs(z.data_ptr(), 0, 1, rows, 0, vocab, vocab, tokens.data_ptr(), 1, top, logprobs.data_ptr(), entropy.data_ptr(), tops.data_ptr() if top else None,
                                      best.data_ptr() if top else None, None, torch.cuda.current_stream().cuda_stream) == 0
    picked, want, values, order, logp, p, dead = _definition(z, tokens, top)
    log_s, e_log_s, e_entropy = _errors(z, logp, p, dead)
    assert torch.equal(best, order) and ((entropy.double() - want).abs() <= e_entropy).all()
    for got, exact in ((logprobs.unsqueeze(-1), picked.unsqueeze(-1)), (tops, values)):
        assert ((got.double() - exact).abs() <= e_log_s.unsqueeze(-1) + 2.0 ** -23 * (exact.abs() + log_s.unsqueeze(-1))).all()


def test_no_derivative_is_dropped_without_a_word(built_lib, monkeypatch):
    z, tokens = _case(3, 1000, "f32", 23)
    for grads in (True, False):
        with torch.set_grad_enabled(grads):
            with forward_ad.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
                token_logprobs(forward_ad.make_dual(z, torch.ones_like(z)), tokens, 2)
            with pytest.raises(RuntimeError, match="traced"):
                torch.jit.trace(lambda t: token_logprobs(t, tokens, 2).entropy, z, check_trace=False)
    monkeypatch.delattr(forward_ad, "_current_level")          # a torch without its own name for it
    for grads in (True, False):
        with torch.set_grad_enabled(grads):
            assert torch.equal(token_logprobs(z, tokens, 2).entropy, token_logprobs(z.clone().requires_grad_(True), tokens, 2).entropy.detach())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_gradient_of_rows_without_a_logit_whatever_their_cotangents(built_lib, dtype):
    """A loss that divides or takes an exponential of the -inf of such a row hands back what is no number: the row has no gradient all the same, nor do the others lose theirs."""
    z, tokens = _case(4, 3001, dtype, 41, n=2)
    tokens = tokens.clamp(min=0)
    z[1] = -math.inf
    z.requires_grad_(True)
    out = token_logprobs(z, tokens, 3)
    cotangents = [torch.ones_like(t) for t in (out.logprobs, out.entropy, out.top_logprobs)]
    (want,) = torch.autograd.grad(out[:3], z, cotangents, retain_graph=True)
    for bad in (math.nan, math.inf, -math.inf):
        for which in range(3):
            g = [c.clone() for c in cotangents]
            g[which][1] = bad
            (got,) = torch.autograd.grad(out[:3], z, g, retain_graph=True)
            assert torch.equal(got, want) and (got[1] == 0).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_gradient_of_masked_logits_under_large_cotangents(built_lib, dtype):
    """What has no probability has no gradient, however large the entropy's cotangent is; the others' is that many times the one of a cotangent of 1."""
    z, _ = _case(3, 2003, dtype, 43, sharp=1.0)
    z[0, 5:1000] = -math.inf
    z[1, 7:] = torch.finfo(z.dtype).min
    z.requires_grad_(True)
    entropy = token_logprobs(z).entropy
    (one,) = torch.autograd.grad(entropy.sum(), z, retain_graph=True)
    for power in (29, 60, 90, 110):
        (got,) = torch.autograd.grad(entropy, z, torch.full_like(entropy, 2.0 ** power), retain_graph=True)
        assert (got[0, 5:1000] == 0).all() and (got[1, 7:] == 0).all()
        # what is below the type's normal numbers for a cotangent of 1 has fewer bits there
        fine = one.abs() >= 2.0 ** -100
        assert torch.equal(got[fine], (one.double() * 2.0 ** power).to(z.dtype)[fine]) and torch.isfinite(got).all()


def test_gradient_of_a_row_read_by_several_texts(built_lib):
    z, _ = _case(1, 1003, "f32", 47)
    shared = z[None].detach().requires_grad_(True)
    t = torch.tensor([[1], [2], [2]], device="cuda")
    token_logprobs(shared.expand(3, 1, -1), t).logprobs.sum().backward()
    want = -3 * torch.softmax(z.double(), -1)[0]
    want[1] += 1; want[2] += 2
    assert (shared.grad[0, 0].double() - want).abs().max() <= 3 * 2.0 ** -20


def test_a_number_of_alternatives_is_whole(built_lib):
    z, tokens = _case(3, 1000, "f32", 3)
    for bad in (2.5, 2.0, "2", None):
        with pytest.raises(TypeError):
            token_logprobs(z, tokens, bad)
    assert torch.equal(token_logprobs(z, tokens, torch.tensor(2)).top_tokens, token_logprobs(z, tokens, 2).top_tokens)
