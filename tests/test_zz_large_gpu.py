"""Offsets beyond 32 bits.  The file name sorts behind the others: what an allocator keeps of arrays of gigabytes is no matter to them then."""
import pytest
import torch

from pratchya_b200._nnx_impl import token_logprobs
from pratchya_b200._qualia import dequantize_int4_impl, int4_matmul_impl

pytestmark = pytest.mark.gpu


def test_rows_beyond_two_to_the_31(built_lib):
    """33000 x 65536 logits: the last rows, and their gradient, as if they were alone (their place among 16 bytes is the same)."""
    z = torch.zeros(33000, 65536, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(17)
    few = (torch.randn(5, 65536, generator=g, device="cuda") * 3).bfloat16()
    tokens = torch.randint(0, 65536, (5,), generator=g, device="cuda")
    z[-5:] = few
    t = torch.zeros(33000, dtype=torch.int64, device="cuda")
    t[-5:] = tokens
    z.requires_grad_(True)
    out = token_logprobs(z, t, 3)
    logp = torch.log_softmax(few.double(), -1)
    order = torch.sort(few, dim=-1, descending=True, stable=True).indices[:, :3]
    assert torch.equal(out.top_tokens[-5:], order) and (out.entropy[-5:].double() + (logp.exp() * logp).sum(-1)).abs().max() <= 1e-4
    assert (out.logprobs[-5:].double() - logp.gather(1, tokens[:, None])[:, 0]).abs().max() <= 1e-4
    (g,) = torch.autograd.grad(out.logprobs[-5:].sum(), z)
    alone = few.clone().requires_grad_(True)
    (want,) = torch.autograd.grad(token_logprobs(alone, t[-5:], 3).logprobs.sum(), alone)
    assert (g[-5:].float() - want.float()).abs().max() <= 2.0 ** -8 and (g[:-5] == 0).all()


def test_codes_beyond_two_to_the_32(built_lib):
    """4.6 GB of codes: the last tile's columns as if it were alone."""
    depth, cols = 16384, 562000
    tiles = (-(-cols // 16), depth // 128)
    q = torch.randint(0, 256, (*tiles, 1024), dtype=torch.uint8, device="cuda")
    scale = torch.rand(*tiles, 16, 1, device="cuda").bfloat16()
    assert q.numel() > 2 ** 32
    x = torch.randn(2, depth, device="cuda")
    y = int4_matmul_impl(x, q, scale, None, cols)
    w = dequantize_int4_impl(q[-1:], scale[-1:], None, (depth, 16)).double()
    want = x.double() @ w
    # whole numbers up to a block's scale: a row's error is that of 128 + 3 additions in f32
    assert ((y[:, -16:].double() - want).abs() <= 140 * 2.0 ** -24 * (x.double().abs() @ w.abs())).all()


def test_weights_and_tables_beyond_two_to_the_31(built_lib):
    """140001 words of 16384, 2.3 billion numbers: the losses of the last words, and the weight's gradient there, as if those words' weights were alone at their place among logits that are
    far below; a table of a billion rows' bytes: its last rows and their gradient."""
    from pratchya_b200._nnx_impl import embedding_lookup, linear_cross_entropy
    vocab, depth = 140001, 16384
    g = torch.Generator(device="cuda").manual_seed(19)
    w = torch.zeros(vocab, depth, dtype=torch.bfloat16, device="cuda")
    few = (torch.randn(9, depth, generator=g, device="cuda") / 16).bfloat16()
    w[-9:] = few
    assert w.numel() > 2 ** 31
    x = torch.randn(20, depth, generator=g, device="cuda").bfloat16()
    t = torch.randint(vocab - 9, vocab, (20,), generator=g, device="cuda")
    w.requires_grad_(True)
    loss = linear_cross_entropy(x, w.t(), t)
    z = x.double() @ few.double().t()
    lse = torch.logsumexp(torch.cat([z, torch.full((20, 1), 0.0, device="cuda", dtype=torch.float64) + torch.log(torch.tensor(vocab - 9.0, device="cuda", dtype=torch.float64))], 1), 1)
    want = lse - z.gather(1, (t - vocab + 9)[:, None])[:, 0]
    assert (loss.double() - want).abs().max() <= 1e-4
    (d,) = torch.autograd.grad(loss.sum(), w)
    p = (z - lse[:, None]).exp() - torch.nn.functional.one_hot(t - vocab + 9, 9)
    exact = p.t() @ x.double()
    assert (d[-9:].double() - exact).norm() <= 3 * 2.0 ** -8 * exact.norm()
    rest = (torch.zeros_like(lse) - lse).exp() @ x.double()                # what every other word's row is
    assert (d[:2].double() - rest).norm() <= 3 * 2.0 ** -8 * 2 ** 0.5 * rest.norm()
    del w, d
    table = torch.zeros(2 ** 20 + 3, 2056, dtype=torch.bfloat16, device="cuda").requires_grad_(True)
    with torch.no_grad():
        table[-3:] = torch.randn(3, 2056, generator=g, device="cuda").bfloat16()
    ids = torch.tensor([2 ** 20 + 2, 5, -1, 2 ** 20, -3], device="cuda")
    rows = embedding_lookup(table, ids)
    assert torch.equal(rows, table[ids]) and table.numel() > 2 ** 31
    (d,) = torch.autograd.grad(rows, table, torch.ones_like(rows))
    assert (d[-1] == 2).all() and (d[-2] == 0).all() and (d[-3] == 2).all() and (d[5] == 1).all() and d.float().sum() == 5 * 2056
