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
