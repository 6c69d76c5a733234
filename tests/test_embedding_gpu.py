"""The embedding lookup and its gradient by sorted tokens: rows to the bit, gradients against sums in 64 bits over runs of tokens of every length, at and
around the edges of the blocks that add them up and of the sort's tiles and digits.

A gradient is a sum of n numbers in f32, in blocks of 32 and then eight ways: any order is within (n - 1) 2^-24 of the sum of magnitudes, this one within (32 + n / 256 + 10) 2^-24;
the product with scale and the rounding to the table's type half a step each."""
import math

import pytest
import torch

from pratchya_b200._nnx_impl import embedding_lookup

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _check(table, ids, scale=1.0, padding=None, seed=1):
    vocab, channels = table.shape
    row = torch.where(ids < 0, ids + vocab, ids)
    there = (row >= 0) & (row < vocab)
    pad = torch.zeros_like(there) if padding is None else there & (row == padding % vocab)
    want = (table[row.clamp(0, vocab - 1)].float() * scale).to(table.dtype)
    want = torch.where(pad.unsqueeze(-1), 0.0, torch.where(there.unsqueeze(-1), want, math.nan)).to(table.dtype)
    leaf = table.detach().requires_grad_(True)
    rows = embedding_lookup(leaf, ids, scale, padding)
    assert rows.dtype == table.dtype and rows.shape == want.shape and torch.equal(rows.nan_to_num(7.5), want.nan_to_num(7.5))
    with torch.no_grad():
        assert torch.equal(embedding_lookup(table, ids, scale, padding).nan_to_num(7.5), rows.nan_to_num(7.5))
    g = torch.randn(rows.shape, generator=_gen(seed), device="cuda").to(table.dtype)
    (d,) = torch.autograd.grad(rows, leaf, g)
    use = (there & ~pad).reshape(-1)
    at, gg = row.reshape(-1)[use], g.reshape(-1, channels)[use].double()
    zeros = torch.zeros(table.shape, dtype=torch.float64, device="cuda")
    exact = zeros.index_add(0, at, gg) * scale
    size = zeros.index_add(0, at, gg.abs()) * abs(scale)
    n = torch.zeros(vocab, dtype=torch.float64, device="cuda").index_add(0, at, torch.ones_like(at, dtype=torch.float64)).unsqueeze(-1)
    bound = torch.minimum(n, 42 + n / 256) * 2.0 ** -24 * size + (2.0 ** -23 + torch.finfo(table.dtype).eps / 2) * exact.abs() + 2.0 ** -126 * (size > 0)
    assert d.dtype == table.dtype and d.shape == table.shape
    off = (d.double() - exact).abs()
    assert (off <= bound).all(), (off / bound.clamp(min=1e-300)).max().item()
    assert not d[(n == 0).squeeze(-1)].any()
    assert torch.equal(torch.autograd.grad(embedding_lookup(leaf, ids, scale, padding), leaf, g)[0], d)      # the same bits again
    return rows.detach(), d


def _table(vocab, channels, dtype=F32, seed=0):
    return torch.randn(vocab, channels, generator=_gen(seed + vocab), device="cuda").to(dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab,channels", [(1, 1), (2, 3), (31, 4), (33, 8), (100, 127), (511, 128), (512, 130), (513, 1000), (1000, 1001), (5000, 2048), (300, 5003), (262143, 8), (262144, 8), (300000, 5)])
def test_any_table(built_lib, vocab, channels, dtype):
    for n in (1, 7, 500):
        ids = torch.randint(0, vocab, (n,), generator=_gen(n), device="cuda")
        _check(_table(vocab, channels, dtype), ids, 1.0 if n == 7 else 45.25)


@pytest.mark.parametrize("n", [1, 31, 32, 33, 63, 64, 65, 1023, 2047, 2048, 2049, 4096, 10001])
def test_runs_of_every_length(built_lib, n):
    table = _table(700, 20)
    _check(table, torch.full((n,), 699, device="cuda"))                                                   # one token throughout
    _check(table, torch.arange(n, device="cuda") % 700)                                                   # all of them in turn
    _check(table, torch.arange(n, device="cuda") // 31 % 700)                                             # runs that end around a block's end
    _check(table, torch.arange(n, device="cuda") // 32 % 700)
    _check(table, torch.arange(n, device="cuda") // 65 % 700)
    _check(table, torch.where(torch.rand(n, generator=_gen(n), device="cuda") < 0.9, 3, torch.randint(0, 700, (n,), generator=_gen(n), device="cuda")))
    _check(table, torch.where(torch.arange(n, device="cuda") % 2 == 0, 0, 699))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_text(built_lib, dtype):
    """Tokens as frequent as in a text, a step of training."""
    ids = (torch.exp(torch.rand(8, 1024, generator=_gen(5), device="cuda") * math.log(65536)) - 1).long().clamp(0, 65535)
    _check(_table(65536, 256, dtype), ids, 16.0)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_padding_and_ids_outside(built_lib, dtype):
    table = _table(300, 72, dtype)
    ids = torch.randint(0, 300, (4, 90), generator=_gen(6), device="cuda")
    for padding in (0, 299, -1, 150):
        padded = torch.where(torch.arange(90, device="cuda") > 40, padding % 300, ids)
        rows, d = _check(table, padded, 2.0, padding)
        assert not d[padding % 300].any() and not rows[:, 41:].any()
    _check(table, torch.full((70,), 5, device="cuda"), 1.0, 5)                                            # nothing but padding
    _check(table, ids - 300)                                                                              # from the end
    odd = ids.clone()
    odd[0, :4] = torch.tensor([300, -301, 1 << 40, -(1 << 62)], device="cuda")
    rows, _ = _check(table, odd, 1.0, 7)
    assert rows[0, :4].isnan().all() and not rows[0, 4:].isnan().any()
    table[9] = math.nan                                                                                   # a row that no token has reaches nothing
    _check(table, torch.where(ids == 9, 10, ids))


def test_views_types_and_devices_streams(built_lib):
    base = _table(400, 96)
    ids = torch.randint(0, 400, (3, 50), generator=_gen(7), device="cuda")
    for table in (base[:, 1:], base[1:], base[::2], base.t().contiguous().t(), base[:, ::3], base.flatten()[1:1 + 300 * 96].view(300, 96)):
        _check(table, ids % table.shape[0])
    for view in (ids.t(), ids[:, ::2], ids[0], ids[0, 0], ids[:1].expand(4, -1), ids[:0], ids[:, :0]):
        _check(base, view)
    for kind in (torch.int32, torch.int16, torch.uint8):
        assert torch.equal(embedding_lookup(base, (ids % 200).to(kind)), embedding_lookup(base, ids % 200))
    leaf = base.detach().requires_grad_(True)
    g = torch.randn(50, 96, generator=_gen(8), device="cuda")
    for gg in (g.expand(3, -1, -1), g[:, :1].expand(3, 50, 96), g.t().contiguous().t().expand(3, -1, -1)):      # broadcast and permuted cotangents
        got = torch.autograd.grad(embedding_lookup(leaf, ids), leaf, gg)[0]
        assert torch.equal(got, torch.autograd.grad(embedding_lookup(leaf, ids), leaf, gg.contiguous())[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = embedding_lookup(base, ids)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(there, embedding_lookup(base, ids))


def test_gradient_by_differences(built_lib):
    table, ids = _table(40, 12).double().float(), torch.randint(0, 40, (60,), generator=_gen(9), device="cuda")
    leaf = table.requires_grad_(True)
    w = torch.randn(60, 12, generator=_gen(10), device="cuda")
    (d,) = torch.autograd.grad(embedding_lookup(leaf, ids, 3.0), leaf, w)
    with torch.no_grad():
        step = torch.randn(40, 12, generator=_gen(11), device="cuda")
        moved = ((embedding_lookup(leaf + step, ids, 3.0).double() - embedding_lookup(leaf - step, ids, 3.0).double()) * w).sum() / 2
    assert (moved - (d.double() * step).sum()).abs() <= 720 * 16 * 3 * 2.0 ** -23      # linear: roundings of 720 numbers below 16 times w alone


def test_refusals(built_lib):
    table, ids = _table(10, 4), torch.zeros(3, dtype=torch.int64, device="cuda")
    for bad, error in (((table.cpu(), ids), RuntimeError), ((table, ids.cpu()), RuntimeError), ((table.half(), ids), TypeError), ((table, ids.float()), TypeError), ((table, ids.bool()), TypeError),
                       ((table[0], ids), ValueError), ((table[:0], ids), ValueError), ((table, ids, 1.0, 10), ValueError), ((table, ids, 1.0, -11), ValueError), ((table, ids, 1.0, 1.5), TypeError)):
        with pytest.raises(error):
            embedding_lookup(*bad)
    leaf = table.detach().requires_grad_(True)
    g = torch.ones(3, 4, device="cuda", requires_grad=True)
    (d,) = torch.autograd.grad(embedding_lookup(leaf, ids), leaf, g, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(d.sum(), g)


def test_captured(built_lib):
    table = _table(1000, 64)
    ids = torch.randint(0, 1000, (3000,), generator=_gen(12), device="cuda")
    g = torch.randn(3000, 64, generator=_gen(13), device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        leaf = table.detach().requires_grad_(True)
        torch.autograd.grad(embedding_lookup(leaf, ids), leaf, g)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            (d,) = torch.autograd.grad(embedding_lookup(leaf, ids, 2.0), leaf, g)
    torch.cuda.current_stream().wait_stream(side)
    for seed in (14, 15):
        ids.copy_(torch.randint(0, 1000, (3000,), generator=_gen(seed), device="cuda") % (10 if seed == 15 else 1000))
        graph.replay()
        own = table.detach().requires_grad_(True)
        assert torch.equal(d, torch.autograd.grad(embedding_lookup(own, ids, 2.0), own, g)[0])
