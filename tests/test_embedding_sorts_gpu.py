"""The embedding's gradient behind the sort by many CTAs (more than 4096 tokens): its passes, its tiles, and what is no token.

A sum of n numbers in f32 goes by blocks of at most 32, then four ways: within (32 + n / 128 + 10) 2^-24 of the sum of magnitudes, or (n - 1) 2^-24 of it where that is less;
the product with scale and the rounding to the table's type half a step each."""
import pytest
import torch

from pratchya_b200._nnx_impl import embedding_lookup

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
TILE = 2048


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _check(vocab, channels, dtype, ids, scale=1.0, padding=None):
    table = torch.randn(vocab, channels, generator=_gen(vocab), device="cuda").to(dtype).requires_grad_(True)
    rows = embedding_lookup(table, ids, scale, padding)
    g = torch.randn(rows.shape, generator=_gen(1), device="cuda").to(dtype)
    (d,) = torch.autograd.grad(rows, table, g, retain_graph=True)
    row = torch.where(ids < 0, ids + vocab, ids)
    use = (row >= 0) & (row < vocab) & (row != (-1 if padding is None else padding % vocab))
    at, gg = row[use], g[use].double()
    zeros = torch.zeros(table.shape, dtype=torch.float64, device="cuda")
    exact, size = zeros.index_add(0, at, gg) * scale, zeros.index_add(0, at, gg.abs()) * abs(scale)
    n = torch.bincount(at, minlength=vocab).double().unsqueeze(-1)
    bound = torch.minimum(n, 42 + n / 128) * 2.0 ** -24 * size + (2.0 ** -23 + torch.finfo(dtype).eps / 2) * exact.abs() + 2.0 ** -126 * (size > 0)
    off = (d.double() - exact).abs()
    assert d.dtype == dtype and (off <= bound).all(), (off / bound.clamp(min=1e-300)).max().item()
    assert not d[(n == 0).squeeze(-1)].any()
    assert torch.equal(torch.autograd.grad(rows, table, g)[0], d)
    return d


@pytest.mark.parametrize("n", [320 * TILE - 1, 320 * TILE, 320 * TILE + 1, 512 * TILE, 512 * TILE + 1, 520 * TILE + 77])
def test_counts_of_many_tiles(built_lib, n):
    """Around the number of tiles from which their counts are added up ahead of the pass, and around a chunk of them; one pass to three."""
    for vocab, channels in ((1, 1), (300, 8), (511, 3), (70000, 4), (300000, 2)):
        ids = torch.randint(-vocab, vocab, (n,), generator=_gen(n + vocab), device="cuda")
        _check(vocab, channels, F32, ids)
        odd = torch.where(torch.rand(n, generator=_gen(2), device="cuda") < 0.2, vocab + 3, ids)
        _check(vocab, channels, BF16, odd, 0.5, vocab // 2)


def test_workspace_of_many_tiles(built_lib):
    """The sums of the tiles' counts lie in it where they are used."""
    few, many = (built_lib.pb_embedding_lookup_bwd_workspace_size(n, 1000, 1) for n in (320 * TILE, 320 * TILE + 1))
    assert many >= few + 3 * 2048


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [4097, 9001])
@pytest.mark.parametrize("vocab,channels", [(1, 1), (2, 3), (300, 5), (300, 72), (511, 128), (512, 129), (513, 1001), (262143, 4), (262144, 3), (300000, 5), (300000, 8)])
def test_any_table(built_lib, vocab, channels, n, dtype):
    """One pass to three, rows in vectors and not, zeros beside the first pass, in tables of no whole tile of them."""
    ids = torch.randint(-vocab, vocab, (n,), generator=_gen(n + vocab), device="cuda")
    _check(vocab, channels, dtype, ids, 45.25)
    _check(vocab, channels, dtype, torch.sort(ids).values)
    _check(vocab, channels, dtype, torch.full((n,), vocab - 1, device="cuda"))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [4097, 9001])
@pytest.mark.parametrize("vocab,channels", [(1, 3), (300, 72), (700, 5), (65536, 9), (300000, 4)])
def test_padding_and_ids_outside(built_lib, vocab, channels, n, dtype):
    """What is padding or beyond the table sorts behind every token, by the same passes, and has no part in any row."""
    ids = torch.randint(-vocab, vocab, (n,), generator=_gen(n + vocab), device="cuda")
    chance = torch.rand(n, generator=_gen(3), device="cuda")
    for padding in sorted({0, vocab // 2, vocab - 1, -1, -vocab}):
        d = _check(vocab, channels, dtype, torch.where(chance < 0.4, padding, ids), 2.0, padding)
        assert not d[padding].any()
    for far in (vocab, -vocab - 1, 1 << 40, -(1 << 62)):
        _check(vocab, channels, dtype, torch.where(chance < 0.5, far, ids), 1.0, 0)
    assert not _check(vocab, channels, dtype, torch.full((n,), vocab, device="cuda")).any()                # no token at all
    assert not _check(vocab, channels, dtype, torch.full((n,), vocab - 1, device="cuda"), 1.0, -1).any()


@pytest.mark.parametrize("n", [4097, 9001, 320 * TILE + 5])
def test_captured(built_lib, n):
    """Replays with other tokens: nothing of a pass, its counts or its bitmap among them, is left for the next one."""
    table, g = torch.randn(1000, 8, generator=_gen(1), device="cuda"), torch.randn(n, 8, generator=_gen(2), device="cuda")
    ids = torch.randint(-1000, 1000, (n,), generator=_gen(3), device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        leaf, graph = table.detach().requires_grad_(True), torch.cuda.CUDAGraph()
        torch.autograd.grad(embedding_lookup(leaf, ids), leaf, g)
        with torch.cuda.graph(graph, stream=side):
            rows = embedding_lookup(leaf, ids, 2.0, 7)
            (d,) = torch.autograd.grad(rows, leaf, g)
    torch.cuda.current_stream().wait_stream(side)
    for most in (1000, 10, 1, 1003):
        ids.copy_(torch.randint(0, most, (n,), generator=_gen(most), device="cuda"))
        graph.replay()
        own = table.detach().requires_grad_(True)
        want = embedding_lookup(own, ids, 2.0, 7)
        assert torch.equal(rows.nan_to_num(7.5), want.nan_to_num(7.5)) and torch.equal(d, torch.autograd.grad(want, own, g)[0])
