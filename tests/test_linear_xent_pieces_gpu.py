"""Cross entropy without logits where a call has more of something than one launch or piece takes: rows of a weight that is copied first, pieces of a vocabulary with few positions.

Against the definition in 64 bits with the bounds that test_linear_xent_gpu.py derives."""
import pytest
import torch

from test_linear_xent_gpu import _check, _gen, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [65535, 65536, 65601])
def test_copied_weights_of_many_rows(built_lib, vocab):
    """A tied table of odd depth: its rows are copied 65535 a launch."""
    x, w, t, g = _inputs(40, 9, vocab, True)
    t[:3] = torch.tensor([vocab - 1, 65534, 0], device="cuda")
    loss, dx, dw = _check(x, w, t, 0.1, g)
    wide = torch.zeros(vocab, 16, dtype=torch.bfloat16, device="cuda")
    wide[:, :9] = w.t()
    same = _check(x, wide[:, :9].t(), t, 0.1, g)                   # read in place, rows of 16 bytes
    assert torch.equal(loss, same[0]) and torch.equal(dx, same[1]) and torch.equal(dw, same[2])


@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("smoothing", [0.0, 0.1])
def test_pieces_with_few_positions(built_lib, smoothing, tied):
    """Beyond 524288 words 256 rows of dz are more than is held at a time: one CTA's tiles, dx added up over two pieces."""
    x, w, t, g = _inputs(20, 8, 530003, tied, ignored=0.2)
    t[0], t[1], t[2] = 530002, 0, 300000
    _check(x, w, t, smoothing, g)


@pytest.mark.parametrize("smoothing", [0.1, 0.7])
@pytest.mark.parametrize("tied", [False, True])
def test_smoothed_pieces(built_lib, tied, smoothing):
    x, w, t, g = _inputs(16300, 64, 20001, tied, ignored=0.1)
    t[:2] = torch.tensor([20000, 8192], device="cuda")
    _check(x, w, t, smoothing, g)


def test_weights_that_end_with_their_memory(built_lib):
    """Many rows of a view at every offset from 16 bytes: the last row ends where the array does."""
    base = torch.randn(65540, 11, generator=_gen(5), device="cuda").bfloat16()
    for first in range(4):
        w = base[:, first:].t()
        x = torch.randn(5, 11 - first, generator=_gen(6), device="cuda").bfloat16()
        t = torch.randint(0, 65540, (5,), generator=_gen(7), device="cuda")
        t[0] = 65539
        _check(x, w, t, 0.0, torch.rand(5, generator=_gen(8), device="cuda"))
