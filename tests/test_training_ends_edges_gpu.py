"""Edges of the operators at the ends of a training step, as the model and its optimizer meet them."""
import pytest
import torch

from pratchya_b200._nnx_impl import generate, orthogonalize
from pratchya_b200._nnx_impl._model import PratchyaCausalLM, PratchyaConfig

pytestmark = pytest.mark.gpu


def _model(vocab=640):
    return PratchyaCausalLM(PratchyaConfig(vocab_size=vocab, hidden_size=256, intermediate_size=512, lora_rank=128, n_layers=2), seed=3)


def _ids(most, seed=0, shape=(3, 40)):
    return torch.randint(0, most, shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


@pytest.mark.parametrize("kind", [torch.uint8, torch.int8, torch.int16, torch.int32, torch.uint16])
@pytest.mark.parametrize("vocab", [128, 640])
def test_labels_of_any_whole_type(built_lib, vocab, kind):
    """The last position of a sequence has no target, whether or not the labels' type has a -1 to say so: the bits of int64 labels."""
    ids, got = _ids(128), []
    for label in (ids, ids.to(kind)):
        model = _model(vocab)
        loss = model.loss_without_logits(ids, label)
        loss.backward()
        got.append([loss.detach(), model.lm_head.kernel.grad, model.embedding.grad])
    assert torch.isfinite(got[0][0]) and all(torch.equal(a, b) for a, b in zip(*got))


def test_labels_that_are_no_whole_numbers(built_lib):
    ids = _ids(128)
    for label in (ids.float(), ids.bool(), ids.to(torch.complex64)):
        with pytest.raises(TypeError):
            _model().loss_without_logits(ids, label)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(3, 40, 50), (2048, 64), (200, 300), (2, 700, 260)])
def test_zeros_stay_zeros_under_any_eps(built_lib, shape, dtype):
    """0 / (0 + eps), beside a matrix that is not zero in a stack; down to the least double."""
    for eps in (5e-324, 1e-310, 1e-100, 1e-74, 1e-60, 1e-7, 1e300):
        g = torch.zeros(shape, dtype=dtype, device="cuda")
        assert torch.equal(orthogonalize(g, eps=eps), torch.zeros(shape, dtype=torch.bfloat16, device="cuda")), eps
        if len(shape) == 3 and eps < 1e-7:
            g[0] = torch.randn(shape[1:], generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(dtype)
            got = orthogonalize(g, eps=eps)
            assert torch.equal(got[0], orthogonalize(g, eps=0.0)[0]) and not got[1:].any(), eps      # the norm is 40 and more: no eps of these moves a bit of it


def _polynomial(g, eps, steps=5):
    x = g.double()
    x = x / (x.norm(dim=(-2, -1), keepdim=True) + eps)
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    for _ in range(steps):
        p = x @ x.mT
        x = 3.4445 * x + (-4.7750 * p + 2.0315 * p @ p) @ x
    return x.mT if tall else x


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(200, 300), (700, 260), (2, 131, 2000), (129, 6000)])
def test_updates_of_any_scale_by_products(built_lib, shape, dtype):
    """As test_orthogonalize_gpu.py has it for one launch, with the errors that it derives: squares beyond f32 on either side, an eps beside the norm and one of 10^4 of it.

    X's numbers have two fp16 terms of 2^12 of them, within 2^-25 where both are subnormal: 2^-37, of m n of them 2^-37 sqrt(m n), which of X's norm 10^-4 is 6e-5 at most here."""
    for scale in (1e-42, 1e-30, 1e-12, 1.0, 1e15, 1e30, 1e36):
        g = (torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(9), device="cuda", dtype=torch.float64) * scale).to(dtype)
        norm = g.double().norm(dim=(-2, -1)).max().item()
        for eps in (0.0, norm, 1e4 * norm):
            got, want = orthogonalize(g, eps=eps), _polynomial(g, eps)
            if norm == 0.0:                                        # 1e-42 in bf16, by an eps of zero
                assert got.isnan().all() and want.isnan().all()
                continue
            assert ((got.double() - want).norm(dim=(-2, -1)) <= 5e-3 * want.norm(dim=(-2, -1))).all(), (scale, eps)


def test_a_token_beyond_the_vocabulary(built_lib):
    """Its sequence's logits are NaN, with the loss, and those of the others are not: nothing in between takes the NaN for a number."""
    model, ids = _model(), _ids(640)
    wrong = ids.clone()
    wrong[1, 17] = 640
    with torch.no_grad():
        logits, loss = model(wrong, ids)
        assert logits[1].isnan().all() and loss.isnan() and model.loss_without_logits(wrong, ids).isnan()
        assert not logits[0].isnan().any() and not logits[2].isnan().any()
        assert generate(model, wrong, 2).logprobs[1].isnan().all()


def test_more_matrices_than_a_call_of_the_library_takes(built_lib):
    g = torch.randn(65535 + 70, 3, 2, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda")
    for update in (g, g.bfloat16(), g.mT):
        got = orthogonalize(update)
        assert torch.equal(got[-100:], orthogonalize(update[-100:])) and torch.equal(got[:100], orthogonalize(update[:100]))
        want = _polynomial(update, 1e-7)
        # few numbers may all be rounded the worst way: test_orthogonalize_gpu.py derives it
        assert ((got.double() - want).norm(dim=(1, 2)) <= (7.6 * 2.0 ** -11 * 5.2 + 2.0 ** -8) * want.norm(dim=(1, 2))).all()


@pytest.mark.parametrize("shape", [(200, 64), (1500, 128), (2, 4096, 100), (200, 6000), (2, 300, 260)])
def test_updates_captured(built_lib, shape):
    """One CTA, clusters of eight and of sixteen, products cut and not."""
    g = torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda")
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            out = orthogonalize(g)
    torch.cuda.current_stream().wait_stream(side)
    for k in range(3):
        g.copy_(torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(6 + k), device="cuda"))
        graph.replay()
        assert torch.equal(out, orthogonalize(g))
