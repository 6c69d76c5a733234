"""Edges of the operators at the ends of a training step, as the model and its optimizer meet them."""
import pytest
import torch

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
