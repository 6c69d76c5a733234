"""A model that answers: Linears in 4 bits in every layer, a state carried from call to call, tokens with their scores."""
import copy
import math
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from pratchya_b200._nnx_impl import Int4Linear, generate, score, token_logprobs
from pratchya_b200._nnx_impl._model import Linear, PratchyaCausalLM, PratchyaConfig

pytestmark = pytest.mark.gpu

SMALL = dict(vocab_size=640, hidden_size=256, intermediate_size=512, lora_rank=128, n_layers=2)


class _Dense(torch.nn.Module):
    """The product with the values that an Int4Linear stands for, as plain torch computes it."""
    def __init__(self, layer):
        super().__init__()
        self.w = layer.weight()

    def forward(self, x, raw=False):
        return torch.matmul(x, self.w)


def _plain(model):
    """The same model without this package's products and fused kernels (but for the scan)."""
    plain = PratchyaCausalLM(PratchyaConfig(**{**SMALL, "fused_glue": False}), seed=1)
    plain.load_state_dict(model.state_dict())
    plain.to_int4(64, True)
    for module in list(plain.modules()):
        for name, child in list(module.named_children()):
            if isinstance(child, Int4Linear):
                setattr(module, name, _Dense(child))
    return plain


def _model():
    torch.manual_seed(0)
    model = PratchyaCausalLM(PratchyaConfig(**SMALL), seed=1)
    plain = _plain(model)
    return model.to_int4(64, True), plain


def test_every_linear_is_taken(built_lib):
    model, _ = _model()
    assert not any(isinstance(m, Linear) for m in model.modules())
    assert sum(isinstance(m, Int4Linear) for m in model.modules()) == 2 * (4 + 2 * 4 + 2) - 2 + 1          # the first layer has no nu_lora
    assert not any(name.endswith("kernel") for name, _ in model.named_parameters())


def test_a_prompt_and_single_tokens_against_the_plain_model(built_lib):
    """The two differ by f32 rounding alone.  Behind two layers of some thirty operations each, at 2^-24 apiece and grown by norms of a random model by
    ten or so, 1e-4 of the logits' size leaves room for two orders of magnitude."""
    model, plain = _model()
    ids = torch.randint(0, 640, (3, 9), device="cuda")
    states = [None, None]
    for part in (ids[:, :6], ids[:, 6:7], ids[:, 7:8], ids[:, 8:]):
        got, states[0] = model.advance(part, states[0])
        want, states[1] = plain.advance(part, states[1])
        assert got.shape == (3, part.shape[1], 640)
        assert float((got - want).norm() / want.norm()) <= 1e-4
    assert states[0][0] == 9
    for (a, b) in zip(states[0][1], states[1][1]):
        for x, y in zip(a, b):
            assert float((x - y).norm()) <= 1e-4 * float(y.norm())


def test_a_state_of_zeros_is_the_beginning(built_lib):
    model, _ = _model()
    ids = torch.randint(0, 640, (2, 5), device="cuda")
    with torch.no_grad():
        assert torch.equal(model.advance(ids)[0], model.advance(ids, model.init_state(2))[0]) and torch.equal(model.advance(ids)[0], model(ids)[0])


def test_generate_takes_the_best_or_by_the_numbers_given(built_lib):
    model, _ = _model()
    prompt = torch.randint(0, 640, (2, 4), device="cuda")
    answer = generate(model, prompt, 5, top=3)
    assert answer.tokens.shape == (2, 5) and answer.top_tokens.shape == (2, 5, 3) and torch.equal(answer.tokens, answer.top_tokens[..., 0])
    state, ids = None, prompt
    for i in range(5):          # the same by hand
        logits, state = model.advance(ids, state)
        logp = torch.log_softmax(logits[:, -1].double(), -1)
        ids = logits[:, -1].argmax(-1, keepdim=True)
        assert torch.equal(answer.tokens[:, i], ids[:, 0])
        assert (answer.logprobs[:, i].double() - logp.gather(1, ids)[:, 0]).abs().max() <= 1e-5
        assert (answer.entropy[:, i].double() + (logp.exp() * logp).sum(-1)).abs().max() <= 1e-5
    u = torch.tensor([[0.0, 0.999999], [0.4, 0.6]], device="cuda")
    sampled = generate(model, prompt, 2, top=4, uniform=u)
    first = torch.softmax(answer.top_logprobs[:, 0].double(), -1)
    assert sampled.tokens[0, 0] == answer.tokens[0, 0] and sampled.tokens[0, 1] == sampled.top_tokens[0, 1, 3]
    assert all(t in row for t, row in zip(sampled.tokens[:, 1].tolist(), sampled.top_tokens[:, 1].tolist())) and first.shape == (2, 3)
    for bad in (dict(steps=0), dict(steps=1, top=0), dict(steps=3, uniform=u)):
        with pytest.raises(ValueError):
            generate(model, prompt, **bad)


def test_score_trains_a_model_of_fp8_linears(built_lib):
    """A policy's loss through the whole model: the gradient of its lm_head is what the log probabilities' own gradient gives."""
    model = PratchyaCausalLM(PratchyaConfig(**SMALL), seed=1, remat=False)
    ids = torch.randint(0, 640, (2, 8), device="cuda")
    out = score(model, ids, top=2)
    assert out.logprobs.shape == (2, 7) and out.top_tokens.shape == (2, 7, 2)
    loss = -out.logprobs.mean() - 0.01 * out.entropy.mean()
    loss.backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in (model.lm_head.kernel, model.embedding, model.blocks[0].tm.w_key.kernel))
    again = copy.deepcopy(model)
    again.zero_grad()
    logits, _ = again(ids)
    logp = torch.log_softmax(logits[:, :-1], -1)
    plain = -logp.gather(-1, ids[:, 1:, None]).mean() + 0.01 * (logp.exp() * logp).sum(-1).mean()
    plain.backward()
    # the cotangents of the logits agree to 2^-20 or so; an fp8 step here and there behind them is what the Linear's backward pass makes of that
    a, b = model.lm_head.kernel.grad, again.lm_head.kernel.grad
    assert float((a - b).norm() / b.norm()) <= 1e-2


def test_a_model_in_4_bits_refuses_gradients(built_lib):
    model, _ = _model()
    with pytest.raises(RuntimeError, match="backward"):
        model(torch.randint(0, 640, (1, 4), device="cuda"))


def test_token_logprobs_of_one_step(built_lib):
    model, _ = _model()
    logits, _ = model.advance(torch.randint(0, 640, (1, 3), device="cuda"))
    one = token_logprobs(logits[0, -1], top=640 if 640 <= 128 else 128)
    assert one.entropy.shape == () and one.top_tokens.shape == (128,)


def test_the_example_runs(built_lib):
    root = Path(__file__).resolve().parent.parent
    r = subprocess.run([sys.executable, str(root / "examples" / "answer.py"), "--layers", "1", "--vocab", "1024", "--tokens", "3", "--batch", "2"], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    assert "log probability of the whole text" in r.stdout


def test_casts_leave_the_weights_parts_as_they_are(built_lib):
    """Module.float(), .half() and the like are about parameters; a scale in another type would be no weight of 4 bits."""
    model, _ = _model()
    ids = torch.randint(0, 640, (1, 5), device="cuda")
    want, _ = model.advance(ids)
    assert torch.equal(model.float().advance(ids)[0], want)
    layer = Int4Linear(torch.randn(300, 70, device="cuda"), 64, True)
    x = torch.randn(2, 300, device="cuda")
    parts, y = [t.clone() for t in (layer.q, layer.scale, layer.zero)], layer(x)
    for cast in (lambda m: m.half(), lambda m: m.double(), lambda m: m.float(), lambda m: m.bfloat16(), lambda m: m.to(torch.float16), lambda m: m.type(torch.float32), lambda m: m.to("cuda:0", torch.float32)):
        layer = cast(layer)
        assert all(a.dtype is b.dtype and torch.equal(a, b) for a, b in zip((layer.q, layer.scale, layer.zero), parts)) and torch.equal(layer(x), y)
    moved = copy.deepcopy(layer).cpu().half()
    assert moved.scale.device.type == "cpu" and moved.scale.dtype is torch.bfloat16 and torch.equal(moved.cuda()(x), y)
    assert layer.half().state_dict()["scale"].dtype is torch.bfloat16 and Int4Linear(torch.randn(128, 16, device="cuda")).float().zero is None


class _Fixed:
    """A model whose next-token logits [B, V] are given, the same at every step."""
    def __init__(self, logits):
        self.logits = logits

    def advance(self, ids, state=None, **_):
        return self.logits.unsqueeze(1), state


def test_the_number_given_decides_among_the_alternatives(built_lib):
    """The expected pick in 64 bits from the alternatives' own log probabilities, for numbers a thousandth away from where it changes."""
    g = torch.Generator(device="cuda").manual_seed(3)
    logits = torch.randn(2000, 50, generator=g, device="cuda") * 2
    u = torch.rand(2000, 2, generator=g, device="cuda")
    answer = generate(_Fixed(logits), torch.zeros(2000, 1, dtype=torch.int64, device="cuda"), 2, top=7, uniform=u)
    ends = torch.softmax(answer.top_logprobs.double(), -1).cumsum(-1)
    clear = ((ends - u.double().unsqueeze(-1)).abs() > 1e-3).all(-1)
    pick = (ends <= u.double().unsqueeze(-1)).sum(-1, keepdim=True)
    assert clear.float().mean() > 0.9 and set(pick[clear].flatten().tolist()) == set(range(7))
    assert torch.equal(answer.tokens[clear], answer.top_tokens.gather(-1, pick.clamp(max=6))[..., 0][clear])
    assert torch.equal(answer.logprobs[clear], answer.top_logprobs.gather(-1, pick.clamp(max=6))[..., 0][clear])


def test_what_is_ruled_out_is_never_taken(built_lib):
    """Shares that add up to less than the largest number below 1: the last alternative is one that can be taken, not one of those that fill up behind it."""
    g = torch.Generator(device="cuda").manual_seed(4)
    logits = torch.full((4096, 40), -math.inf, device="cuda")
    logits[:, 3:20] = torch.randn(4096, 17, generator=g, device="cuda")
    u = torch.full((4096, 1), 1.0 - 2.0 ** -24, device="cuda")
    answer = generate(_Fixed(logits), torch.zeros(4096, 1, dtype=torch.int64, device="cuda"), 1, top=30, uniform=u)
    shares = torch.softmax(answer.top_logprobs[:, 0], -1).cumsum(-1)[:, -1]
    assert (shares <= u[:, 0]).any() and torch.isfinite(answer.logprobs).all() and (answer.tokens >= 3).all() and (answer.tokens < 20).all()
    nothing = generate(_Fixed(torch.full((2, 40), -math.inf, device="cuda")), torch.zeros(2, 1, dtype=torch.int64, device="cuda"), 1, top=5, uniform=u[:2])
    assert nothing.tokens.tolist() == [[0], [0]] and (nothing.logprobs == -math.inf).all()


def test_a_prompt_takes_the_memory_of_one_positions_logits(built_lib):
    """4096 tokens of a vocabulary of 65536: 1 GB of logits, of which the next token needs a row."""
    model = PratchyaCausalLM(PratchyaConfig(**{**SMALL, "vocab_size": 65536, "n_layers": 1}), seed=1).to_int4()
    prompt = torch.randint(0, 65536, (1, 4096), device="cuda")
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    generate(model, prompt, 2, top=3)
    assert torch.cuda.max_memory_allocated() - before < 1 << 28


@pytest.mark.parametrize("hidden,steps", [(256, 9), (1024, 5), (1024, 1)])
def test_the_last_positions_logits_are_those_of_all(built_lib, hidden, steps):
    """In fp8 to the bit, also where the rows of lm_head's input share scales; in 4 bits the sums may be taken in another order, 2^-24 of their size at each of some thirty steps."""
    model = PratchyaCausalLM(PratchyaConfig(**{**SMALL, "hidden_size": hidden}), seed=2)
    ids = torch.randint(0, 640, (3, steps), device="cuda")
    for bits in (8, 4):
        whole, state = model.advance(ids)
        last, behind = model.advance(ids, last=True)
        assert last.shape == (3, 1, 640) and behind[0] == steps and all(torch.equal(a, b) for x, y in zip(state[1], behind[1]) for a, b in zip(x, y))
        if bits == 8:
            assert torch.equal(last, whole[:, -1:])
        else:
            assert float((last - whole[:, -1:]).norm() / last.norm()) <= 1e-6
        model.to_int4(64, True)


def test_advance_refuses_what_it_cannot_go_on_from(built_lib):
    model, _ = _model()
    ids = torch.randint(0, 640, (2, 3), device="cuda")
    position, layers = model.advance(ids)[1]
    for bad, state in ((ids[:, :0], None), (ids[0], None), (ids, (position, layers[:1])), (ids, (position, layers + layers[:1])), (ids[:1], (position, layers))):
        with pytest.raises(ValueError):
            model.advance(bad, state)
