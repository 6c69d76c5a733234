"""The operators at the ends of a training step together, as the model and the optimizer call them: embedding, loss without logits, gradients, momentum,
orthogonalised update; and what their bounded waits do when they run out."""
import ctypes as C

import pytest
import torch
from torch.autograd import forward_ad
from torch.utils._python_dispatch import TorchDispatchMode

from pratchya_b200 import _lib
from pratchya_b200._nnx_impl import embedding_lookup, linear_cross_entropy, momentum_update_stacked, muon_update, orthogonalize
from pratchya_b200._nnx_impl._model import PratchyaCausalLM, PratchyaConfig, read_param
from pratchya_b200._qualia import QArrayImpl

pytestmark = pytest.mark.gpu

SMALL = dict(vocab_size=640, hidden_size=256, intermediate_size=512, lora_rank=128, n_layers=2)


def _model():
    return PratchyaCausalLM(PratchyaConfig(**SMALL), seed=3, remat=1)


def _ids(seed=0, shape=(3, 40)):
    return torch.randint(0, 640, shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def test_the_loss_without_logits_against_the_logits(built_lib):
    """The same bf16 operands through a plain product in 64 bits: the loss within f32 sums, lm_head's gradient within the roundings of its operand to bf16, of its result, and of that
    of the cast's cotangent (all half a step or less: 2^-8 each)."""
    model, ids = _model(), _ids()
    loss = model.loss_without_logits(ids, ids, alpha=0.1)
    loss.backward()
    with torch.no_grad():
        x, w = model.hidden(ids).to(torch.bfloat16).double()[:, :-1], model.lm_head.kernel.to(torch.bfloat16).double()
    w.requires_grad_(True)
    logp = torch.log_softmax(x @ w, -1)
    want = -(0.9 * logp.gather(-1, ids[:, 1:, None])[..., 0] + 0.1 * logp.mean(-1)).mean()
    (dw,) = torch.autograd.grad(want, w)
    assert (loss.double() - want).abs() <= 1e-5 * want.abs()
    assert (model.lm_head.kernel.grad.double() - dw).norm() <= 3 * 2.0 ** -8 * dw.norm()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for n, p in model.named_parameters() if "nu_lora" not in n or ".0." not in n)
    # forward's own loss has fp8 operands: 2^-4 a value at most, and of the loss less
    assert (model(ids, ids)[1] - loss).abs() <= 2.0 ** -4 * loss


def test_the_embeddings_gradient_against_indexing(built_lib):
    """Everything but the order of a token's sum is the same in both, to the bit."""
    model, ids = _model(), _ids(1) % 50
    model(ids, ids)[1].backward()
    got = model.embedding.grad.clone()
    model.zero_grad()
    model.embed = lambda i: read_param(model.embedding[i], (1, model.cfg.blksize)) * model.cfg.hidden_size ** 0.5
    model(ids, ids)[1].backward()
    want = model.embedding.grad
    assert (got - want).norm() <= 1e-6 * want.norm() and not got[50:].any()


def test_a_step_of_training(built_lib):
    """Gradients, a quantized momentum, orthogonalised updates of every layer's key weights at once, and the next loss."""
    model, ids = _model(), _ids(2)
    weights = [b.tm.w_key.kernel for b in model.blocks]
    m = QArrayImpl(torch.zeros(2, 256, 256, device="cuda"), (128, 128))
    for _ in range(2):
        model.zero_grad()
        model.loss_without_logits(ids, ids).backward()
        g = QArrayImpl(torch.stack([w.grad for w in weights]), (128, 128))
        c, m = momentum_update_stacked(g, m, 0.9, 0.99)
        update = muon_update(c, torch.stack([w.detach() for w in weights]), lr=0.02, weight_decay=0.1)
        assert update.dtype == torch.float32 and torch.isfinite(update).all()
        plain = orthogonalize(c)
        values = torch.linalg.svdvals(plain.float())
        assert values.max() <= 1.3                       # what five steps make of [0, 1] is at most 1.21, within the errors of the products
        with torch.no_grad():
            for w, u in zip(weights, update):
                before = w.clone()
                w += u
                assert not torch.equal(w, before)
    assert torch.isfinite(model.loss_without_logits(ids, ids))


def test_refusals(built_lib):
    model, ids = _model(), _ids(3)
    with pytest.raises(ValueError):
        model.loss_without_logits(ids[:, :1], ids[:, :1])
    with pytest.raises(ValueError):
        model.loss_without_logits(ids, ids[:, :-1])
    with pytest.raises(TypeError):
        model.to_int4().loss_without_logits(ids, ids)


@pytest.mark.parametrize("rows,depth,vocab", [(100, 512, 700), (600, 512, 700), (600, 64, 300)])
def test_waits_that_run_out_are_reported_cross_entropy(built_lib, diag_lib, rows, depth, vocab):
    """The diagnostics build leaves the first stage of each launch unfilled, with a poll budget of about two milliseconds a wait."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    x, w = torch.randn(rows, depth, generator=g, device="cuda").bfloat16(), torch.randn(depth, vocab, generator=g, device="cuda").bfloat16()
    t, st = torch.randint(0, vocab, (rows,), generator=g, device="cuda"), torch.cuda.current_stream().cuda_stream
    size = diag_lib.pb_linear_xent_workspace_size(rows, depth, w.data_ptr(), vocab, 0, vocab, 1) + diag_lib.pb_linear_xent_workspace_size(rows, depth, w.data_ptr(), vocab, 0, vocab, 0)
    ws = torch.zeros(size, dtype=torch.uint8, device="cuda")

    def run():
        loss, lse, dx, dw = torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda"), torch.zeros_like(x), torch.zeros_like(w)
        at = (x.data_ptr(), 1, rows, 0, depth, depth, w.data_ptr(), vocab, 0, vocab, t.data_ptr(), 0.0)
        assert diag_lib.pb_linear_xent(*at, loss.data_ptr(), lse.data_ptr(), ws.data_ptr(), size, st) == 0
        assert diag_lib.pb_linear_xent_bwd(*at, lse.data_ptr(), torch.ones_like(loss).data_ptr(), dx.data_ptr(), dw.data_ptr(), ws.data_ptr(), size, st) == 0
        torch.cuda.synchronize()
        return loss, dx, dw

    before = run()
    assert diag_lib.pb_gemm_check(st) == 0
    try:
        assert diag_lib.pb_debug_product_control(1 << 10, 1) == 0
        run()
        assert diag_lib.pb_gemm_check(st) == 7 and b"cross entropy" in diag_lib.pb_last_error()
        assert diag_lib.pb_gemm_check(st) == 0
    finally:
        diag_lib.pb_debug_product_control(0, 0)
    after = run()
    assert diag_lib.pb_gemm_check(st) == 0 and all(torch.equal(a, b) for a, b in zip(before, after))
    assert built_lib.pb_gemm_check(st) == 0


@pytest.mark.parametrize("rows,cols", [(300, 520), (1400, 1300), (200, 6000)])
def test_waits_that_run_out_are_reported_update(built_lib, diag_lib, rows, cols):
    g = torch.randn(rows, cols, generator=torch.Generator(device="cuda").manual_seed(rows), device="cuda")
    st, numbers = torch.cuda.current_stream().cuda_stream, (C.c_float * 6)(*((3.4445, -4.7750, 2.0315) * 2))
    size = diag_lib.pb_orthogonalize_workspace_size(1, rows, cols)
    ws = torch.zeros(size, dtype=torch.uint8, device="cuda")

    def run():
        out = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
        assert diag_lib.pb_orthogonalize(g.data_ptr(), 0, 1, rows, cols, 2, C.addressof(numbers), 1e-7, out.data_ptr(), ws.data_ptr(), size, st) == 0
        torch.cuda.synchronize()
        return out

    before = run()
    assert diag_lib.pb_gemm_check(st) == 0
    try:
        assert diag_lib.pb_debug_product_control(1 << 10, 1) == 0
        run()
        assert diag_lib.pb_gemm_check(st) == 7 and b"orthogonalised" in diag_lib.pb_last_error()
        assert diag_lib.pb_gemm_check(st) == 0
    finally:
        diag_lib.pb_debug_product_control(0, 0)
    assert torch.equal(before, run()) and diag_lib.pb_gemm_check(st) == 0


def test_two_calls_at_once(built_lib):
    """On two streams, with workspaces of their own."""
    g = torch.Generator(device="cuda").manual_seed(5)
    x = [torch.randn(700, 128, generator=g, device="cuda").bfloat16() for _ in range(2)]
    w = torch.randn(128, 3000, generator=g, device="cuda").bfloat16()
    t = torch.randint(0, 3000, (700,), generator=g, device="cuda")
    u = [torch.randn(400, 900, generator=g, device="cuda") for _ in range(2)]
    want = [(linear_cross_entropy(a, w, t), orthogonalize(b)) for a, b in zip(x, u)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append((linear_cross_entropy(x[i], w, t), orthogonalize(u[i])))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, want[i][0]) and torch.equal(b, want[i][1]) for a, b in got[i])


def test_no_derivative_is_dropped_without_a_word(built_lib):
    """Forward-mode differentiation, function transforms and traces are refused by each; a dispatch mode that watches changes nothing."""
    g = torch.Generator(device="cuda").manual_seed(6)
    table, ids = torch.randn(50, 64, generator=g, device="cuda"), torch.randint(0, 50, (7,), generator=g, device="cuda")
    x, w, t = torch.randn(7, 64, generator=g, device="cuda").bfloat16(), torch.randn(64, 30, generator=g, device="cuda").bfloat16(), torch.randint(0, 30, (7,), generator=g, device="cuda")
    calls = [lambda v: embedding_lookup(v, ids), lambda v: linear_cross_entropy(v, w, t), lambda v: linear_cross_entropy(x, v, t), lambda v: orthogonalize(v)]
    inputs = [table, x, w, table]
    for call, v in zip(calls, inputs):
        with forward_ad.dual_level(), pytest.raises(RuntimeError):
            call(forward_ad.make_dual(v, torch.ones_like(v)))
        with pytest.raises(RuntimeError):
            torch.func.jvp(call, (v,), (torch.ones_like(v),))
        with torch.no_grad(), pytest.raises(RuntimeError):
            torch.func.vmap(call)(torch.stack([v, v]))
        with pytest.raises(RuntimeError):
            torch.jit.trace(call, (v,), check_trace=False)

    class Watching(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    for call, v in zip(calls, inputs):
        want = call(v)
        with Watching():
            assert torch.equal(call(v), want)
        if call is calls[3]:
            continue
        leaf = v.detach().requires_grad_(True)
        (d,) = torch.autograd.grad(call(leaf).float().sum(), leaf)
        with Watching():
            (again,) = torch.autograd.grad(call(leaf).float().sum(), leaf)
        assert torch.equal(d, again)


def test_coefficients_of_another_number_than_three(built_lib):
    g = torch.randn(40, 300, device="cuda")
    a, b, c = 3.4445, -4.7750, 2.0315
    want = orthogonalize(g, steps=2)
    assert torch.equal(orthogonalize(g, steps=2, coefficients=[a, b, c]), want) and torch.equal(orthogonalize(g, steps=2, coefficients=((a, b, c), [a, b, c])), want)
    for wrong in ((), (a, b), (a, b, c, a), ((a, b), (c, a, b, c)), ((a, b, c),), ((a, b, c), a, b), ((a, b, c), (a, b, c), (a, b, c))):
        with pytest.raises(ValueError):
            orthogonalize(g, steps=2, coefficients=wrong)
