"""The operators at the ends of a training step, as cases that can be timed: the lookup of token embeddings and its gradient, softmax cross
entropy of hidden states against a vocabulary's weight without keeping the logits and its gradients, and the orthogonalised update of a weight
by Newton-Schulz products.

A case is a dict of plain values.  `listed()` gives the listed ones, `draw(rng)` one more of the same ranges, `prepare` what a
program holds before the call, `run` one pass: the plain form in elementary torch operations, or, where `own` is set, the call of this
framework; `exact` what the definition gives in 64 bits, `work` the bytes and operations that a pass cannot do without."""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5


def listed():
    return [
        # one token of eight sequences that are being answered
        dict(name="embed_step", kind="embed", batch=8, steps=1, vocab=65536, channels=2048, scale=45.25, padded=0.0, dtype="f32", train=False),
        # a padded batch of prompts of no particular length, rows of no particular width
        dict(name="embed_prompt_odd", kind="embed", batch=3, steps=777, vocab=32003, channels=1001, scale=1.0, padded=0.3, dtype="bf16", train=False),
        # fine-tuning on a padded batch: the table's gradient is mostly rows that no token has
        dict(name="embed_tune_odd", kind="embed", batch=3, steps=341, vocab=32003, channels=1000, scale=31.6, padded=0.3, dtype="bf16", train=True),
        # a step of pretraining: 32768 tokens of text, lookup and gradient
        dict(name="embed_train", kind="embed", batch=8, steps=4096, vocab=65536, channels=2048, scale=45.25, padded=0.0, dtype="f32", train=True),
        # the loss of 64 answers' last tokens
        dict(name="xent_few", kind="xent", batch=64, steps=1, channels=2048, vocab=65536, smoothing=0.0, ignored=0.0, tied=False, sliced=False, train=False),
        # the loss of held-out texts with a table that is also the embedding
        dict(name="xent_eval_odd", kind="xent", batch=3, steps=1023, channels=1000, vocab=32003, smoothing=0.0, ignored=0.2, tied=True, sliced=True, train=False),
        # a step of pretraining
        dict(name="xent_train", kind="xent", batch=8, steps=1024, channels=2048, vocab=65536, smoothing=0.1, ignored=0.0, tied=False, sliced=True, train=True),
        # fine-tuning on answers only: the prompts' positions have no target
        dict(name="xent_tune_odd", kind="xent", batch=3, steps=777, channels=1000, vocab=32003, smoothing=0.0, ignored=0.5, tied=True, sliced=False, train=True),
        # the update of one low-rank layer's down-projection
        dict(name="ortho_lora", kind="ortho", layers=1, rows=2048, cols=128, rank=0.5, dtype="f32"),
        # stacked updates of no particular size
        dict(name="ortho_odd", kind="ortho", layers=3, rows=777, cols=1000, rank=1.0, dtype="bf16"),
        # the update of one projection
        dict(name="ortho_square", kind="ortho", layers=1, rows=2048, cols=2048, rank=1.0, dtype="f32"),
        # the updates of a stack of ChannelMix weights, few directions in each
        dict(name="ortho_stack", kind="ortho", layers=4, rows=2048, cols=8192, rank=0.25, dtype="bf16"),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["embed", "xent", "ortho"])
    if kind == "embed":
        train = rng.random() < 0.6
        channels = _log(rng, 64, 4096)
        if rng.random() < 0.6:
            channels -= channels % 8
        vocab = _log(rng, 1000, min(131072, (1 << 27) // channels))
        tokens = _log(rng, 1, min(32768, (1 << 26) // channels))
        batch = min(rng.choice([1, 2, 3, 8]), tokens)
        return dict(kind=kind, batch=batch, steps=tokens // batch, vocab=vocab, channels=channels, scale=rng.choice([1.0, round(math.sqrt(channels), 2)]),
                    padded=rng.choice([0.0, 0.0, 0.1, 0.5]), dtype=rng.choice(["f32", "bf16"]), train=train)
    if kind == "xent":
        channels = _log(rng, 64, 4096)
        if rng.random() < 0.6:
            channels = max(64, channels - channels % 64)
        vocab = _log(rng, 1000, min(131072, (1 << 27) // channels))
        if rng.random() < 0.6:
            vocab -= vocab % 8
        tokens = _log(rng, 1, min(8192, (1 << 40) // (vocab * channels), (1 << 29) // vocab))
        batch = min(rng.choice([1, 2, 3, 8]), tokens)
        return dict(kind=kind, batch=batch, steps=max(1, tokens // batch), channels=channels, vocab=vocab, smoothing=rng.choice([0.0, 0.0, 0.1]),
                    ignored=rng.choice([0.0, 0.0, 0.2, 0.6]), tied=rng.random() < 0.5, sliced=rng.random() < 0.5, train=rng.random() < 0.6)
    rows, cols = _log(rng, 16, 4096), _log(rng, 16, 8192)
    if rng.random() < 0.6:
        rows, cols = max(16, rows - rows % 16), max(16, cols - cols % 16)
    less, more = min(rows, cols), max(rows, cols)
    if less > 2048:
        rows, cols = (2048, cols) if rows == less else (rows, 2048)
        less = 2048
    layers = _log(rng, 1, max(1, min(24, (1 << 37) // (less * less * (less + more)), (1 << 25) // (rows * cols))))
    return dict(kind=kind, layers=layers, rows=rows, cols=cols, rank=rng.choice([1.0, 1.0, 0.5, 0.1]), dtype=rng.choice(["f32", "bf16"]))


# ---- inputs ----------------------------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 31)


def _words(shape, vocab, g):
    """Tokens as texts have them: the n-th most frequent one every 1 / n times; frequent ones lie anywhere in the vocabulary."""
    n = torch.exp(torch.rand(shape, generator=g, device=DEV, dtype=torch.float64) * math.log(vocab)).to(torch.int64).clamp(1, vocab) - 1
    return torch.randperm(vocab, generator=g, device=DEV)[n]


def prepare(case, seed):
    c, g = case, _gen(seed)
    s = {"case": c}
    if c["kind"] == "embed":
        lead = (c["batch"], c["steps"])
        s["table"] = (torch.randn(c["vocab"], c["channels"], generator=g, device=DEV) / math.sqrt(c["channels"])).to(DTYPES[c["dtype"]])
        ids = _words(lead, c["vocab"], g)
        s["padding"] = 0 if c["padded"] else None
        if c["padded"]:                 # sequences of different lengths, the rest of each row is padding
            ids = ids.clamp(min=1)
            lengths = torch.rand(c["batch"], 1, generator=g, device=DEV) * (2 * c["padded"])
            ids = torch.where(torch.arange(c["steps"], device=DEV) >= (1.0 - lengths) * c["steps"], 0, ids)
        s["ids"] = ids
        if c["train"]:
            s["g"] = (torch.randn(*lead, c["channels"], generator=g, device=DEV) * 1e-3).to(DTYPES[c["dtype"]])
        return s
    if c["kind"] == "xent":
        lead, extra = (c["batch"], c["steps"]), 1 if c["sliced"] else 0
        # logits of every sharpness: hidden states of unit size, some far larger
        x = torch.randn(lead[0], lead[1] + extra, c["channels"], generator=g, device=DEV)
        x *= torch.exp(0.5 * torch.randn(lead[0], lead[1] + extra, 1, generator=g, device=DEV))
        s["x"] = x.to(torch.bfloat16)
        w = torch.randn(c["vocab"], c["channels"], generator=g, device=DEV).mul_(2.0 / math.sqrt(c["channels"])).to(torch.bfloat16)
        s["weight"] = w.t() if c["tied"] else w.t().contiguous()
        t = _words(lead, c["vocab"], g)
        s["targets"] = torch.where(torch.rand(lead, generator=g, device=DEV) < c["ignored"], -1, t)
        if c["train"]:                  # a mean's cotangent, with weights of its own for each sequence
            s["g"] = ((0.5 + torch.rand(lead[0], 1, generator=g, device=DEV)) / (lead[0] * lead[1])).expand(lead).contiguous()
        return s
    less = min(c["rows"], c["cols"])
    r = max(1, int(c["rank"] * less))
    left = torch.randn(c["layers"], c["rows"], r, generator=g, device=DEV) * torch.arange(1, r + 1, device=DEV) ** -0.5
    s["update"] = (torch.bmm(left, torch.randn(c["layers"], r, c["cols"], generator=g, device=DEV)) * 1e-4).to(DTYPES[c["dtype"]])
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------------

def _plain_embed(s):
    c, ids, table = s["case"], s["ids"], s["table"]
    there = torch.ones_like(ids, dtype=torch.bool) if s["padding"] is None else ids != s["padding"]
    out = {"rows": torch.where(there.unsqueeze(-1), table[ids].float() * c["scale"], 0.0).to(table.dtype)}
    if c["train"]:
        g = torch.where(there.unsqueeze(-1), s["g"].float(), 0.0).view(-1, c["channels"])
        out["d_table"] = (torch.zeros(table.shape, device=table.device).index_add_(0, ids.view(-1), g) * c["scale"]).to(table.dtype)
    return out


def _positions(s):
    """The hidden states of the positions that count: all, or all but each sequence's last."""
    return s["x"][:, :-1] if s["case"]["sliced"] else s["x"]


def _plain_xent(s):
    c, t = s["case"], s["targets"].view(-1)
    x, w = _positions(s).float().reshape(t.shape[0], -1), s["weight"].float()
    z = torch.matmul(x, w)
    top = z.amax(-1, keepdim=True)
    lse = top + torch.log(torch.exp(z - top).sum(-1, keepdim=True))
    some = t >= 0
    at = t.clamp(min=0).unsqueeze(-1)
    loss = lse - (1.0 - c["smoothing"]) * z.gather(-1, at) - c["smoothing"] * z.mean(-1, keepdim=True)
    out = {"loss": torch.where(some, loss.squeeze(-1), 0.0).view(s["targets"].shape)}
    if c["train"]:
        g = torch.where(some, s["g"].view(-1), 0.0).unsqueeze(-1)
        dz = (torch.exp(z - lse) - c["smoothing"] / c["vocab"]) * g
        dz.scatter_add_(-1, at, g * (c["smoothing"] - 1.0))
        out["d_x"] = torch.matmul(dz, w.t()).to(torch.bfloat16).view(*s["targets"].shape, -1)
        out["d_weight"] = torch.matmul(x.t(), dz).to(torch.bfloat16)
    return out


def _plain_ortho(s):
    a, b, c = COEFFICIENTS
    x = s["update"].float()
    tall = x.shape[-2] > x.shape[-1]
    x = x.transpose(-2, -1) if tall else x
    size = x.double().square().sum((-2, -1), keepdim=True).sqrt()
    x = (x.double() / (size + 1e-7)).float()
    for _ in range(STEPS):
        gram = torch.matmul(x, x.transpose(-2, -1))
        x = a * x + torch.matmul(b * gram + c * torch.matmul(gram, gram), x)
    return {"update": (x.transpose(-2, -1) if tall else x).to(torch.bfloat16)}


# ---- one pass ----------------------------------------------------------------------------------------------------------

def run(state):
    return _own(state) if own else _plain(state)


def _plain(s):
    kind = s["case"]["kind"]
    return _plain_embed(s) if kind == "embed" else _plain_xent(s) if kind == "xent" else _plain_ortho(s)


def _own(s):
    from pratchya_b200._nnx_impl import embedding_lookup, linear_cross_entropy, orthogonalize
    c = s["case"]
    if c["kind"] == "embed":
        if not c["train"]:
            return {"rows": embedding_lookup(s["table"], s["ids"], scale=c["scale"], padding_id=s["padding"])}
        table = s["table"].detach().requires_grad_(True)
        rows = embedding_lookup(table, s["ids"], scale=c["scale"], padding_id=s["padding"])
        (d_table,) = torch.autograd.grad(rows, table, s["g"])
        return {"rows": rows.detach(), "d_table": d_table}
    if c["kind"] == "xent":
        if not c["train"]:
            return {"loss": linear_cross_entropy(_positions(s), s["weight"], s["targets"], smoothing=c["smoothing"])}
        x, w = _positions(s).detach().requires_grad_(True), s["weight"].detach().requires_grad_(True)
        loss = linear_cross_entropy(x, w, s["targets"], smoothing=c["smoothing"])
        d_x, d_weight = torch.autograd.grad(loss, (x, w), s["g"])
        return {"loss": loss.detach(), "d_x": d_x, "d_weight": d_weight}
    return {"update": orthogonalize(s["update"], steps=STEPS, coefficients=COEFFICIENTS)}


def work(case):
    c = case
    if c["kind"] == "embed":
        e, tokens = {"f32": 4, "bf16": 2}[c["dtype"]], c["batch"] * c["steps"]
        row = c["channels"] * e
        size = tokens * (8 + row) + min(tokens, c["vocab"]) * row
        if c["train"]:
            size += tokens * row + c["vocab"] * row
        return {"bytes": size, "flops": tokens * c["channels"] * (2 if c["train"] else 1)}
    if c["kind"] == "xent":
        tokens = c["batch"] * c["steps"]
        size, products = 2 * c["channels"] * (tokens + c["vocab"]), 2 * tokens * c["channels"] * c["vocab"]
        if c["train"]:              # the logits, their gradient to the hidden states, and to the weight
            return {"bytes": 2 * size + 16 * tokens, "flops": 3 * products}
        return {"bytes": size + 12 * tokens, "flops": products}
    less, more = min(c["rows"], c["cols"]), max(c["rows"], c["cols"])
    e = {"f32": 4, "bf16": 2}[c["dtype"]]
    # a step's Gram matrix and its square are symmetric: half of each
    step = less * less * more + less ** 3 + 2 * less * less * more
    return {"bytes": c["layers"] * c["rows"] * c["cols"] * (e + 2), "flops": c["layers"] * STEPS * step}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------

def _exact_xent(c, x, w, t, g):
    """One block of positions by torch's own log-softmax and its derivative."""
    x, z = x.double(), None
    z = (x @ w).requires_grad_(g is not None)
    logp = torch.log_softmax(z, -1)
    hit = -logp.gather(-1, t.clamp(min=0).unsqueeze(-1)).squeeze(-1)
    loss = torch.where(t < 0, 0.0, (1.0 - c["smoothing"]) * hit - c["smoothing"] * logp.mean(-1))
    if g is None:
        return loss, None, None
    (dz,) = torch.autograd.grad(loss, z, g.double())
    return loss.detach(), dz @ w.t(), x.t() @ dz


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "embed":
        ids, width = s["ids"].reshape(-1), c["channels"]
        keep = ids != (-1 if s["padding"] is None else s["padding"])
        rows = torch.zeros(ids.numel(), width, dtype=torch.float64, device=ids.device)
        rows[keep] = s["table"].index_select(0, ids[keep]).double() * c["scale"]
        out = {"rows": rows.view(*s["ids"].shape, width)}
        if c["train"]:
            d = torch.zeros(c["vocab"], width, dtype=torch.float64, device=ids.device)
            d.index_put_((ids[keep],), s["g"].reshape(-1, width)[keep].double() * c["scale"], accumulate=True)
            out["d_table"] = d
        return out
    if c["kind"] == "xent":
        x, w, t = s["x"][:, : c["steps"]].reshape(-1, c["channels"]), s["weight"].double(), s["targets"].reshape(-1)
        g = s["g"].reshape(-1) if c["train"] else None
        step, losses, dxs, dw = max(1, (1 << 27) // c["vocab"]), [], [], 0.0
        for r in range(0, t.shape[0], step):
            at = slice(r, r + step)
            loss, dx, more = _exact_xent(c, x[at], w, t[at], g[at] if g is not None else None)
            losses.append(loss)
            if g is not None:
                dxs.append(dx)
                dw = dw + more
        out = {"loss": torch.cat(losses).view(s["targets"].shape)}
        if c["train"]:
            out["d_x"], out["d_weight"] = torch.cat(dxs).view(*s["targets"].shape, -1), dw
        return out
    a, b, k = COEFFICIENTS
    outs = []
    for u in s["update"]:               # X (a + S (b + k S)), S the smaller of X^T X and X X^T
        x = u.double()
        x = x / (torch.linalg.matrix_norm(x) + 1e-7)
        for _ in range(STEPS):
            if x.shape[0] >= x.shape[1]:
                p = x.t() @ x
                x = a * x + (b * x + k * (x @ p)) @ p
            else:
                p = x @ x.t()
                x = a * x + p @ (b * x + k * (p @ x))
        outs.append(x)
    return {"update": torch.stack(outs)}
