"""The operators that take a trained model to answers and scores, as cases that can be timed: log probabilities of given tokens with
entropy and top alternatives (and their gradient), products of few rows with 4-bit weights, and the 4-bit quantizer.

A case is a dict of plain values.  `listed()` gives the listed ones, `draw(rng)` one more of the same ranges, `prepare` what a
program holds before the call, `run` one pass: the plain form in elementary torch operations, or, where `own` is set, the call of this
framework; `exact` what the definition gives in 64 bits, `work` the bytes and operations that a pass cannot do without."""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # one decoding step: one row of logits, the five best next tokens
        dict(name="score_step", kind="score", batch=1, steps=1, vocab=65536, tokens=1, top=5, dtype="f32", sliced=False, masked=False),
        # a decoding step of a batch under a grammar that rules most of the vocabulary out
        dict(name="score_batch_masked", kind="score", batch=48, steps=1, vocab=65536, tokens=1, top=20, dtype="f32", sliced=False, masked=True),
        # scoring texts: position t's logits against token t+1, so the last position's logits are sliced away; an odd vocabulary
        dict(name="score_text_odd", kind="score", batch=3, steps=777, vocab=32003, tokens=1, top=1, dtype="bf16", sliced=True, masked=False),
        # a teacher's alternatives over a long batch, to distil from
        dict(name="score_teacher", kind="score", batch=8, steps=1024, vocab=65536, tokens=1, top=64, dtype="bf16", sliced=False, masked=False),
        # a policy's loss: log probabilities of the sampled tokens and an entropy bonus, forward and the logits' gradient
        dict(name="policy_train", kind="train", batch=4, steps=1024, vocab=65536, tokens=1, top=0, dtype="f32", sliced=False, masked=False),
        # distillation: log probabilities of a teacher's sixteen alternatives at each position, and of the student's own best
        dict(name="distil_train_odd", kind="train", batch=3, steps=341, vocab=32003, tokens=16, top=4, dtype="bf16", sliced=True, masked=False),
        # the smallest product of a decoding step: a low-rank layer's down-projection
        dict(name="int4_lora_down", kind="matvec", rows=1, fan_in=2048, fan_out=128, group=128, zero_points=False, dtype="f32"),
        # the logits of one token
        dict(name="int4_lm_head", kind="matvec", rows=1, fan_in=2048, fan_out=65536, group=128, zero_points=False, dtype="f32"),
        # a small batch's up-projection
        dict(name="int4_up_batch", kind="matvec", rows=8, fan_in=2048, fan_out=8192, group=64, zero_points=True, dtype="bf16"),
        # a larger batch's down-projection: a long contraction, few columns, small groups
        dict(name="int4_down_batch", kind="matvec", rows=32, fan_in=8192, fan_out=2048, group=32, zero_points=True, dtype="bf16"),
        # a ChannelMix weight taken to 4 bits and read back
        dict(name="int4_quantize_up", kind="quantize", fan_in=2048, fan_out=8192, group=128, zero_points=False, dtype="f32"),
        # a weight of no particular size, with zero points
        dict(name="int4_quantize_odd", kind="quantize", fan_in=1000, fan_out=777, group=32, zero_points=True, dtype="bf16"),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["score", "score", "train", "matvec", "matvec", "quantize"])
    dtype = rng.choice(["f32", "bf16"])
    if kind in ("score", "train"):
        vocab = _log(rng, 1000, 131072)
        if rng.random() < 0.5:
            vocab -= vocab % 8
        rows = _log(rng, 1, min(4096, (1 << 28) // vocab))
        batch = rng.choice([1, 2, 3, 8])
        return dict(kind=kind, batch=min(batch, rows), steps=max(1, rows // batch), vocab=vocab, tokens=rng.choice([1, 1, 4, 16]),
                    top=rng.choice([0, 1, 5, 20, 64, 128]), dtype=dtype, sliced=rng.random() < 0.5, masked=rng.random() < 0.3)
    group, zeros = rng.choice([32, 64, 128]), rng.random() < 0.5
    fan_in = _log(rng, 128, 16384)
    fan_out = _log(rng, 64, min(65536, (1 << 27) // fan_in))
    if rng.random() < 0.6:
        fan_in, fan_out = max(128, fan_in - fan_in % 128), max(64, fan_out - fan_out % 16)
    if kind == "matvec":
        return dict(kind=kind, rows=_log(rng, 1, 32), fan_in=fan_in, fan_out=fan_out, group=group, zero_points=zeros, dtype=dtype)
    return dict(kind=kind, fan_in=fan_in, fan_out=min(fan_out, (1 << 24) // fan_in), group=group, zero_points=zeros, dtype=dtype)


# ---- inputs ----------------------------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 17)


def _logits(c, g):
    """Rows of every sharpness.  masked: nine logits in ten are ruled out in every second row, by -inf or by the type's lowest value, and one
    row in sixteen has nothing left."""
    rows, extra = (c["batch"], c["steps"]), 1 if c["sliced"] else 0
    z = torch.randn(rows[0], rows[1] + extra, c["vocab"], generator=g, device=DEV)
    z *= torch.exp(torch.randn(rows[0], rows[1] + extra, 1, generator=g, device=DEV) * 0.6) * 2.5
    z = z.to(DTYPES[c["dtype"]])
    if c["masked"]:
        which = torch.randint(0, 16, (rows[0], rows[1] + extra, 1), generator=g, device=DEV)
        out = torch.rand(z.shape, generator=g, device=DEV) < 0.9
        z.masked_fill_(out & (which % 4 == 0), -math.inf)
        z.masked_fill_(out & (which % 4 == 2), torch.finfo(z.dtype).min)
        z.masked_fill_(which == 15, -math.inf)
    return z


def prepare(case, seed):
    c, g = case, _gen(seed)
    s = {"case": c}
    if c["kind"] in ("score", "train"):
        lead = (c["batch"], c["steps"])
        s["logits"] = _logits(c, g)
        t = torch.randint(0, c["vocab"], (*lead, c["tokens"]), generator=g, device=DEV)
        if c["masked"]:                                                                       # nobody answers with what is ruled out
            z = _positions(s)
            t = torch.where(z.gather(-1, t) <= torch.finfo(z.dtype).min, z.argmax(-1, keepdim=True), t)
        t = torch.where(torch.rand(t.shape, generator=g, device=DEV) < 0.05, -1, t)          # positions without a token
        s["tokens"] = t if c["tokens"] > 1 else t[..., 0].contiguous()
        if c["kind"] == "train":
            scale = 1.0 / (lead[0] * lead[1])
            s["g_logprobs"] = torch.randn(s["tokens"].shape, generator=g, device=DEV) * scale
            s["g_entropy"] = torch.randn(lead, generator=g, device=DEV) * (0.1 * scale)
            s["g_top"] = torch.randn(*lead, c["top"], generator=g, device=DEV) * scale
        return s
    w = (torch.randn(c["fan_in"], c["fan_out"], generator=g, device=DEV) / math.sqrt(c["fan_in"])).to(DTYPES[c["dtype"]])
    if c["kind"] == "quantize":
        s["w"] = w
        return s
    s["q"], s["scale"], s["zero"], _ = _to_int4(w, c["group"], c["zero_points"])
    x = torch.randn(c["rows"], c["fan_in"], generator=g, device=DEV)
    x = torch.where(torch.rand(x.shape, generator=g, device=DEV) < 0.01, x * 16.0, x)         # the outliers that activations have
    s["x"] = x.to(DTYPES[c["dtype"]])
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------------

def _positions(s):
    """The logits of the positions that count: all, or all but each sequence's last."""
    return s["logits"][:, :-1] if s["case"]["sliced"] else s["logits"]


def _order(z):
    """A whole number for each value that is larger for larger values and, among equal ones, for lower indices."""
    bits = (z + 0.0).view(torch.int32)
    value = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).to(torch.int64)
    return value * (1 << 32) + ((1 << 32) - 1 - torch.arange(z.shape[-1], device=z.device))


def _logprobs(z):
    """(logp, p, empty) of rows of f32 logits; a row without any logit has logp = -inf and p = 0."""
    top = z.amax(-1, keepdim=True)
    d = z - torch.where(top == -math.inf, 0.0, top)
    e = torch.exp(d)
    total = e.sum(-1, keepdim=True)
    empty = total == 0
    logp = torch.where(empty, -math.inf, d - torch.log(total))
    return logp, torch.where(empty, 0.0, e / total), empty


def _plain_score(s):
    z = _positions(s).float()
    logp, p, empty = _logprobs(z)
    t = s["tokens"].reshape(*z.shape[:-1], -1)
    picked = torch.where(t < 0, 0.0, logp.gather(-1, t.clamp(min=0))).reshape(s["tokens"].shape)
    entropy = -torch.where(p > 0, p * logp, 0.0).sum(-1)
    order = torch.topk(_order(z), s["case"]["top"], dim=-1).indices if s["case"]["top"] else t[..., :0]
    out = {"logprobs": picked, "entropy": entropy, "top_logprobs": logp.gather(-1, order), "top_tokens": order}
    return out, logp, p, empty, t


def _plain_train(s):
    out, logp, p, empty, t = _plain_score(s)
    g = torch.where(t < 0, 0.0, s["g_logprobs"].reshape(t.shape))
    total = g.sum(-1, keepdim=True) + s["g_top"].sum(-1, keepdim=True)
    minus_h = torch.where(p > 0, logp + out["entropy"].unsqueeze(-1), 0.0)
    dz = -p * (total + s["g_entropy"].unsqueeze(-1) * minus_h)
    dz.scatter_add_(-1, t.clamp(min=0), torch.where(empty, 0.0, g))
    dz.scatter_add_(-1, out["top_tokens"], torch.where(empty, 0.0, s["g_top"]))
    out["d_logits"] = dz.to(s["logits"].dtype)
    return out


def _pad(w, rows, cols):
    return torch.nn.functional.pad(w, (0, cols - w.shape[1], 0, rows - w.shape[0]))


def _to_tiles(u):
    """[128 Kb, 16 A] numbers of 0 to 15 -> uint8 [A, Kb, 1024]: the order in which a 4-bit weight is stored."""
    kb, a = u.shape[0] // 128, u.shape[1] // 16
    u = u.view(kb, 4, 4, 2, 2, 2, a, 2, 8).permute(6, 0, 7, 8, 2, 1, 5, 3, 4)       # k = (c, t, byte's low bit, high half, byte's high bit), n = (half, g)
    u = u.to(torch.uint8)
    return (u[..., 0] | (u[..., 1] << 4)).reshape(a, kb, 1024)


def _from_tiles(q):
    """The inverse of _to_tiles."""
    a, kb = q.shape[:2]
    u = torch.stack([q & 15, q >> 4], dim=-1).view(a, kb, 2, 8, 4, 4, 2, 2, 2)
    return u.permute(1, 5, 4, 7, 8, 6, 0, 2, 3).reshape(kb * 128, a * 16)


def _to_int4(w, group, zero_points):
    """(q, scale, zero or None, the values they stand for) of w [K, N], groups of `group` along K."""
    k, n = w.shape
    kp, np_ = -(-k // 128) * 128, -(-n // 16) * 16
    w = _pad(w.float(), kp, np_).view(kp // group, group, np_)
    steps = torch.full((1,), 15.0 if zero_points else 7.0, device=w.device)          # a tensor: torch multiplies by a number's reciprocal instead of dividing
    if zero_points:
        low, high = w.amin(1, keepdim=True).clamp(max=0.0), w.amax(1, keepdim=True).clamp(min=0.0)
        s = ((high - low) / steps).to(torch.bfloat16).float()
        some = s > 0
        z = torch.where(some, torch.round(-low / s).clamp(0.0, 15.0), 0.0)
        u = torch.where(some, (torch.round(w / s) + z).clamp(0.0, 15.0), 0.0)
    else:
        s = (w.abs().amax(1, keepdim=True) / steps).to(torch.bfloat16).float()
        z = torch.full_like(s, 8.0)
        u = torch.where(s > 0, torch.round(w / s).clamp(-8.0, 7.0), 0.0) + 8.0
    values = ((u - z) * s).view(kp, np_)[:k, :n]

    def parts(t, dtype):         # [K/g, 1, N] -> [A, Kb, 16, 128/g]
        return t.view(kp // 128, 128 // group, np_ // 16, 16).permute(2, 0, 3, 1).contiguous().to(dtype)

    return _to_tiles(u.view(kp, np_)), parts(s, torch.bfloat16), parts(z, torch.uint8) if zero_points else None, values


def _plain_matvec(s):
    c, q = s["case"], s["q"]
    a, kb = q.shape[:2]

    def spread(t):               # [A, Kb, 16, 128/g] -> [K/g, 1, N]
        return t.permute(1, 3, 0, 2).reshape(-1, 1, a * 16).float()

    u = _from_tiles(q).float().view(-1, c["group"], a * 16)
    z = spread(s["zero"]) if s["zero"] is not None else 8.0
    w = ((u - z) * spread(s["scale"])).view(kb * 128, a * 16)[: c["fan_in"], : c["fan_out"]]
    return torch.matmul(s["x"].float(), w).to(s["x"].dtype)


# ---- one pass ----------------------------------------------------------------------------------------------------------

def run(state):
    return _own(state) if own else _plain(state)


def _plain(s):
    kind = s["case"]["kind"]
    if kind == "score":
        return _plain_score(s)[0]
    if kind == "train":
        return _plain_train(s)
    if kind == "matvec":
        return _plain_matvec(s)
    _, scale, zero, values = _to_int4(s["w"], s["case"]["group"], s["case"]["zero_points"])
    return {"values": values.to(s["w"].dtype), "scale": scale, "zero": zero}


def _own(s):
    from pratchya_b200._nnx_impl import token_logprobs
    from pratchya_b200._qualia import dequantize_int4_impl, int4_matmul_impl, quantize_int4_impl
    c = s["case"]
    if c["kind"] == "matvec":
        return int4_matmul_impl(s["x"], s["q"], s["scale"], s["zero"], c["fan_out"])
    if c["kind"] == "quantize":
        q, scale, zero = quantize_int4_impl(s["w"], c["group"], c["zero_points"])
        return {"values": dequantize_int4_impl(q, scale, zero, s["w"].shape, s["w"].dtype), "scale": scale, "zero": zero}
    if c["kind"] == "score":
        r = token_logprobs(_positions(s), s["tokens"], top=c["top"])
        return {"logprobs": r.logprobs, "entropy": r.entropy, "top_logprobs": r.top_logprobs, "top_tokens": r.top_tokens}
    z = _positions(s).detach().requires_grad_(True)
    r = token_logprobs(z, s["tokens"], top=c["top"])
    outs, gs = [r.logprobs, r.entropy], [s["g_logprobs"], s["g_entropy"]]
    if c["top"]:
        outs.append(r.top_logprobs)
        gs.append(s["g_top"])
    (dz,) = torch.autograd.grad(outs, z, gs)
    return {"logprobs": r.logprobs.detach(), "entropy": r.entropy.detach(), "top_logprobs": r.top_logprobs.detach(), "top_tokens": r.top_tokens, "d_logits": dz}


def work(case):
    c, e = case, {"f32": 4, "bf16": 2}[case["dtype"]]
    if c["kind"] in ("score", "train"):
        rows, n = c["batch"] * c["steps"], c["batch"] * c["steps"] * c["vocab"]
        small = rows * (12 * c["tokens"] + 12 * c["top"] + 4)
        if c["kind"] == "score":
            return {"bytes": n * e + small, "flops": 6 * n}
        return {"bytes": 3 * n * e + 2 * small, "flops": 14 * n}          # the logits twice, since a sum over a row stands between, and their gradient
    n = c["fan_in"] * c["fan_out"]
    groups = -(-c["fan_in"] // c["group"]) * c["fan_out"]
    stored = n / 2 + groups * (3 if c["zero_points"] else 2)
    if c["kind"] == "matvec":
        return {"bytes": stored + c["rows"] * (c["fan_in"] + c["fan_out"]) * e, "flops": 2 * c["rows"] * n}
    return {"bytes": n * e + 2 * stored + n * e, "flops": 6 * n}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------

def _exact_rows(z, t, top, gs):
    """One block of rows: z [r, V], t [r, n], in 64 bits, by torch's own log-softmax and its derivative."""
    z = z.double()
    dead = (z == -math.inf).all(-1, keepdim=True)
    x = torch.where(dead, 0.0, z).requires_grad_(gs is not None)
    logp = torch.log_softmax(x, -1)
    plogp = torch.where(logp == -math.inf, 0.0, logp.exp() * torch.where(logp == -math.inf, 0.0, logp))
    entropy = torch.where(dead[:, 0], 0.0, -plogp.sum(-1))
    picked = torch.where(t < 0, 0.0, logp.gather(-1, t.clamp(min=0)))
    best = torch.sort(x.detach(), dim=-1, descending=True, stable=True).indices[:, :top]
    tops = logp.gather(-1, best)
    grad = None
    if gs is not None:
        live = ~dead
        total = (torch.where(live & (t >= 0), picked * gs[0].double(), 0.0).sum() + torch.where(live[:, 0], entropy * gs[1].double(), 0.0).sum()
                 + torch.where(live, tops * gs[2].double(), 0.0).sum())
        (grad,) = torch.autograd.grad(total, x)
    none = torch.tensor(-math.inf, dtype=torch.float64, device=z.device)
    picked = torch.where(dead & (t >= 0), none, picked)
    return picked.detach(), entropy.detach(), torch.where(dead, none, tops).detach(), grad


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] in ("score", "train"):
        z = s["logits"][:, : c["steps"]]
        rows = c["batch"] * c["steps"]
        t = s["tokens"].reshape(rows, -1)
        gs = [s["g_logprobs"].reshape(rows, -1), s["g_entropy"].reshape(rows), s["g_top"].reshape(rows, -1)] if c["kind"] == "train" else None
        step, parts = max(1, (1 << 26) // c["vocab"]), []
        flat = z.reshape(rows, c["vocab"])
        for r in range(0, rows, step):
            parts.append(_exact_rows(flat[r:r + step], t[r:r + step], c["top"], [g[r:r + step] for g in gs] if gs else None))
        picked, entropy, tops = (torch.cat([p[i] for p in parts]) for i in range(3))
        out = {"logprobs": picked.reshape(s["tokens"].shape), "entropy": entropy.reshape(z.shape[:2]), "top_logprobs": tops.reshape(*z.shape[:2], c["top"]), "top_tokens": None}
        if gs:
            out["d_logits"] = torch.cat([p[3] for p in parts]).reshape(z.shape)
        return out
    if c["kind"] == "quantize":
        w, g = s["w"].double(), c["group"]
        k, n = w.shape
        values, scales, zeros = torch.zeros_like(w), [], []
        for lo in range(0, k, g):
            block = w[lo:lo + g]
            if c["zero_points"]:
                low, high = block.amin(0).clamp(max=0), block.amax(0).clamp(min=0)
                step = ((high - low) / 15).to(torch.bfloat16).double()
                z = torch.where(step > 0, torch.round(-low / step).clamp(0, 15), 0.0)
                values[lo:lo + g] = torch.where(step > 0, (torch.clamp(torch.round(block / step) + z, 0, 15) - z) * step, 0.0)
            else:
                step = (block.abs().amax(0) / 7).to(torch.bfloat16).double()
                values[lo:lo + g] = torch.where(step > 0, torch.round(block / step) * step, 0.0)
            scales.append(step)
        scale = torch.zeros(-(-k // 128) * (128 // g), -(-n // 16) * 16, dtype=torch.float64, device=w.device)
        scale[: len(scales), :n] = torch.stack(scales)
        scale = scale.view(-1, 128 // g, -(-n // 16), 16).permute(2, 0, 3, 1).contiguous()
        return {"values": values, "scale": scale, "zero": None}
    # a column's weights from their stored bytes, one nibble position at a time
    q, k, n, g = s["q"], c["fan_in"], c["fan_out"], c["group"]
    a, kb = q.shape[:2]
    words = q.view(a, kb, 2, 8, 4, 4, 4).to(torch.int64)                                # half, g, t, c, byte
    w = torch.zeros(kb * 128, a * 16, dtype=torch.float64, device=q.device).view(kb, 4, 4, 8, a, 2, 8)      # c, t, place, half, g
    for place in range(8):
        p = place // 2 + 4 * (place % 2)
        code = (words[..., p // 2] >> (4 * (p % 2))) & 15                               # A, Kb, half, g, t, c
        w[:, :, :, place] = code.permute(1, 5, 4, 0, 2, 3).double()
    w = w.reshape(kb * 128 // g, g, a, 16)
    scale = s["scale"].double().permute(1, 3, 0, 2).reshape(kb * 128 // g, 1, a, 16)
    zero = s["zero"].double().permute(1, 3, 0, 2).reshape(kb * 128 // g, 1, a, 16) if s["zero"] is not None else 8.0
    w = ((w - zero) * scale).reshape(kb * 128, a * 16)[:k, :n]
    return s["x"].double() @ w
