"""Operators of a student model without attention in every layer, as cases with inputs, one pass and its useful work.

Three places of its training step, and its serving: the gated delta rule that mixes a sequence in time linear in its length
(`ops.gated_delta_rule_fwd` / `_bwd`, and `ops.gated_delta_step_` token by token), layer norms with the residual addition and the sums of their weights'
gradients (`ops.layernorm_fwd` / `_bwd`), and the loss against a teacher's top logits (`blockops.distill_loss`).
Sizes are those of the framework's own models and benchmarks: the 35 M parameter Llama (8 heads of 64, d = 512, 32000 words, 8 x 1024 tokens), grouped
heads of a half-billion-parameter model (14 to 2, head size 64), 16 heads of 128 over 4 x 4096 tokens.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
F32, F64 = torch.float32, torch.float64


# ---- cases -----------------------------------------------------------------------------------------------------------


def _delta(name, B, T, Hk, Hv, dk, dv, dtype, train, state=False, pad=0, documents=1):
    """train: forward and backward. state: a state comes in (and its gradient goes out). pad: tokens behind the last of some sequences. documents: in each row,
    each of them starting afresh."""
    return {"name": name, "kind": "delta", "B": B, "T": T, "Hk": Hk, "Hv": Hv, "dk": dk, "dv": dv, "dtype": dtype, "train": train, "state": state,
            "pad": pad, "documents": documents}


def _step(name, B, T, Hk, Hv, dk, dv, dtype):
    return {"name": name, "kind": "step", "B": B, "T": T, "Hk": Hk, "Hv": Hv, "dk": dk, "dv": dv, "dtype": dtype}


def _norm(name, rows, cols, dtype, train, residual=True, bias=True):
    return {"name": name, "kind": "norm", "rows": rows, "cols": cols, "dtype": dtype, "train": train, "residual": residual, "bias": bias}


def _distill(name, rows, vocab, top, dtype, train, tau=1.0, unused=0.0, ragged=False, tail=False):
    """top: the teacher's words for each row; ragged: some rows have fewer. unused: share of rows of weight zero. tail: the teacher's own sum is known, so its words
    have less than all of the mass."""
    return {"name": name, "kind": "distill", "rows": rows, "vocab": vocab, "top": top, "dtype": dtype, "train": train, "tau": tau, "unused": unused,
            "ragged": ragged, "tail": tail}


def listed():
    return [
        # One new token of one sequence, heads of the 35 M parameter model: latency.
        _step("step_one", 1, 1, 8, 8, 64, 64, "bf16"),
        # One new token of each of 256 sequences, 16 heads of 128: the states' traffic.
        _step("step_batch", 256, 1, 16, 16, 128, 128, "bf16"),
        # A prompt of 8192 tokens on grouped heads, forward only.
        _delta("delta_prompt", 1, 8192, 2, 14, 64, 64, "bf16", False),
        # Training of the 35 M parameter model's batch.
        _delta("delta_train", 8, 1024, 8, 8, 64, 64, "bf16", True),
        # Long-context training, 16 heads of 128.
        _delta("delta_train_long", 4, 4096, 16, 16, 128, 128, "bf16", True),
        # Full precision, head sizes between the usual ones, an odd number of tokens, several documents in a row, padding, a state that comes in.
        _delta("delta_odd_fp32", 3, 1021, 3, 6, 48, 80, "fp32", True, state=True, pad=37, documents=3),
        # Residual addition and norm of 64 tokens that are being generated: latency.
        _norm("norm_small", 64, 512, "bf16", False),
        # Training, 4 x 4096 tokens of 16 heads of 128.
        _norm("norm_train", 16384, 2048, "bf16", True),
        # Full precision, odd sizes, no residual, no bias.
        _norm("norm_odd_fp32", 3001, 1001, "fp32", True, residual=False, bias=False),
        # A small step in full precision: odd vocabulary, temperature, a third of the rows unused, rows with fewer words.
        _distill("distill_small", 250, 32003, 20, "fp32", True, tau=2.0, unused=0.3, ragged=True),
        # The 35 M parameter model's batch against 64 words of the teacher.
        _distill("distill_step", 8192, 32000, 64, "bf16", True),
        # Validation: the loss alone, the teacher's sum known.
        _distill("distill_score", 2000, 32003, 128, "fp32", False, tail=True),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["delta", "delta", "step", "norm", "distill"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if kind in ("delta", "step"):
        dk = rng.choice([32, 64, 64, 96, 128, 128, rng.randint(1, 128)])
        dv = rng.choice([dk, dk, 64, 128, 256, rng.randint(1, 256)])
        Hk, rep = rng.randint(1, 8), rng.choice([1, 1, 2, 7])
        Hv = Hk * rep
        if kind == "step":
            T = rng.choice([1, 1, 1, rng.randint(2, 8)])
            B = max(1, min(256 * 16 * 128 * 128 // (Hv * dk * dv), _log_uniform(rng, 1, 256)))
            return _step(None, B, T, Hk, Hv, dk, dv, dtype)
        T = _log_uniform(rng, 1, 8192)
        most = 4 * 4096 * 16 * 128 * 128 // (4 if dtype == "fp32" else 1)
        T = max(1, min(T, most // (Hv * dk * dv)))
        B = max(1, min(most // (T * Hv * dk * dv), _log_uniform(rng, 1, 16)))
        return _delta(None, B, T, Hk, Hv, dk, dv, dtype, rng.random() < 0.7, rng.random() < 0.4, rng.choice([0, 0, min(T - 1, 50)]), rng.choice([1, 1, min(T, 4)]))
    if kind == "norm":
        cols = rng.choice([512, 1024, 2048, 4096, _log_uniform(rng, 1, 20000)])
        rows = max(1, min(_log_uniform(rng, 1, 20000), 16384 * 2048 // cols))
        return _norm(None, rows, cols, dtype, rng.random() < 0.7, rng.random() < 0.6, rng.random() < 0.7)
    vocab = _log_uniform(rng, 50, 150000)
    rows = max(1, min(_log_uniform(rng, 1, 8192), 8192 * 16000 // vocab))
    return _distill(None, rows, vocab, min(vocab, _log_uniform(rng, 1, 200)), dtype, rng.random() < 0.7, rng.choice([1.0, 2.0, 0.7]), rng.choice([0.0, 0.25]),
                    rng.random() < 0.3, rng.random() < 0.3)


# ---- inputs ----------------------------------------------------------------------------------------------------------


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.rand(s, generator=gen, device="cuda")        # noqa: E731
    randn = lambda *s: torch.randn(s, generator=gen, device="cuda")      # noqa: E731
    s, kind, dtype = {"case": case}, case["kind"], DTYPES[case["dtype"]]
    if kind in ("delta", "step"):
        B, T, Hk, Hv, dk, dv = (case[n] for n in ("B", "T", "Hk", "Hv", "dk", "dv"))
        unit = lambda x: x / x.square().sum(-1, keepdim=True).sqrt().clamp(min=1e-6)  # noqa: E731
        drift = randn(1, 1, Hk, dk)   # keys of one head have something in common
        s["q"], s["k"] = unit(randn(B, T, Hk, dk)).to(dtype), unit(randn(B, T, Hk, dk) + 0.5 * drift).to(dtype)
        s["v"] = randn(B, T, Hv, dv).to(dtype)
        s["beta"] = torch.sigmoid(randn(B, T, Hv) + 0.5)
        # Log-decays: heads that forget within ten tokens and heads that remember thousands.
        s["g"] = -torch.nn.functional.softplus(randn(B, T, Hv)) * torch.exp(-7.0 * rand(1, 1, Hv))
        s["scale"] = float(torch.tensor(dk ** -0.5, dtype=F32))
        if kind == "step" or case["state"]:
            s["state"] = randn(B, Hv, dk, dv) * dk ** -0.5
        if kind == "delta":
            pick = random.Random(T * 7919 + case["documents"])
            for at in sorted(pick.sample(range(T), case["documents"] - 1)) if case["documents"] > 1 else ():
                s["g"][:, at] = -math.inf        # a token that starts afresh
            if case["pad"]:                      # padding leaves the state as it is
                s["g"][::2, T - case["pad"]:], s["beta"][::2, T - case["pad"]:] = 0.0, 0.0
            if case["train"]:
                s["do"], s["dstate"] = randn(B, T, Hv, dv).to(dtype), randn(B, Hv, dk, dv)
    elif kind == "norm":
        rows, cols = case["rows"], case["cols"]
        s["x"] = (randn(rows, cols) * torch.exp(0.5 * randn(rows, 1)) + 0.3 * randn(rows, 1)).to(dtype)
        s["w"] = 1.0 + 0.2 * randn(cols)
        s["b"] = 0.2 * randn(cols) if case["bias"] else None
        s["residual"] = (randn(rows, cols) * torch.exp(0.5 * randn(1, cols))).to(dtype) if case["residual"] else None
        if case["train"]:
            s["dy"] = randn(rows, cols).to(dtype)
            s["dh"] = randn(rows, cols).to(dtype) if case["residual"] else None   # what comes down the residual stream
    else:
        rows, vocab, top = case["rows"], case["vocab"], case["top"]
        teacher = randn(rows, vocab).mul_(2.5)
        best = teacher.topk(top, 1)
        s["teacher"], s["indices"] = best.values.contiguous(), best.indices.to(torch.int32)
        if case["tail"]:
            z = teacher / case["tau"]
            s["lse"] = (torch.log(torch.exp(z - z.amax(1, keepdim=True)).sum(1, dtype=F64)) + z.amax(1).double()).to(F32)
        if case["ragged"]:
            keep = (rand(rows, 1) * (top + 1)).long().clamp(min=1)
            s["indices"] = torch.where(torch.arange(top, device="cuda") < keep, s["indices"], -1)
        s["logits"] = teacher.mul_(0.8).add_(randn(rows, vocab)).to(dtype)       # the student is on its way there
        used = (rand(rows) >= case["unused"]).to(F32)
        s["weights"] = used / used.sum().clamp(min=1.0)
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------


def run(s):
    return {"delta": _run_delta, "step": _run_step, "norm": _run_norm, "distill": _run_distill}[s["case"]["kind"]](s)


CHUNK = 64
LEAST = -1000.0   # a decay of e^-1000 is 0 in 64 bits; so is one of e^-inf, whose differences would be no numbers


def _chunked(q, k, v, g, beta, scale, state):
    """The rule over chunks of 64 tokens: with the sum G of a chunk's log-decays and D_ij = exp(G_i - G_j), the chunk's
    u = (I + strict lower(beta_i D_ij k_i.k_j))^-1 beta (v - e^G k S), o = scale (e^G q S + lower(D q k^T) u), S' = e^Gend S + (e^(Gend - G) k)^T u."""
    B, T, Hk, dk = q.shape
    Hv, dv = v.shape[2], v.shape[3]
    short = -T % CHUNK
    put = lambda x: torch.nn.functional.pad(x, (0, 0) * (x.dim() - 2) + (0, short)).unflatten(1, (-1, CHUNK)).transpose(2, 3)  # noqa: E731
    q, k = (put(x.repeat_interleave(Hv // Hk, 2)) for x in (q, k))       # [B, chunks, Hv, 64, dk]
    v, beta, total = put(v), put(beta)[..., None], put(g.clamp(min=LEAST).double()).cumsum(-1)
    lower = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=q.device).tril()
    D = torch.exp(torch.where(lower, total[..., :, None] - total[..., None, :], -math.inf).float())
    M = (beta * D * (k @ k.transpose(-1, -2).contiguous())).tril(-1)
    with torch.no_grad():
        inverse = torch.eye(CHUNK, device=q.device).expand(M.shape).clone()
        for i in range(1, CHUNK):
            inverse[..., i, :] -= (M[..., i:i + 1, :i].contiguous() @ inverse[..., :i, :].contiguous())[..., 0, :]
    inverse = 2.0 * inverse - inverse @ (M @ inverse + inverse)          # of the same value, and with the derivative -inverse dM inverse
    attn = scale * D * (q @ k.transpose(-1, -2).contiguous())
    enter, leave, whole = torch.exp(total.float())[..., None], torch.exp((total[..., -1:] - total).float())[..., None], torch.exp(total[..., -1:].float())[..., None]
    kin, qin, kout = enter * k, scale * enter * q, (leave * k).transpose(-1, -2).contiguous()
    S, outs = state, []
    for c in range(q.shape[1]):
        u = inverse[:, c] @ (beta[:, c] * (v[:, c] - kin[:, c] @ S))
        outs.append(qin[:, c] @ S + attn[:, c] @ u)
        S = whole[:, c] * S + kout[:, c] @ u
    return torch.stack(outs, 1).transpose(2, 3).flatten(1, 2)[:, :T], S


def _run_delta(s):
    c = s["case"]
    if own:
        from paperkiln_amd import ops
        o, state = ops.gated_delta_rule_fwd(s["q"], s["k"], s["v"], s["g"], s["beta"], s["scale"], s.get("state"))
        out = {"o": o, "state": state}
        if c["train"]:
            grads = ops.gated_delta_rule_bwd(s["do"], s["q"], s["k"], s["v"], s["g"], s["beta"], s["scale"], s.get("state"), s["dstate"])
            out.update(zip(("dq", "dk", "dv", "dg", "dbeta", "dstate"), grads[:6 if c["state"] else 5]))
        return out
    B, Hv, dk, dv, kept = c["B"], c["Hv"], c["dk"], c["dv"], s["v"].dtype
    state = s["state"] if c["state"] else torch.zeros(B, Hv, dk, dv, device="cuda")
    leaves = [s["q"].float(), s["k"].float(), s["v"].float(), s["g"], s["beta"], state]
    if not c["train"]:
        with torch.no_grad():
            o, state = _chunked(*leaves[:5], s["scale"], state)
        return {"o": o.to(kept), "state": state}
    leaves = [x.detach().requires_grad_() for x in leaves]
    o, state = _chunked(*leaves[:5], s["scale"], leaves[5])
    grads = torch.autograd.grad([o, state], leaves, [s["do"].float(), s["dstate"]])
    out = {"o": o.detach().to(kept), "state": state.detach()}
    for n, x, g in zip(("dq", "dk", "dv", "dg", "dbeta", "dstate"), ("q", "k", "v", "g", "beta", "state"), grads):
        if n != "dstate" or c["state"]:
            out[n] = g.to(s[x].dtype)
    return out


def _run_step(s):
    if own:
        from paperkiln_amd import ops
        return {"o": ops.gated_delta_step_(s["q"], s["k"], s["v"], s["g"], s["beta"], s["scale"], s["state"]), "state": s["state"]}
    rep = s["case"]["Hv"] // s["case"]["Hk"]
    q, k = (s[n].float().repeat_interleave(rep, 2) for n in ("q", "k"))
    S, outs = s["state"], []
    for t in range(q.shape[1]):
        S = torch.exp(s["g"][:, t])[..., None, None] * S
        u = s["beta"][:, t, :, None] * (s["v"][:, t].float() - (k[:, t, :, :, None] * S).sum(2))
        S = S + k[:, t, :, :, None] * u[:, :, None, :]
        outs.append(s["scale"] * (q[:, t, :, :, None] * S).sum(2))
    s["state"].copy_(S)
    return {"o": torch.stack(outs, 1).to(s["v"].dtype), "state": s["state"]}


EPS = 1e-5


def _run_norm(s):
    c = s["case"]
    if own:
        from paperkiln_amd import ops
        y, h, mean, rstd = ops.layernorm_fwd(s["x"], s["w"], s["b"], EPS, s["residual"])
        out = {"y": y, "h": h, "mean": mean, "rstd": rstd} if c["residual"] else {"y": y, "mean": mean, "rstd": rstd}
        if c["train"]:
            dx, dw, db = ops.layernorm_bwd(s["dy"], h, s["w"], mean, rstd, s["dh"])
            out.update({"dx": dx, "dw": dw, "db": db})
        return out
    h = s["x"]
    if c["residual"]:
        h = (s["x"].float() + s["residual"].float()).to(h.dtype)
    x = h.float()
    mean = x.mean(1, keepdim=True)
    rstd = torch.rsqrt((x - mean).square().mean(1, keepdim=True) + EPS)
    unit = (x - mean) * rstd
    y = unit * s["w"] + s["b"] if c["bias"] else unit * s["w"]
    out = {"y": y.to(h.dtype), "mean": mean[:, 0], "rstd": rstd[:, 0]}
    if c["residual"]:
        out["h"] = h
    if c["train"]:
        dy = s["dy"].float()
        du = dy * s["w"]
        dx = rstd * (du - du.mean(1, keepdim=True) - unit * (du * unit).mean(1, keepdim=True))
        if c["residual"]:
            dx = dx + s["dh"].float()
        out.update({"dx": dx.to(h.dtype), "dw": (dy * unit).sum(0), "db": dy.sum(0)})
    return out


def _run_distill(s):
    c = s["case"]
    tau, w = c["tau"], s["weights"]
    if own:
        from paperkiln_amd import blockops
        loss, dlogits, kl = blockops.distill_loss(s["logits"], s["indices"], s["teacher"], w, temperature=tau, teacher_lse=s.get("lse"), grad=c["train"])
        return {"loss": loss, "dlogits": dlogits, "kl": kl} if c["train"] else {"loss": loss, "kl": kl}
    # Log-probabilities in 64 bits: the loss is a difference of near numbers.
    z = s["logits"].float() / tau
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True, dtype=F64)
    slot = s["indices"] >= 0
    at = s["indices"].clamp(min=0).long()
    logq = s["logits"].gather(1, at).double() / tau - (torch.log(total) + top.double())
    t = torch.where(slot, s["teacher"].double() / tau, -math.inf)
    high = t.amax(1, keepdim=True)
    logp = t - (s["lse"].double()[:, None] if c["tail"] else high + torch.log(torch.exp(t - high).sum(1, keepdim=True)))
    p = torch.exp(logp)
    used = (w != 0) & slot.any(1)
    kl = torch.where(used, torch.where(p > 0, p * (logp - logq), 0.0).sum(1), 0.0)
    out = {"loss": (tau * tau * (w.double() * kl).sum()).float(), "kl": kl.float()}
    if c["train"]:
        coef = (w * tau)[:, None]
        grad = e * (coef * p.sum(1, keepdim=True).float() / total.float())
        grad.scatter_add_(1, at, -coef * p.float())
        out["dlogits"] = torch.where(used[:, None], grad, 0.0).to(s["logits"].dtype)
    return out


# ---- what a pass cannot do without -----------------------------------------------------------------------------------


def work(case):
    kind, size = case["kind"], 4 if case["dtype"] == "fp32" else 2
    if kind in ("delta", "step"):
        B, T, Hk, Hv, dk, dv = (case[n] for n in ("B", "T", "Hk", "Hv", "dk", "dv"))
        qk, v, scalars, state = 2 * B * T * Hk * dk * size, B * T * Hv * dv * size, 8 * B * T * Hv, 4 * B * Hv * dk * dv
        products = B * T * Hv * dk * dv            # a token's products of a vector and a state, two operations each
        if kind == "step":
            return {"bytes": qk + 2 * v + scalars + 2 * state, "flops": 7 * products}
        forward = qk + 2 * v + scalars + (2 if case["state"] else 1) * state
        if not case["train"]:
            return {"bytes": forward, "flops": 7 * products}
        return {"bytes": forward + 2 * qk + 3 * v + 2 * scalars + (3 if case["state"] else 1) * state, "flops": 28 * products}
    if kind == "norm":
        n = case["rows"] * case["cols"]
        passes = (4 if case["residual"] else 2) + ((4 if case["residual"] else 3) if case["train"] else 0)
        return {"bytes": n * size * passes + 8 * case["rows"], "flops": n * (20 if case["train"] else 8)}
    rows, read = case["rows"], case["rows"] * (1 - case["unused"])
    written = rows if case["train"] else 0
    return {"bytes": (read + written) * case["vocab"] * size + 8 * read * case["top"] + 8 * rows, "flops": (read + written) * case["vocab"] * 5}


# ---- the same from the definitions, in 64 bits -----------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"delta": _exact_delta, "step": _exact_step, "norm": _exact_norm, "distill": _exact_distill}[case["kind"]](s)


def _advance(S, k, v, a, b):
    """One token: the state, what was put into it, and the state before that."""
    kept = S * a[..., None, None]
    u = b[..., None] * (v - torch.einsum("bhkv,bhk->bhv", kept, k))
    return kept + k.unsqueeze(-1) * u.unsqueeze(-2), u, kept


def _exact_step(s):
    rep = s["case"]["Hv"] // s["case"]["Hk"]
    q, k = (torch.repeat_interleave(s[n].double(), rep, dim=2) for n in ("q", "k"))
    S, outs = s["state"].double(), []
    for t in range(s["case"]["T"]):
        S, _, _ = _advance(S, k[:, t], s["v"][:, t].double(), s["g"][:, t].double().exp(), s["beta"][:, t].double())
        outs.append(s["scale"] * torch.einsum("bhkv,bhk->bhv", S, q[:, t]))
    return {"o": torch.stack(outs, 1), "state": S}


def _exact_delta(s):
    """Token by token; the gradients by walking back, the states of 64 tokens at a time formed again."""
    c = s["case"]
    B, T, Hk, Hv, dk, dv = (c[n] for n in ("B", "T", "Hk", "Hv", "dk", "dv"))
    rep = Hv // Hk
    q, k = (torch.repeat_interleave(s[n].double(), rep, dim=2) for n in ("q", "k"))
    v, a, b = s["v"].double(), s["g"].double().exp(), s["beta"].double()
    S = s["state"].double() if c["state"] else torch.zeros(B, Hv, dk, dv, dtype=F64, device="cuda")
    outs, marks = [], []
    for t in range(T):
        if t % 64 == 0:
            marks.append(S)
        S, _, _ = _advance(S, k[:, t], v[:, t], a[:, t], b[:, t])
        outs.append(s["scale"] * torch.einsum("bhkv,bhk->bhv", S, q[:, t]))
    out = {"o": torch.stack(outs, 1), "state": S}
    if not c["train"]:
        return out
    dS, do = s["dstate"].double(), s["do"].double()
    grads = {n: torch.zeros_like(x) for n, x in (("dq", q), ("dk", k), ("dv", v), ("dg", a), ("dbeta", b))}
    for m in reversed(range(len(marks))):
        S, steps = marks[m], []
        for t in range(64 * m, min(T, 64 * m + 64)):
            before = S
            S, u, kept = _advance(S, k[:, t], v[:, t], a[:, t], b[:, t])
            steps.append((t, before, S, u, kept))
        for t, before, after, u, kept in reversed(steps):
            grads["dq"][:, t] = s["scale"] * torch.einsum("bhkv,bhv->bhk", after, do[:, t])
            dS = dS + s["scale"] * q[:, t].unsqueeze(-1) * do[:, t].unsqueeze(-2)
            du = torch.einsum("bhkv,bhk->bhv", dS, k[:, t])
            dw = b[:, t].unsqueeze(-1) * du                                 # by what u is beta times of
            grads["dv"][:, t] = dw
            grads["dbeta"][:, t] = (du * (v[:, t] - torch.einsum("bhkv,bhk->bhv", kept, k[:, t]))).sum(-1)
            grads["dk"][:, t] = torch.einsum("bhkv,bhv->bhk", dS, u) - torch.einsum("bhkv,bhv->bhk", kept, dw)
            dkept = dS - k[:, t].unsqueeze(-1) * dw.unsqueeze(-2)
            grads["dg"][:, t] = a[:, t] * (dkept * before).sum((-1, -2))
            dS = dkept * a[:, t][..., None, None]
    for n in ("dq", "dk"):
        grads[n] = grads[n].unflatten(2, (Hk, rep)).sum(3)
    out.update(grads)
    if c["state"]:
        out["dstate"] = dS
    return out


def _exact_norm(s):
    """y by torch's own variance, its gradients by differentiating that; h is rounded before the norm sees it."""
    c = s["case"]
    h = s["x"].double() + s["residual"].double() if c["residual"] else s["x"].double()
    x = h.to(s["x"].dtype).double().requires_grad_()
    w = s["w"].double().requires_grad_()
    b = (s["b"].double() if c["bias"] else torch.zeros_like(w)).detach().requires_grad_()
    var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
    y = torch.addcmul(b, (x - mean) / (var + EPS).sqrt(), w)
    out = {"y": y.detach(), "mean": mean.detach()[:, 0], "rstd": (1.0 / (var + EPS).sqrt()).detach()[:, 0]}
    if c["residual"]:
        out["h"] = h
    if c["train"]:
        dx, out["dw"], out["db"] = torch.autograd.grad(y, [x, w, b], s["dy"].double())
        out["dx"] = dx + s["dh"].double() if c["residual"] else dx
    return out


def _exact_distill(s):
    """The loss by log_softmax, differentiated, some rows at a time."""
    c = s["case"]
    tau, kls, grads = c["tau"], [], []
    for r in torch.arange(c["rows"], device="cuda").split(512):
        z = s["logits"][r].double().requires_grad_()
        i, w = s["indices"][r].long(), s["weights"][r].double()
        logq = torch.log_softmax(z / tau, 1)
        p = torch.zeros_like(logq.detach())
        row, slot = (i >= 0).nonzero(as_tuple=True)
        t = torch.full_like(i, -math.inf, dtype=F64)
        t[row, slot] = s["teacher"][r].double()[row, slot] / tau
        p[row, i[row, slot]] = torch.exp(t - s["lse"][r].double()[:, None] if c["tail"] else torch.log_softmax(t, 1))[row, slot]
        counts = (w != 0) & (i >= 0).any(1)
        kl = torch.where(counts, (torch.special.xlogy(p, p) - p * logq).sum(1), 0.0)
        kls.append(kl.detach())
        if c["train"]:
            grads.append(torch.autograd.grad((tau * tau * w * kl).sum(), z)[0].to(F32))
    kl = torch.cat(kls)
    out = {"loss": tau * tau * (kl * s["weights"].double()).sum(), "kl": kl}
    if c["train"]:
        out["dlogits"] = torch.cat(grads)
    return out
