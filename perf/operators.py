"""The operators that training past the first language-model loss adds to this framework, as cases with inputs, one pass and its useful work.

Four places of one training step: queries and keys normalised head by head and turned by their positions on the way into attention
(`ops.qk_norm_rope_fwd` / `_bwd`), the log-probabilities of chosen tokens (`ops.token_logprobs_fwd` / `_bwd`), the losses that are built on them
(`blockops.policy_loss`, `blockops.preference_loss`), and the optimiser over all parameters at once (`blockops.adamw_many_`).
Sizes are those of the framework's own models and benchmarks: the 35 M parameter Llama (6 layers, d = 512, 32000 words, 8 x 1024 tokens), grouped
queries of a half-billion-parameter model (14 heads to 2, head size 64, 4 x 2048 tokens), 16 heads of 128 over 4 x 4096 tokens.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
BLOCK = 256            # elements of an 8-bit state that share a scale
F32 = torch.float32


def _f32(x):
    """A number as the operators hold it: rounded to 32 bits."""
    return float(torch.tensor(x, dtype=F32))


# ---- cases -----------------------------------------------------------------------------------------------------------


def _qk(name, B, T, Hq, Hkv, dk, dtype, train, halves=False, rotary=0, far=0, theta=10000.0):
    """train: forward and backward. rotary: columns of a head that are turned, 0 = all. far: the first token's position is drawn up to there."""
    return {"name": name, "kind": "qk", "B": B, "T": T, "Hq": Hq, "Hkv": Hkv, "dk": dk, "dtype": dtype, "train": train, "halves": halves,
            "rotary": rotary, "far": far, "theta": theta}


def _logprobs(name, rows, vocab, dtype, train, scale=1.0):
    return {"name": name, "kind": "logprobs", "rows": rows, "vocab": vocab, "dtype": dtype, "train": train, "scale": scale}


def _policy(name, rows, vocab, dtype, kl, unused, scale=1.0, forbidden=0):
    """unused: share of rows whose weight is zero (padding, prompts). forbidden: last words of the vocabulary whose logit is -inf."""
    return {"name": name, "kind": "policy", "rows": rows, "vocab": vocab, "dtype": dtype, "kl": kl, "unused": unused, "scale": scale,
            "forbidden": forbidden}


def _preference(name, pairs, length, vocab, dtype, prompt, behind=0, smoothing=0.0):
    """Sequences of length/2 to length tokens, the share `prompt` of each of them the prompt's; `behind` rows of padding after the last one."""
    return {"name": name, "kind": "preference", "pairs": pairs, "length": length, "vocab": vocab, "dtype": dtype, "prompt": prompt,
            "behind": behind, "smoothing": smoothing}


def _adamw(name, bits, grads, clip, copies, layers=0, d=0, d_ff=0, vocab=0, tensors=0, most=0):
    """The parameters of a Llama, or `tensors` ragged ones of up to `most` elements. copies: a bf16 copy of each is written along."""
    return {"name": name, "kind": "adamw", "bits": bits, "grads": grads, "clip": clip, "copies": copies, "layers": layers, "d": d, "d_ff": d_ff,
            "vocab": vocab, "tensors": tensors, "most": most}


def listed():
    return [
        # One new token of each of 64 sequences that are being generated, at positions of their own: latency.
        _qk("qk_decode", 64, 1, 14, 2, 64, "bf16", False, far=30000, theta=1e6),
        # Grouped-query attention of a half-billion-parameter model in training, heads read in the fused projection.
        _qk("qk_train_gqa", 4, 2048, 14, 2, 64, "bf16", True),
        # Long-context training, 16 heads of 128, rotation of halves.
        _qk("qk_train_long", 4, 4096, 16, 16, 128, "bf16", True, halves=True, theta=1e6),
        # Full precision, a head size between the usual ones of which only a part is turned, an odd number of tokens, far positions.
        _qk("qk_odd_fp32", 3, 1021, 6, 3, 80, "fp32", True, rotary=48, far=900000),
        # Scoring a batch of answers with the reference model: forward only, full precision, a vocabulary of odd size.
        _logprobs("logprobs_score", 1000, 32003, "fp32", False),
        # The same for training on a loss of the program's own.
        _logprobs("logprobs_train", 8192, 32000, "bf16", True),
        # A small policy step in full precision at a sampling temperature, odd vocabulary, words that a grammar forbids.
        _policy("policy_small", 250, 32003, "fp32", 0.05, 0.3, scale=1.25, forbidden=3),
        # A policy step over the 35 M parameter model's batch, a quarter of it padding.
        _policy("policy_step", 8192, 32000, "bf16", 0.04, 0.25),
        # Three ragged pairs of short answers with padding behind them.
        _preference("preference_small", 3, 61, 10007, "fp32", 0.3, behind=17, smoothing=0.1),
        # Four pairs of 512 to 1024 tokens on the 35 M parameter model's vocabulary.
        _preference("preference_step", 4, 1024, 32000, "bf16", 0.25),
        # Adapters and norms: many small ragged tensors, the gradients in bf16, 32-bit states, no clip. Latency and raggedness.
        _adamw("adamw_ragged", 32, "bf16", 0.0, False, tensors=96, most=60000),
        # The 35 M parameter model with 8-bit states, global-norm clip and the bf16 copies that its products read.
        _adamw("adamw_35m_8bit", 8, "fp32", 1.0, True, layers=6, d=512, d_ff=1376, vocab=32000),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["qk", "logprobs", "policy", "preference", "adamw"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if kind == "qk":
        dk = rng.choice([32, 64, 64, 80, 96, 128, 128, 256, 2 * rng.randint(1, 128)])
        Hkv, rep, halves = rng.randint(1, 8), rng.choice([1, 2, 4, 7]), rng.random() < 0.5
        rotary = 0 if rng.random() < 0.7 else 2 * rng.randint(1, dk // 2)
        train = rng.random() < 0.7
        T = _log_uniform(rng, 1, 4096)
        most = 4 * 4096 * 32 * 128 // (2 if dtype == "fp32" else 1)
        B = max(1, min(most // (T * Hkv * (rep + 1) * dk), _log_uniform(rng, 1, 64)))
        return _qk(None, B, T, Hkv * rep, Hkv, dk, dtype, train, halves, rotary, rng.choice([0, 0, 30000, 900000]), rng.choice([10000.0, 1e6]))
    if kind == "preference":
        vocab, pairs = _log_uniform(rng, 50, 60000), rng.randint(1, 8)
        length = max(1, min(_log_uniform(rng, 1, 1024), 8192 * 16000 // (2 * pairs * vocab)))
        return _preference(None, pairs, length, vocab, dtype, rng.choice([0.0, 0.25, 0.6]), rng.choice([0, 0, 5]), rng.choice([0.0, 0.1]))
    if kind == "adamw":
        bits, grads, clip, copies = rng.choice([8, 32]), rng.choice(["fp32", "bf16"]), rng.choice([0.0, 1.0]), rng.random() < 0.5
        if rng.random() < 0.5:
            return _adamw(None, bits, grads, clip, copies, tensors=_log_uniform(rng, 1, 300), most=_log_uniform(rng, 1, 100000))
        d = 8 * rng.randint(4, 64)
        return _adamw(None, bits, grads, clip, copies, rng.randint(1, 6), d, _log_uniform(rng, d, 3 * d), _log_uniform(rng, 500, 30000))
    vocab = _log_uniform(rng, 50, 150000)
    rows = max(1, min(_log_uniform(rng, 1, 8192), 8192 * 16000 // vocab))
    if kind == "logprobs":
        return _logprobs(None, rows, vocab, dtype, rng.random() < 0.6, rng.choice([1.0, 1.0, 1.25]))
    return _policy(None, rows, vocab, dtype, rng.choice([0.0, 0.04]), rng.choice([0.0, 0.25]), rng.choice([1.0, 0.8]), rng.choice([0, 3]))


# ---- inputs ----------------------------------------------------------------------------------------------------------


def _lengths(case):
    """The sequences' lengths, chosen ones first: the case's own, the same for every seed."""
    rng = random.Random(case["pairs"] * 7919 + case["length"])
    return [rng.randint(max(1, case["length"] // 2), case["length"]) for _ in range(2 * case["pairs"])]


def _shapes(case):
    if case["tensors"]:
        rng = random.Random(case["tensors"] * 7919 + case["most"])
        return [(_log_uniform(rng, 1, case["most"]),) for _ in range(case["tensors"])]
    d, ff = case["d"], case["d_ff"]
    block = [(d,), (d, d), (d, d), (d, d), (d, d), (d,), (d, ff), (d, ff), (ff, d)]
    return [(case["vocab"], d)] + block * case["layers"] + [(d,)]


def _rows_of(case):
    return sum(_lengths(case)) + case["behind"] if case["kind"] == "preference" else case["rows"]


def _prompts(case):
    """For each sequence (its first row, its first answer's row, its end)."""
    at, out = 0, []
    for n in _lengths(case):
        out.append((at, at + int(n * case["prompt"]), at + n))
        at += n
    return out


def _logits(case, gen):
    """Logits of a model that gives the token which was sampled a few per cent of the mass and more; the tokens; their log-probability in 64 bits."""
    rows, vocab, dtype = _rows_of(case), case["vocab"], DTYPES[case["dtype"]]
    x = torch.randn((rows, vocab), generator=gen, device="cuda").mul_(2.0)
    if case.get("forbidden"):
        x[:, vocab - case["forbidden"]:] = -math.inf
    t = torch.randint(0, max(1, vocab - case.get("forbidden", 0)), (rows,), generator=gen, device="cuda")
    at = torch.arange(rows, device="cuda")
    x[at, t] += torch.rand(rows, generator=gen, device="cuda") * 12.0
    x = x.to(dtype)
    scale = case.get("scale", 1.0)
    logp = torch.cat([r.double().mul_(scale).log_softmax(1).gather(1, i[:, None])[:, 0] for r, i in zip(x.split(512), t.split(512))])
    return x, t.to(torch.int32), logp


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    rand = lambda *s: torch.rand(s, generator=gen, device="cuda")        # noqa: E731
    randn = lambda *s: torch.randn(s, generator=gen, device="cuda")      # noqa: E731
    s = {"case": case}
    if kind == "qk":
        B, T, Hq, Hkv, dk, dtype = case["B"], case["T"], case["Hq"], case["Hkv"], case["dk"], DTYPES[case["dtype"]]
        qkv = randn(B, T, Hq + 2 * Hkv, dk).mul_(torch.exp(0.5 * randn(1, 1, Hq + 2 * Hkv, 1))).to(dtype)   # the fused projection, heads of different sizes
        s["q"], s["k"] = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hkv]
        s["wq"], s["wk"] = 1.0 + 0.2 * randn(dk), 1.0 + 0.2 * randn(dk)
        first = (rand(B, 1) * case["far"]).to(torch.int32)
        s["pos"] = (first + torch.arange(T, device="cuda", dtype=torch.int32)).contiguous()
        if case["train"]:
            s["dyq"], s["dyk"] = randn(B, T, Hq, dk).to(dtype), randn(B, T, Hkv, dk).to(dtype)
    elif kind in ("logprobs", "policy", "preference"):
        s["logits"], s["targets"], logp = _logits(case, gen)
        rows = logp.numel()
        if kind == "logprobs":
            s["dlogp"] = randn(rows) / rows
        elif kind == "policy":
            # The policy has moved away from the one that sampled. No ratio lies within 1e-4 of where the clip begins: which side such a row is on is
            # decided by the last bits of its sum, and its gradient is there or not.
            drift = 0.15 * randn(rows).double()
            for edge in (math.log(0.8), math.log(1.2)):
                near = drift - edge
                drift = torch.where(near.abs() < 1e-4, drift + 2e-4, drift)
            s["old"] = (logp - drift).to(F32)
            s["ref"] = (logp + 0.1 * randn(rows)).to(F32)
            s["adv"] = randn(rows)
            used = (rand(rows) >= case["unused"]).to(F32)
            s["weights"] = used / used.sum().clamp(min=1.0)
        else:
            s["ref"] = (logp + 0.3 * randn(rows)).to(F32)
            ends = [0]
            for _, answer, end in (p := _prompts(case)):
                ends.append(end)
            for begin, answer, _ in p:
                s["targets"][begin:answer] = -1
            s["targets"][ends[-1]:] = -1
            s["starts"] = torch.tensor(ends, dtype=torch.int32, device="cuda")
    else:
        # Parameters, gradients, states and copies lie in slabs, as this framework's models keep theirs, every tensor at the beginning of a block.
        s["t"], shapes = 1000, _shapes(case)
        counts = [math.prod(x) for x in shapes]
        room = [-(-n // BLOCK) * BLOCK for n in counts]
        s["counts"], s["room"] = torch.tensor(counts, device="cuda"), torch.tensor(room, device="cuda")
        for name in ("p", "g", "m", "v"):
            s[name] = torch.zeros(sum(room), device="cuda")
        at = 0
        for shape, n, more in zip(shapes, counts, room):
            size = 1e-3 * math.exp(float(torch.randn((), generator=torch.Generator().manual_seed(seed + at))))
            g = randn(n) * torch.exp(randn(n)) * size   # spread over orders of magnitude, as gradients are
            s["p"][at:at + n], s["g"][at:at + n] = 0.02 * randn(n), g
            s["m"][at:at + n], s["v"][at:at + n] = 0.3 * size * randn(n), g.square() * torch.exp(0.5 * randn(n))
            at += more
        s["g"] = s["g"].to(DTYPES[case["grads"]])
        if case["bits"] == 8:
            half = torch.full((), 1 << 15, dtype=torch.int64, device="cuda")
            (s["m"], s["m_scale"]), (s["v"], s["v_scale"]) = _pack(s["m"], half, False), _pack(s["v"], half, True)
        if case["copies"]:
            s["copies"] = s["p"].to(torch.bfloat16)
        begins = [sum(room[:i]) for i in range(len(room))]
        for name in ("p", "g", "m", "v", "copies"):
            if name in s:
                s[name + "_of"] = [s[name][b:b + n].view(shape) for b, n, shape in zip(begins, counts, shapes)]
        for name in ("m_scale", "v_scale"):
            if name in s:
                s[name + "_of"] = [s[name][b // BLOCK:(b + r) // BLOCK] for b, r in zip(begins, room)]
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------

LR, B1, B2, EPS, WD = (_f32(x) for x in (3e-4, 0.9, 0.95, 1e-8, 0.1))


def run(s):
    return {"qk": _run_qk, "logprobs": _run_logprobs, "policy": _run_policy, "preference": _run_preference, "adamw": _run_adamw}[s["case"]["kind"]](s)


def _turn(x, c, s, halves, rotary):
    """The first `rotary` columns turned pair by pair."""
    y = x.clone()
    a, b = (x[..., :rotary // 2], x[..., rotary // 2:rotary]) if halves else (x[..., 0:rotary:2], x[..., 1:rotary:2])
    if halves:
        y[..., :rotary // 2], y[..., rotary // 2:rotary] = a * c - b * s, a * s + b * c
    else:
        y[..., 0:rotary:2], y[..., 1:rotary:2] = a * c - b * s, a * s + b * c
    return y


def _run_qk(s):
    c = s["case"]
    if own:
        from paperkiln_amd import ops
        yq, yk = ops.qk_norm_rope_fwd(s["q"], s["k"], s["wq"], s["wk"], s["pos"], c["theta"], 1e-5, c["rotary"], c["halves"])
        if not c["train"]:
            return {"yq": yq, "yk": yk}
        dq, dk, dwq, dwk = ops.qk_norm_rope_bwd(s["dyq"], s["dyk"], s["q"], s["k"], s["wq"], s["wk"], s["pos"], c["theta"], 1e-5, c["rotary"], c["halves"])
        return {"yq": yq, "yk": yk, "dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}
    rotary = c["rotary"] or c["dk"]
    freq = c["theta"] ** (-torch.arange(0, rotary, 2, device="cuda", dtype=torch.float64) / rotary)
    angle = s["pos"].double()[:, :, None, None] * freq
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    out = {}
    for n in ("q", "k"):
        x, w = s[n].float(), s["w" + n]
        r = 1.0 / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-5)
        out["y" + n] = _turn(x * r * w, cos, sin, c["halves"], rotary).to(s[n].dtype)
        if c["train"]:
            du = _turn(s["dy" + n].float(), cos, -sin, c["halves"], rotary)
            out["dw" + n] = (du * x * r).sum((0, 1, 2))
            wdu = du * w
            out["d" + n] = (r * (wdu - x * r * r * (wdu * x).mean(-1, keepdim=True))).to(s[n].dtype)
    return out


def _rows(logits, targets, scale):
    """For each row: scale * logits in 32 bits, the log of its sum of exponentials and its token's log-probability in 64 (a difference of near numbers)."""
    z = logits.float() * scale
    top = z.amax(1, keepdim=True)
    lse = torch.log(torch.exp(z - top).sum(1, dtype=torch.float64)) + top[:, 0].double()
    return z, lse, z.gather(1, targets.clamp(min=0).long()[:, None])[:, 0].double() - lse


def _gradient(z, lse, targets, coef, dtype):
    """coef * ([j = target] - softmax), where coef is not zero."""
    g = torch.exp(z - lse.float()[:, None]).mul_(-coef[:, None])
    g.scatter_add_(1, targets.clamp(min=0).long()[:, None], coef[:, None])
    return torch.where(coef[:, None] != 0, g, 0.0).to(dtype)


def _run_logprobs(s):
    c = s["case"]
    if own:
        from paperkiln_amd import ops
        logp, lse = ops.token_logprobs_fwd(s["logits"], s["targets"], c["scale"])
        if not c["train"]:
            return {"logp": logp, "lse": lse}
        return {"logp": logp, "lse": lse, "dlogits": ops.token_logprobs_bwd(s["logits"], s["targets"], lse, s["dlogp"], c["scale"])}
    z, lse, logp = _rows(s["logits"], s["targets"], c["scale"])
    if not c["train"]:
        return {"logp": logp.float(), "lse": lse.float()}
    return {"logp": logp.float(), "lse": lse.float(), "dlogits": _gradient(z, lse, s["targets"], s["dlogp"] * c["scale"], s["logits"].dtype)}


def _run_policy(s):
    c = s["case"]
    if own:
        from paperkiln_amd import blockops
        loss, dlogits, logp = blockops.policy_loss(s["logits"], s["targets"], s["old"], s["adv"], s["weights"], clip_low=0.2, clip_high=0.2,
                                                   ref_logp=s["ref"] if c["kl"] else None, kl_coef=c["kl"], scale=c["scale"])
        return {"loss": loss, "dlogits": dlogits, "logp": logp}
    z, lse, logp = _rows(s["logits"], s["targets"], c["scale"])
    used, adv = s["weights"] != 0, s["adv"].double()
    ratio = torch.exp(logp - s["old"].double())
    free, held = ratio * adv, ratio.clamp(1.0 - _f32(0.2), 1.0 + _f32(0.2)) * adv
    each, slope = -torch.minimum(free, held), torch.where(free <= held, -free, 0.0)
    if c["kl"]:
        apart = s["ref"].double() - logp
        each = each + c["kl"] * (torch.exp(apart) - apart - 1.0)
        slope = slope + c["kl"] * (1.0 - torch.exp(apart))
    w = s["weights"].double()
    coef = torch.where(used, w * slope * c["scale"], 0.0).float()
    return {"loss": torch.where(used, w * each, 0.0).sum().float(), "dlogits": _gradient(z, lse, s["targets"], coef, s["logits"].dtype),
            "logp": torch.where(used, logp, 0.0).float()}


BETA = _f32(0.1)


def _run_preference(s):
    c = s["case"]
    if own:
        from paperkiln_amd import blockops
        loss, dlogits, margins, logp = blockops.preference_loss(s["logits"], s["targets"], s["starts"], s["ref"], beta=BETA, label_smoothing=c["smoothing"])
        return {"loss": loss, "dlogits": dlogits, "margins": margins, "logp": logp}
    z, lse, logp = _rows(s["logits"], s["targets"], 1.0)
    used = s["targets"] >= 0
    so_far = torch.cat([torch.zeros(1, dtype=torch.float64, device="cuda"), torch.where(used, logp - s["ref"].double(), 0.0).cumsum(0)])
    begin, end = s["starts"][:-1].long(), s["starts"][1:].long()
    sums = so_far[end] - so_far[begin]
    pairs = c["pairs"]
    margins = BETA * (sums[:pairs] - sums[pairs:])
    e = _f32(c["smoothing"])
    near, far = 1.0 / (1.0 + torch.exp(margins)), 1.0 / (1.0 + torch.exp(-margins))
    loss = ((1.0 - e) * -torch.log(far) + e * -torch.log(near)).mean()
    slope = (e * far - (1.0 - e) * near) * (BETA / pairs)
    row = torch.arange(used.numel(), device="cuda")
    of = torch.bucketize(row, end, right=True)
    coef = torch.where(used & (of < 2 * pairs), torch.cat([slope, -slope, slope.new_zeros(1)])[of], 0.0).float()
    return {"loss": loss.float(), "dlogits": _gradient(z, lse, s["targets"], coef, s["logits"].dtype), "margins": margins.float(),
            "logp": torch.where(used, logp, 0.0).float()}


def _mix(x):
    """The low 32 bits of x scrambled, as whole numbers in 64."""
    low = 0xFFFFFFFF
    x = x & low
    x = x ^ (x >> 16)
    x = (x * 0xBB67AE85) & low
    x = x ^ (x >> 15)
    x = (x * 0x6A09E667) & low
    return x ^ (x >> 16)


def _pack(x, chance, square):
    """A state of whole blocks in 8 bits and its blocks' scales. square: e5m2 for the (nonnegative) mean square, else e4m3 for the mean. `chance`: 16
    random bits of each element; the bits below the last kept one are rounded up with the probability that they stand for. A scale is the
    power of two that puts its block's largest value just under the format's largest, so that scaling rounds nothing; a block that holds a value
    which is not finite is all NaN; a mean square that is not zero does not become zero."""
    top, drop, bias, kind = (15, 21, 112, torch.float8_e5m2) if square else (8, 20, 120, torch.float8_e4m3fn)
    most = x.view(-1, BLOCK).abs().amax(1)
    fine = torch.isfinite(most)
    part, power = torch.frexp(torch.where(fine & (most > 0), most, 1.0))
    power = torch.where(most == 0, -126, power - 1 - top + (part > 0.875).int()).clamp(min=-126)
    one = torch.ones_like(most)
    y = (x.view(-1, BLOCK) * torch.ldexp(one, -power)[:, None]).view(-1)
    bits = (y.abs() * 2.0 ** -bias).view(torch.int32).long()
    bits = (bits + (chance << (drop - 16)) + (1 << (drop - 17))) >> drop
    bits = torch.maximum(bits, (x > 0).long()) if square else bits | (torch.signbit(y).long() << 7)
    bits = torch.where(fine[:, None], bits.view(-1, BLOCK), 0x7F).view(-1)
    return bits.to(torch.uint8).view(kind), torch.where(fine, torch.ldexp(one, power), math.nan)


def _unpack(x, scale):
    """A state's values in 32 bits."""
    return (x.float().view(-1, BLOCK) * scale[:, None]).view(-1)


def _run_adamw(s):
    c = s["case"]
    s["t"] += 1
    bits8, norm = c["bits"] == 8, None
    if own:
        from paperkiln_amd import blockops
        state = blockops.AdamWState(s["m_of"], s["v_of"], s.get("m_scale_of"), s.get("v_scale_of"))
        norm = blockops.adamw_many_(s["p_of"], s["g_of"], state, LR, B1, B2, EPS, WD, t=s["t"], max_norm=c["clip"], copies=s.get("copies_of"), seed=s["t"])
    else:
        g, p = s["g"].float(), s["p"]
        if c["clip"]:
            total = torch.sqrt(g.double().square().sum())
            norm = total.float()
            g = g * torch.where((total > c["clip"]) & (total > 0), c["clip"] / total, 1.0).float()
        m, v = (_unpack(s[n], s[n + "_scale"]) if bits8 else s[n] for n in ("m", "v"))
        m = m * B1 + g * _f32(1.0 - B1)
        v = v * B2 + (g * _f32(1.0 - B2)) * g
        p.sub_(LR * ((m / (1.0 - B1 ** s["t"])) / (torch.sqrt(v / (1.0 - B2 ** s["t"])) + EPS) + WD * p))
        if bits8:
            which = torch.arange(len(s["room"]), device="cuda")
            key = _mix(s["t"] * 0x9E3779B9 + _mix(which + 0x3C6EF373))
            inside = torch.arange(p.numel(), device="cuda") - torch.repeat_interleave(s["room"].cumsum(0) - s["room"], s["room"], output_size=p.numel())
            h = _mix(inside ^ torch.repeat_interleave(key, s["room"], output_size=p.numel()))
            for n, x, chance in (("m", m, h & 0xFFFF), ("v", v, h >> 16)):
                code, scale = _pack(x, chance, n == "v")
                s[n].view(torch.uint8).copy_(code.view(torch.uint8))
                s[n + "_scale"].copy_(scale)
        else:
            s["m"].copy_(m)
            s["v"].copy_(v)
        if c["copies"]:
            s["copies"].copy_(p)
    out = {n: s[n] for n in ("p", "m", "v", "m_scale", "v_scale", "copies") if n in s}
    return out if norm is None else {**out, "norm": norm}


# ---- what a pass cannot do without -----------------------------------------------------------------------------------


def work(case):
    kind, size = case["kind"], 4 if case.get("dtype") == "fp32" else 2
    if kind == "qk":
        n = case["B"] * case["T"] * (case["Hq"] + case["Hkv"]) * case["dk"]
        return {"bytes": n * size * (4 if case["train"] else 2) + 4 * case["B"] * case["T"], "flops": n * (24 if case["train"] else 8)}
    if kind == "adamw":
        n = sum(math.prod(x) for x in _shapes(case))
        state = 2 * (2 + 8 / BLOCK) if case["bits"] == 8 else 16
        return {"bytes": n * (8 + (4 if case["grads"] == "fp32" else 2) + state + (2 if case["copies"] else 0)), "flops": n * 20}
    rows = _rows_of(case)
    read = {"logprobs": rows, "policy": rows * (1 - case.get("unused", 0)), "preference": sum(e - a for _, a, e in _prompts(case)) if kind == "preference" else 0}[kind]
    written = rows if kind != "logprobs" or case["train"] else 0
    return {"bytes": (read + written) * case["vocab"] * size + 24 * rows, "flops": (read + written) * case["vocab"] * 5}


# ---- the same from the definitions, in 64 bits -----------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"qk": _exact_qk, "logprobs": _exact_rows, "policy": _exact_rows, "preference": _exact_rows, "adamw": _exact_adamw}[case["kind"]](s)


def _exact_qk(s):
    """y as a product of complex numbers; the gradients by differentiating that."""
    c = s["case"]
    half = (c["rotary"] or c["dk"]) // 2
    power = torch.arange(half, device="cuda", dtype=torch.float64) / half
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), s["pos"].double().unsqueeze(-1) * torch.exp(-math.log(c["theta"]) * power)).unsqueeze(2)
    out = {}
    for n in ("q", "k"):
        x, w = s[n].double().requires_grad_(), s["w" + n].double().requires_grad_()
        u = x / torch.sqrt((x * x).sum(-1, keepdim=True) / c["dk"] + 1e-5) * w
        first = u[..., :2 * half]
        pairs = first.unflatten(-1, (2, half)).transpose(-1, -2) if c["halves"] else first.unflatten(-1, (half, 2))
        turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        turned = (turned.transpose(-1, -2) if c["halves"] else turned).flatten(-2)
        y = torch.cat([turned, u[..., 2 * half:]], -1)
        out["y" + n] = y.detach()
        if c["train"]:
            out["d" + n], out["dw" + n] = torch.autograd.grad(y, [x, w], s["dy" + n].double())
    return out


def _exact_rows(s):
    """The loss as a function of the rows' log-probabilities, differentiated there; the softmax's own gradient row block by row block."""
    c, kind = s["case"], s["case"]["kind"]
    scale, t = c.get("scale", 1.0), s["targets"].long()
    used = t >= 0
    parts = s["logits"].split(1024)
    logp = torch.cat([torch.log_softmax(x.double() * scale, 1).gather(1, i.clamp(min=0)[:, None])[:, 0] for x, i in zip(parts, t.split(1024))]).requires_grad_()
    out = {}
    if kind == "logprobs":
        total = (logp * s["dlogp"].double()).sum()
        out["lse"] = torch.cat([torch.logsumexp(x.double() * scale, 1) for x in parts])
    elif kind == "policy":
        used = used & (s["weights"] != 0)
        moved, adv = logp - s["old"].double(), s["adv"].double()
        low, high = math.log1p(-_f32(0.2)), math.log1p(_f32(0.2))
        stopped = ((adv > 0) & (moved > high)) | ((adv < 0) & (moved < low))
        each = -adv * torch.where(stopped, torch.where(adv > 0, 1.0 + _f32(0.2), 1.0 - _f32(0.2)).double(), torch.exp(moved))
        if c["kl"]:
            d = s["ref"].double() - logp
            each = each + c["kl"] * (torch.expm1(d) - d)
        total = (each * s["weights"].double())[used].sum()
    else:
        gain = torch.where(used, logp - s["ref"].double(), 0.0)
        sums = torch.stack([gain[a:b].sum() for a, _, b in _prompts(c)])
        out["margins"] = u = BETA * (sums[:c["pairs"]] - sums[c["pairs"]:])
        e = _f32(c["smoothing"])
        total = torch.nn.functional.softplus(-u).mean() * (1 - e) + torch.nn.functional.softplus(u).mean() * e
    slope, = torch.autograd.grad(total, [logp])
    slope = torch.where(used, slope, 0.0)
    if kind != "logprobs" or c["train"]:
        grads = []
        for x, i, k in zip(parts, t.split(1024), slope.split(1024)):
            p = torch.softmax(x.double() * scale, 1).neg_()
            p[torch.arange(len(i), device="cuda"), i.clamp(min=0)] += 1.0
            grads.append((p * (k * scale)[:, None]).to(F32))
        out["dlogits"] = torch.cat(grads)
    if kind != "logprobs":
        out["loss"] = total.detach()
    out["logp"] = torch.where(used, logp, 0.0).detach()
    return {k: v.detach() for k, v in out.items()}


def _exact_adamw(s):
    """One step from the decoded states, tensor by tensor. What a state becomes in 8 bits has no value in 64: it is drawn, not computed."""
    c, t = s["case"], s["t"] + 1
    norm = math.sqrt(sum(float((g.double() ** 2).sum()) for g in s["g_of"]))
    factor = min(1.0, c["clip"] / norm) if c["clip"] and norm > 0 else 1.0
    out = {n: s[n].double() for n in ("p", "m", "v")}
    at = 0
    for k, (n, room) in enumerate(zip(s["counts"].tolist(), s["room"].tolist())):
        here = slice(at, at + n)
        p, g, m, v = out["p"][here], s["g_of"][k].double().view(-1) * factor, out["m"][here], out["v"][here]
        if c["bits"] == 8:
            block = torch.arange(n, device="cuda") // BLOCK
            m, v = m * s["m_scale_of"][k].double()[block], v * s["v_scale_of"][k].double()[block]
        m, v = torch.lerp(g, m, B1), torch.lerp(g * g, v, B2)
        step = (m / -math.expm1(t * math.log(B1))) * torch.rsqrt(v / -math.expm1(t * math.log(B2))).reciprocal().add(EPS).reciprocal()
        out["p"][here], out["m"][here], out["v"][here] = p * (1.0 - LR * WD) - LR * step, m, v
        at += room
    if c["bits"] == 8:
        out["m"] = out["v"] = None
    if c["copies"]:
        out["copies"] = out["p"]
    return {**out, "norm": torch.tensor(norm, dtype=torch.float64)} if c["clip"] else out
