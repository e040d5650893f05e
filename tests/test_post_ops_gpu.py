"""The post-training operators on the GPU against plain implementations in 64 bits: per-head norms with rotation, token log-probabilities, the policy and
the preference loss, AdamW over many tensors.

Tolerances are counted, u = 2^-24 being half a step of fp32 relative to a value and h half a step of the output's type (u, or 2^-8 for bf16): an
output carries one rounding to its type, h * |value|, and what the 32-bit arithmetic before it adds up to, in u times the largest term that enters
it. The counts stand at each test."""
from __future__ import annotations

import functools
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8}
BF16, FP32, F64 = torch.bfloat16, torch.float32, torch.float64


@pytest.fixture(scope="module")
def pk():
    from paperkiln_amd import _lib, blockops, ops
    _lib.check(_lib.lib().pk_init(0, None, 0))

    class Both:
        pass
    b = Both()
    b.ops, b.blockops, b.lib = ops, blockops, _lib
    return b


def within(name, got, want, tol):
    """got and want agree in where they are not finite, and elsewhere to tol, element by element."""
    got, want, tol = got.double().cpu(), want.double().cpu(), tol.double().cpu() if torch.is_tensor(tol) else torch.tensor(tol, dtype=F64)
    assert got.shape == want.shape, name
    tol = torch.nan_to_num(tol, nan=0.0)   # a count of something that is no number allows nothing
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), name
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), name
    over = ((got - want).abs() / tol.expand_as(want).clamp(min=1e-300))[fine]
    assert over.numel() == 0 or float(over.max()) <= 1.0, f"{name}: {float(over.max()):.3g} times its tolerance"


def same_bits(a, b):
    """Equal, what is no number included."""
    return torch.equal(a, b) or torch.equal(a.view(torch.int16 if a.dtype == BF16 else torch.int32), b.view(torch.int16 if b.dtype == BF16 else torch.int32))


# ---- per-head norms with rotation ----------------------------------------------------------------------------------------


def plain_qk(x, w, pos, theta, eps, rotary, halves):
    """One tensor of heads in 64 bits; x and w may require gradients."""
    dk = x.shape[-1]
    rotary = rotary or dk
    u = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w
    angle = pos.double()[..., None] * theta ** (-torch.arange(0, rotary, 2, dtype=F64, device=x.device) / rotary)
    angle = angle.expand(x.shape[0], x.shape[1], rotary // 2)[:, :, None, :]
    c, s = torch.cos(angle), torch.sin(angle)
    a, b = (u[..., :rotary // 2], u[..., rotary // 2:rotary]) if halves else (u[..., 0:rotary:2], u[..., 1:rotary:2])
    ya, yb = a * c - b * s, a * s + b * c
    y = torch.cat([ya, yb], -1) if halves else torch.stack([ya, yb], -1).flatten(-2)
    return torch.cat([y, u[..., rotary:]], -1)


def qk_inputs(B, T, Hq, Hkv, dk, dtype, seed, layout="fused", pos="rows", far=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    if layout == "fused":       # heads of one projection
        qkv = randn(B, T, Hq + 2 * Hkv, dk).to(dtype)
        q, k = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hkv]
    elif layout == "heads":     # [B, H, T, dk] memory
        q, k = (randn(B, H, T, dk).to(dtype).transpose(1, 2) for H in (Hq, Hkv))
    elif layout == "offset":    # one element past an aligned address, odd pitch
        q, k = (randn(B, T, H, dk + 3).to(dtype)[..., 1:1 + dk] for H in (Hq, Hkv))
    else:
        q, k = (randn(B, T, H, dk).to(dtype) for H in (Hq, Hkv))
    wq, wk = 1 + 0.3 * randn(dk), 1 + 0.3 * randn(dk)
    if pos == "rows":
        p = torch.arange(T, device="cuda", dtype=torch.int32)[None] + torch.arange(B, device="cuda", dtype=torch.int32)[:, None] * 7 + far
    elif pos == "shared":
        p = torch.arange(T, device="cuda", dtype=torch.int32) + far
    else:                       # scattered, negative ones among them
        p = torch.randint(-5000, 5000, (B, T), generator=g, device="cuda").to(torch.int32)
    return q, k, wq, wk, p.contiguous(), randn(B, T, Hq, dk).to(dtype), randn(B, T, Hkv, dk).to(dtype)


QK_CASES = [  # B, T, Hq, Hkv, dk, rotary, halves, layout, pos, far
    (1, 1, 1, 1, 2, 0, False, "plain", "shared", 0), (1, 1, 1, 1, 2, 2, True, "plain", "rows", 9), (2, 1, 14, 2, 64, 0, False, "fused", "rows", 30000),
    (64, 1, 3, 1, 128, 0, True, "fused", "any", 0), (2, 37, 6, 2, 64, 0, True, "heads", "any", 0), (1, 130, 5, 3, 128, 0, False, "fused", "shared", 900000),
    (3, 21, 4, 4, 80, 48, False, "fused", "rows", 100), (3, 21, 4, 4, 80, 48, True, "fused", "rows", 100), (2, 9, 3, 2, 96, 0, True, "plain", "any", 0),
    (2, 9, 3, 2, 96, 90, True, "plain", "any", 0), (2, 9, 3, 2, 96, 90, False, "plain", "any", 0), (1, 33, 2, 1, 256, 0, False, "heads", "rows", 0),
    (1, 33, 2, 1, 256, 128, True, "fused", "rows", 2 ** 31 - 100), (2, 17, 7, 1, 24, 0, False, "fused", "any", 0), (2, 17, 7, 1, 24, 16, True, "offset", "any", 0),
    (1, 40, 3, 3, 64, 0, False, "offset", "rows", 0), (1, 40, 3, 3, 128, 64, True, "offset", "rows", 0), (2, 11, 2, 5, 70, 0, True, "fused", "rows", 0),
    (2, 11, 2, 5, 254, 2, False, "fused", "rows", 0), (1, 700, 16, 16, 32, 0, False, "fused", "rows", 0), (1, 5, 1, 1, 8, 0, True, "plain", "rows", 0),
    (1, 5, 2, 1, 40, 8, False, "plain", "rows", 0), (5, 300, 4, 1, 64, 32, True, "fused", "shared", 0),
    (2, 13, 3, 2, 104, 92, True, "fused", "rows", 50), (2, 13, 3, 2, 8, 2, True, "plain", "any", 50), (2, 13, 3, 2, 8, 4, True, "offset", "any", 50),
    (2, 13, 3, 2, 8, 6, True, "fused", "any", 50), (1, 9, 5, 1, 10, 0, False, "plain", "rows", 3), (1, 9, 5, 1, 10, 10, True, "offset", "rows", 3),
    (1, 9, 5, 1, 14, 6, True, "plain", "rows", 3), (2, 11, 4, 2, 256, 250, True, "fused", "any", 7), (2, 11, 4, 2, 250, 0, True, "offset", "any", 7),
    (2, 11, 4, 2, 248, 234, True, "heads", "any", 7), (3, 40, 2, 2, 66, 2, True, "fused", "rows", 0), (3, 40, 2, 2, 66, 64, False, "heads", "rows", 0),
    (2, 40, 2, 2, 6, 4, True, "fused", "rows", 9), (2, 40, 2, 2, 4, 0, False, "offset", "rows", 9), (2, 700, 8, 2, 100, 52, True, "fused", "rows", 9),
    # tokens enough for a wavefront to take several at a time, sequences that end inside its run
    (3, 6001, 1, 1, 64, 0, False, "fused", "shared", 0), (40, 1031, 4, 1, 32, 16, True, "heads", "any", 9), (5, 2003, 5, 5, 80, 0, True, "plain", "rows", 900000),
    (2, 5003, 8, 2, 72, 40, True, "offset", "any", 3), (9000, 1, 2, 2, 128, 0, False, "plain", "rows", 3), (9000, 1, 2, 2, 128, 0, False, "fused", "shared", 3),
    (4, 2049, 14, 2, 64, 0, False, "fused", "rows", 0), (1, 5000, 1, 1, 200, 64, True, "plain", "any", 0), (3, 6001, 2, 1, 30, 22, True, "offset", "shared", 0),
    (2, 9001, 3, 2, 250, 0, False, "heads", "any", 0), (7000, 3, 1, 2, 16, 6, False, "heads", "shared", 4),
    (1, 1, 4500, 3, 128, 0, True, "plain", "rows", 5), (1, 2, 3, 2100, 256, 0, False, "plain", "rows", 5)]


@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("case", QK_CASES, ids=lambda c: "-".join(map(str, c)))
def test_qk_norm_rope_against_64_bits(pk, case, dtype):
    """y: the sum of dk <= 256 squares is at most 4 terms in a row and a tree of 8 levels, halved by the root: 6 u; mean, eps, root, reciprocal and two
    products: 6 u; the fraction of a turn rounded to 32 bits: pi u of angle; cos and sin 4 u; two products and a sum of two terms: 3 u,
    all of a pair's length, at most sqrt(2) times the row's largest |u_j|: under 32 u of it.
    dx: r (w du - x r^2 mean(w du x)), |mean(w du x) r| at most the largest |w du|: 64 u of r max|w du| (1 + max|x| r).
    dw: one rounding per term added, at most all rows, and 16 u of each term: (rows + 16) u of the terms' magnitudes."""
    B, T, Hq, Hkv, dk, rotary, halves, layout, where, far = case
    theta, eps, h = 10000.0, 1e-5, HALF[dtype]
    q, k, wq, wk, pos, dyq, dyk = qk_inputs(B, T, Hq, Hkv, dk, dtype, 5, layout, where, far)
    kept = [t.clone() for t in (q, k, dyq, dyk)]
    yq, yk = pk.ops.qk_norm_rope_fwd(q, k, wq, wk, pos, theta, eps, rotary, halves)
    dq, dk_, dwq, dwk = pk.ops.qk_norm_rope_bwd(dyq, dyk, q, k, wq, wk, pos, theta, eps, rotary, halves)
    assert all(torch.equal(a, b) for a, b in zip(kept, (q, k, dyq, dyk)))
    for n, x, w, dy, y, dx, dw in (("q", q, wq, dyq, yq, dq, dwq), ("k", k, wk, dyk, yk, dk_, dwk)):
        assert y.dtype == dx.dtype == dtype and y.shape == dx.shape == x.shape and dw.dtype == FP32
        xd, wd = x.double().requires_grad_(), w.double().requires_grad_()
        want = plain_qk(xd, wd, pos, theta, eps, rotary, halves)
        r = torch.rsqrt(xd.detach().square().mean(-1, keepdim=True) + eps)
        top = (xd.detach() * r * wd.detach()).abs().amax(-1, keepdim=True)
        within("y" + n, y, want.detach(), h * want.detach().abs() + 32 * U * top)
        gx, gw = torch.autograd.grad(want, [xd, wd], dy.double())
        du = torch.autograd.grad(plain_qk(xd, wd, pos, theta, eps, rotary, halves), wd, dy.double())[0]  # only for its terms' size below
        assert torch.equal(du, gw)
        size = dy.double().abs().amax(-1, keepdim=True) * 2 ** 0.5
        wtop = wd.detach().abs().max()
        within("d" + n, dx, gx, h * gx.abs() + 64 * U * r * size * wtop * (1 + (xd.detach() * r).abs().amax(-1, keepdim=True)))
        terms = (size * (xd.detach() * r).abs()).sum((0, 1, 2))
        within("dw" + n, dw, gw, (x.shape[0] * T * x.shape[2] + 16) * U * terms)


def dw_terms(x, w, dy, pos, theta, eps, rotary, halves):
    """du x r in 64 bits, element by element: what a column's dw is the sum of."""
    each = w.double().expand(x.shape).clone().requires_grad_()
    return torch.autograd.grad(plain_qk(x.double(), each, pos, theta, eps, rotary, halves), each, dy.double())[0]


def dw_within(name, dw, x, w, dy, pos, rotary, halves):
    """dw by the chain that its additions really are. A lane adds up its rows in turn: those of the tokens that its wavefront takes, a 4096th of them and one more, or fewer where a
    token's heads are dealt out; then come 64 rows of LDS, four loads, trees of 4 and 16 and a store. r, the products and the store's rounding are 16 more, all in u of the
    terms; the turn is 16 u of what a row's pair may be at most, since its parts may cancel. All that is under a hundredth of dw: no part of the
    sum can be missing."""
    terms = dw_terms(x, w, dy, pos, 1e4, 1e-5, rotary, halves)
    tokens, heads = x.shape[0] * x.shape[1], x.shape[2]
    chain = min((-(-tokens // 4096) + 1) * heads, -(-tokens * heads // 256) + 16) + 64 + 4 + 4 + 16
    pair = 2 ** 0.5 * dy.double().abs().amax(-1) * (x.double() * torch.rsqrt(x.double().square().mean(-1, keepdim=True) + 1e-5)).abs().amax(-1)
    want, tol = terms.sum((0, 1, 2)), (chain + 16) * U * terms.abs().sum((0, 1, 2)) + 16 * U * pair.sum()
    assert float(tol.max()) < 0.01 * float(want.square().mean().sqrt()), name
    within(name, dw, want, tol)


@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("case", QK_CASES, ids=lambda c: "-".join(map(str, c)))
def test_qk_norm_rope_weights_gradient(pk, case, dtype):
    B, T, Hq, Hkv, dk, rotary, halves, layout, where, far = case
    q, k, wq, wk, pos, dyq, dyk = qk_inputs(B, T, Hq, Hkv, dk, dtype, 5, layout, where, far)
    _, _, dwq, dwk = pk.ops.qk_norm_rope_bwd(dyq, dyk, q, k, wq, wk, pos, 1e4, 1e-5, rotary, halves)
    dw_within("dwq", dwq, q, wq, dyq, pos, rotary, halves)
    dw_within("dwk", dwk, k, wk, dyk, pos, rotary, halves)


def test_qk_norm_rope_weights_gradient_past_2_to_the_31(pk):
    """Rows that count spread over all of a tensor of more than 2^31 elements, every 1021st token and the last one: one or two to a wavefront. The others' terms are zero and
    round nothing."""
    T, Hq, Hkv, dk = 35000, 480, 2, 128
    g = torch.Generator(device="cuda").manual_seed(8)
    qkv = torch.ones(1, T, Hq + Hkv, dk, dtype=BF16, device="cuda")
    dy = torch.zeros_like(qkv)
    some = torch.cat([torch.arange(0, T, 1021), torch.tensor([T - 1])]).cuda()
    x, d = (torch.randn(1, len(some), Hq + Hkv, dk, generator=g, device="cuda").to(BF16) for _ in range(2))
    qkv[:, some], dy[:, some] = x, d
    w, pos = 1 + 0.2 * torch.randn(dk, generator=g, device="cuda"), torch.arange(T, device="cuda", dtype=torch.int32)
    _, _, dwq, dwk = pk.ops.qk_norm_rope_bwd(dy[:, :, :Hq], dy[:, :, Hq:], qkv[:, :, :Hq], qkv[:, :, Hq:], w, w, pos, 1e4)
    dw_within("dwq", dwq, x[:, :, :Hq], w, d[:, :, :Hq], pos[some], 0, False)
    dw_within("dwk", dwk, x[:, :, Hq:], w, d[:, :, Hq:], pos[some], 0, False)


def test_qk_norm_rope_gradient_against_differences(pk):
    """The derivative of sum(y * dy) along a direction against a central difference of the operator itself in fp32: the difference of two sums of n
    values, each within 32 u of |dy| max|u|, over a step of 2^-6, and the third-order term of the step, below 2^-12 of the sum."""
    q, k, wq, wk, pos, dyq, dyk = qk_inputs(2, 9, 3, 2, 64, FP32, 11, "plain")
    dq, dk, dwq, dwk = pk.ops.qk_norm_rope_bwd(dyq, dyk, q, k, wq, wk, pos, 1e4)
    g = torch.Generator(device="cuda").manual_seed(3)
    dirs = [torch.randn(t.shape, generator=g, device="cuda") for t in (q, k, wq, wk)]
    step = 2.0 ** -6

    def value(s):
        yq, yk = pk.ops.qk_norm_rope_fwd(*(t + s * d for t, d in zip((q, k, wq, wk), dirs)), pos, 1e4)
        return float((yq.double() * dyq.double()).sum() + (yk.double() * dyk.double()).sum()), float((yq.abs() * dyq.abs()).sum() + (yk.abs() * dyk.abs()).sum())

    (up, size), (down, _) = value(step), value(-step)
    slope = sum(float((a.double() * d.double()).sum()) for a, d in zip((dq, dk, dwq, dwk), dirs))
    assert abs((up - down) / (2 * step) - slope) <= (32 * U / step + 2.0 ** -12) * 4 * size


@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("dk,halves", [(64, False), (128, True), (70, True)])
def test_qk_norm_rope_in_place_and_into_views(pk, dtype, dk, halves):
    """y over q and k inside the fused projection, dx into views of a fused gradient and over dy: the bits of the calls into new tensors, nothing else
    in those buffers touched."""
    B, T, Hq, Hkv = 2, 13, 4, 2
    q, k, wq, wk, pos, dyq, dyk = qk_inputs(B, T, Hq, Hkv, dk, dtype, 7)
    yq, yk = pk.ops.qk_norm_rope_fwd(q, k, wq, wk, pos, 1e4, halves=halves)
    want = pk.ops.qk_norm_rope_bwd(dyq, dyk, q, k, wq, wk, pos, 1e4, halves=halves)
    fused = torch.full((B, T, Hq + 2 * Hkv, dk), 3.0, dtype=dtype, device="cuda")
    got = pk.ops.qk_norm_rope_bwd(dyq, dyk, q, k, wq, wk, pos, 1e4, halves=halves, out=(fused[:, :, :Hq], fused[:, :, Hq:Hq + Hkv]))
    assert torch.equal(fused[:, :, :Hq], want[0]) and torch.equal(fused[:, :, Hq:Hq + Hkv], want[1]) and bool((fused[:, :, Hq + Hkv:] == 3.0).all())
    assert torch.equal(got[2], want[2]) and torch.equal(got[3], want[3])
    over = [dyq.clone(), dyk.clone()]
    got = pk.ops.qk_norm_rope_bwd(*over, q, k, wq, wk, pos, 1e4, halves=halves, out=over)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    base = q._base.clone()
    v = base[:, :, Hq + Hkv:].clone()
    pk.ops.qk_norm_rope_fwd(base[:, :, :Hq], base[:, :, Hq:Hq + Hkv], wq, wk, pos, 1e4, halves=halves, out=(base[:, :, :Hq], base[:, :, Hq:Hq + Hkv]))
    assert torch.equal(base[:, :, :Hq], yq) and torch.equal(base[:, :, Hq:Hq + Hkv], yk) and torch.equal(base[:, :, Hq + Hkv:], v)


@pytest.mark.parametrize("layout", ["heads apart", "tokens inside heads", "beside", "other sequences", "other tokens", "every sixth token", "q, k and v of a head", "one token",
                                    "sequences at a pitch of their own"])
def test_qk_norm_rope_into_other_parts_of_the_inputs_buffer(pk, layout):
    """Results, inputs and gradients in parts of one buffer that take turns in it: taken for apart, the bits those of calls into new tensors."""
    B, T, H, dk = 3, 5, 2, 32
    g = torch.Generator(device="cuda").manual_seed(1)
    if layout == "one token":
        B, T = 1, 1
    shape = {"heads apart": (B, T, 6 * H, dk), "tokens inside heads": (B, 6 * H, T, dk), "beside": (6, B, T, H, dk), "other sequences": (6 * B, T, H, dk),
             "other tokens": (B, 6 * T, H, dk), "q, k and v of a head": (B, T, H, 6, dk), "one token": (B, T, H, 6, dk),
             "every sixth token": (B, 6 * T, H, dk), "sequences at a pitch of their own": (B, T * 6 * H * dk + 20)}[layout]
    buffer = torch.randn(shape, generator=g, device="cuda")
    part = {"heads apart": lambda i: buffer[:, :, i * H:(i + 1) * H], "tokens inside heads": lambda i: buffer[:, i * H:(i + 1) * H].transpose(1, 2), "beside": lambda i: buffer[i],
            "other sequences": lambda i: buffer[i::6], "other tokens": lambda i: buffer[:, i * T:(i + 1) * T], "q, k and v of a head": lambda i: buffer[:, :, :, i],
            "one token": lambda i: buffer[:, :, :, i], "every sixth token": lambda i: buffer[:, i::6],
            "sequences at a pitch of their own": lambda i: buffer[:, :-20].unflatten(1, (T, 6 * H, dk))[:, :, i * H:(i + 1) * H]}[layout]
    q, k, dyq, dyk, a, b = (part(i) for i in range(6))
    w, pos = 1 + 0.2 * torch.randn(dk, generator=g, device="cuda"), torch.arange(T, device="cuda", dtype=torch.int32)
    kept = [y.clone() for y in (q, k, dyq, dyk)]
    want = pk.ops.qk_norm_rope_fwd(q, k, w, w, pos, 1e4)
    grad = pk.ops.qk_norm_rope_bwd(dyq, dyk, q, k, w, w, pos, 1e4)
    pk.ops.qk_norm_rope_fwd(q, k, w, w, pos, 1e4, out=(a, b))
    assert torch.equal(a, want[0]) and torch.equal(b, want[1])
    for out in ((a, b), (dyq, dyk), (q, k)):   # the last two write over what they are made of
        for y, x in zip((q, k, dyq, dyk), kept):
            y.copy_(x)
        got = pk.ops.qk_norm_rope_bwd(dyq, dyk, q, k, w, w, pos, 1e4, out=out)
        assert all(torch.equal(y, x) for y, x in zip((*out, *got[2:]), grad))
        assert all(torch.equal(y, x) or y is out[0] or y is out[1] for y, x in zip((q, k, dyq, dyk), kept))
    for y, x in zip((q, k), kept):
        y.copy_(x)
    pk.ops.qk_norm_rope_fwd(q, k, w, w, pos, 1e4, out=(q, k))
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


@pytest.mark.parametrize("pitch", [2 ** 24, 2 ** 24 + 8, 2 ** 24 + 1])
@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
def test_qk_norm_rope_of_heads_far_apart(pk, dtype, pitch):
    """Heads at the largest distance that the row kernels take, past it and off the pieces, as of [B, H, T, dk] memory for very many tokens: what a dense copy gives, each within the counts of
    the test against 64 bits, and both written back at such a distance."""
    T, Hq, Hkv, dk = 5, 5, 3, 64
    far = torch.zeros(2 * (Hq + Hkv) * pitch, dtype=dtype, device="cuda")
    view = lambda first, H: far[first * pitch:].as_strided((1, T, H, dk), (0, dk, pitch, 1))  # noqa: E731
    q, k, wq, wk, pos, dyq, dyk = qk_inputs(1, T, Hq, Hkv, dk, dtype, 6, "plain")
    fq, fk, yq, yk = view(0, Hq), view(Hq, Hkv), view(Hq + Hkv, Hq), view(2 * Hq + Hkv, Hkv)
    fq.copy_(q), fk.copy_(k)
    want, grad = pk.ops.qk_norm_rope_fwd(q, k, wq, wk, pos, 1e4), pk.ops.qk_norm_rope_bwd(dyq, dyk, q, k, wq, wk, pos, 1e4)
    pk.ops.qk_norm_rope_fwd(fq, fk, wq, wk, pos, 1e4, out=(yq, yk))
    ys = yq.clone(), yk.clone()
    got = pk.ops.qk_norm_rope_bwd(dyq, dyk, fq, fk, wq, wk, pos, 1e4, out=(yq, yk))
    for i, (x, w, dy) in enumerate(((q, wq, dyq), (k, wk, dyk))):
        x, w, size = x.double(), w.double(), dy.double().abs().amax(-1, keepdim=True) * 2 ** 0.5
        r = torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5)
        within("y", ys[i], want[i], 2 * HALF[dtype] * want[i].abs().double() + 2 * 32 * U * (x * r * w).abs().amax(-1, keepdim=True))
        within("dx", got[i], grad[i], 2 * HALF[dtype] * grad[i].abs().double() + 2 * 64 * U * r * size * w.abs().max() * (1 + (x * r).abs().amax(-1, keepdim=True)))
        within("dw", got[2 + i], grad[2 + i], 2 * (T * x.shape[2] + 16) * U * (size * (x * r).abs()).sum((0, 1, 2)))
    assert torch.equal(fq, q) and torch.equal(fk, k)


def test_qk_norm_rope_rows_do_not_depend_on_the_batch(pk):
    """A token alone, as in decoding, has the bits that it has inside a long batch."""
    for dtype in (FP32, BF16):
        q, k, wq, wk, pos, *_ = qk_inputs(3, 257, 14, 2, 64, dtype, 9)
        yq, yk = pk.ops.qk_norm_rope_fwd(q, k, wq, wk, pos, 1e6)
        for b, t in ((0, 0), (1, 100), (2, 256)):
            a, c = pk.ops.qk_norm_rope_fwd(q[b:b + 1, t:t + 1], k[b:b + 1, t:t + 1], wq, wk, pos[b:b + 1, t:t + 1], 1e6)
            assert torch.equal(a[0, 0], yq[b, t]) and torch.equal(c[0, 0], yk[b, t])


def test_qk_norm_rope_empty_and_zero_rows(pk):
    q, k, wq, wk, pos, dyq, dyk = qk_inputs(2, 4, 3, 2, 64, FP32, 1, "plain")
    e = lambda t: t[:, :0]  # noqa: E731
    assert pk.ops.qk_norm_rope_fwd(e(q), e(k), wq, wk, pos[:, :0], 1e4)[0].shape == (2, 0, 3, 64)
    dq, dk, dwq, dwk = pk.ops.qk_norm_rope_bwd(e(dyq), e(dyk), e(q), e(k), wq, wk, pos[:, :0], 1e4)
    assert dq.shape == (2, 0, 3, 64) and not dwq.any() and not dwk.any()
    z = torch.zeros_like(q)   # a row of zeros: r = 1/sqrt(eps), finite everywhere
    yq, _ = pk.ops.qk_norm_rope_fwd(z, k, wq, wk, pos, 1e4)
    dz = pk.ops.qk_norm_rope_bwd(dyq, dyk, z, k, wq, wk, pos, 1e4)
    assert not yq.any() and all(bool(torch.isfinite(t).all()) for t in dz) and not dz[2].any()


def test_qk_norm_rope_keeps_a_bad_row_to_itself(pk):
    for dtype in (FP32, BF16):
        q, k, wq, wk, pos, *_ = qk_inputs(1, 6, 4, 2, 64, dtype, 2, "plain")
        want, _ = pk.ops.qk_norm_rope_fwd(q, k, wq, wk, pos, 1e4)
        q = q.clone()
        q[0, 2, 1, 5], q[0, 4, 3, 0] = math.nan, math.inf
        got, _ = pk.ops.qk_norm_rope_fwd(q, k, wq, wk, pos, 1e4)
        bad = torch.zeros(1, 6, 4, dtype=torch.bool, device="cuda")
        bad[0, 2, 1] = bad[0, 4, 3] = True
        assert bool(torch.isnan(got[0, 2, 1]).all()) and torch.equal(got[~bad], want[~bad])


def test_results_written_over_a_tensor_are_seen_by_autograd(pk):
    """A tensor that another node saved and a call then writes over: the backward pass says so."""
    q, k, wq, wk, pos, *_ = qk_inputs(1, 4, 2, 1, 64, FP32, 3, "plain")
    leaf = q.clone().requires_grad_()
    y = (leaf * 1.0)
    z = y * y
    pk.ops.qk_norm_rope_fwd(y.detach(), k, wq, wk, pos, 1e4, out=(y.detach(), k))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.sum().backward()
    with pytest.raises(RuntimeError, match="single memory location"):
        pk.ops.qk_norm_rope_fwd(q, k, wq, wk, pos, 1e4, out=(q[:, :, :1].expand(1, 4, 2, 64), torch.empty_like(k)))


def test_qk_norm_rope_under_autograd(pk):
    """The node gives what the direct backward gives, also where only one output is used and where the gradient that arrives is not dense."""
    q, k, wq, wk, pos, dyq, dyk = qk_inputs(2, 19, 4, 2, 64, BF16, 3)
    leaves = [t.clone().requires_grad_() for t in (q, k, wq, wk)]
    yq, yk = pk.ops.qk_norm_rope(*leaves, pos, 1e4, 1e-5, 32, True)
    got = torch.autograd.grad([yq, yk], leaves, [dyq, dyk], retain_graph=True)
    want = pk.ops.qk_norm_rope_bwd(dyq, dyk, *(t.detach() for t in leaves), pos, 1e4, 1e-5, 32, True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    sideways = dyq.transpose(2, 3).contiguous().transpose(2, 3)   # head_dim not contiguous
    assert torch.equal(torch.autograd.grad(yq, leaves[0], sideways, retain_graph=True)[0],
                       pk.ops.qk_norm_rope_bwd(dyq, torch.zeros_like(dyk), *(t.detach() for t in leaves), pos, 1e4, 1e-5, 32, True)[0])
    got = torch.autograd.grad(yq.sum(), leaves[0], retain_graph=True)[0]
    want = pk.ops.qk_norm_rope_bwd(torch.ones_like(dyq), torch.zeros_like(dyk), *(t.detach() for t in leaves), pos, 1e4, 1e-5, 32, True)
    assert torch.equal(got, want[0])
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(yq.sum(), leaves[0], create_graph=True)
    with torch.no_grad():
        assert not pk.ops.qk_norm_rope(*leaves, pos, 1e4)[0].requires_grad


# ---- token log-probabilities and the losses ----------------------------------------------------------------------------


def loss_inputs(rows, vocab, dtype, seed, pitch=0, offset=0, forbidden=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((rows, max(vocab + offset, pitch)), generator=g, device="cuda").mul_(3.0).to(dtype)[:, offset:offset + vocab]
    if forbidden:
        x[:, ::forbidden] = -math.inf
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda").to(torch.int32)
    return x, t, g


def softmax64(x, t, scale):
    """z, lse, logp and p in 64 bits. A row that holds no number at all is all NaN there, as the formula has it."""
    z = x.double() * scale
    lse = torch.logsumexp(z, 1)
    lse = torch.where(torch.isinf(lse) & (lse < 0), math.nan, lse)
    return z, lse, z.gather(1, t.clamp(0, x.shape[1] - 1).long()[:, None])[:, 0] - lse, torch.exp(z - lse[:, None])


def sizes(z):
    """The largest finite |z| of each row, at least 1."""
    return torch.where(torch.isfinite(z), z, 0.0).abs().amax(1).clamp(min=1.0)


def logp_slack(z, vocab):
    """lse in 32-bit arithmetic: each exponent is within 2 u of its size (the product's constant, the rounding of the difference), each exponential within
    4 u, a chain of at most vocab/64 additions and a tree of 8; z_t - lse is formed in 64 bits and rounded once."""
    return (3 * sizes(z) + 12 + vocab / 64) * U


ROWS = [  # rows, vocab, pitch, offset, forbidden
    (1, 1, 0, 0, 0), (3, 2, 0, 0, 0), (5, 7, 0, 0, 3), (4, 64, 0, 0, 0), (9, 511, 0, 0, 5), (3, 1000, 1008, 0, 0), (2, 2048, 0, 0, 0), (3, 4097, 0, 0, 0),
    (2, 10007, 0, 0, 7), (3, 10007, 10016, 1, 0), (2, 16384, 0, 0, 0), (3, 32000, 0, 0, 0), (2, 32003, 0, 3, 2), (2, 65537, 0, 0, 0), (2, 131072, 0, 0, 0),
    (1, 200001, 0, 0, 0), (300, 33, 0, 0, 0), (1, 32000, 32064, 8, 0),
    (5, 70001, 70016, 3, 9), (130, 66000, 0, 0, 0), (2, 40001, 0, 0, 5)]


@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("case", ROWS, ids=lambda c: "-".join(map(str, c)))
def test_token_logprobs_against_64_bits(pk, case, dtype):
    """dlogits: the exponential's argument carries lse's rounding as well: 2 sizes more; times the coefficient."""
    rows, vocab, pitch, offset, forbidden = case
    x, t, g = loss_inputs(rows, vocab, dtype, 21, pitch, offset, forbidden)
    scale = 1.0 if vocab % 2 else 0.7
    if rows > 2:
        t[1] = -1
    dlogp = torch.randn(rows, generator=g, device="cuda")
    kept = x.clone()
    logp, lse = pk.ops.token_logprobs_fwd(x, t, scale)
    d = pk.ops.token_logprobs_bwd(x, t, lse, dlogp, scale)
    assert torch.equal(x, kept) and d.dtype == dtype
    s = float(np.float32(scale))
    z, wl, wp, p = softmax64(x, t, s)
    used = t >= 0
    wl, wp = torch.where(used, wl, 0.0), torch.where(used, wp, 0.0)
    slack = logp_slack(z, vocab)
    within("lse", lse, wl, U * wl.abs() + slack)
    within("logp", logp, wp, U * wp.abs().nan_to_num() + slack)
    hot = torch.zeros_like(p).scatter_(1, t.clamp(min=0).long()[:, None], 1.0)
    coef = torch.where(used, dlogp.double() * s, 0.0)[:, None]
    want = torch.where(coef != 0, coef * (hot - p), 0.0)
    within("dlogits", d, want, HALF[dtype] * want.abs() + coef.abs() * (slack + 2 * U * sizes(z))[:, None] + 1e-37)
    over = x.clone()   # over the logits: the same bits where the layout is the same
    same = pk.ops.token_logprobs_bwd(x.clone(), t, lse, dlogp, scale)
    assert pk.ops.token_logprobs_bwd(over, t, lse, dlogp, scale, out=over) is over and torch.equal(over, same)
    wide = torch.full((rows, vocab + 5), 7.0, dtype=dtype, device="cuda")   # into a wider matrix: its other columns stay
    pk.ops.token_logprobs_bwd(x, t, lse, dlogp, scale, out=wide[:, 2:2 + vocab])
    assert bool((wide[:, :2] == 7.0).all()) and bool((wide[:, 2 + vocab:] == 7.0).all())
    within("dlogits into a view", wide[:, 2:2 + vocab], want, HALF[dtype] * want.abs() + coef.abs() * (slack + 2 * U * sizes(z))[:, None] + 1e-37)


def test_token_logprobs_of_rows_that_hold_no_number(pk):
    """All -inf, a NaN, +inf; a forbidden target; a target past the vocabulary; a negative one in front of a row of NaN: by the formula, each to itself."""
    for dtype in (FP32, BF16):
        x, t, _ = loss_inputs(8, 3000, dtype, 5)
        fine = x.clone()
        x[0], x[1, 17], x[2, 5] = -math.inf, math.nan, math.inf
        x[3, 40] = -math.inf
        t[3], t[4], t[5] = 40, 3000, -7
        x[5] = math.nan
        logp, lse = pk.ops.token_logprobs_fwd(x, t)
        assert bool(torch.isnan(logp[[0, 1, 2, 4]]).all()) and float(logp[3]) == -math.inf and float(logp[5]) == 0.0 and bool(torch.isfinite(logp[6:]).all())
        dlogp = torch.ones(8, device="cuda")
        dlogp[7] = 0.0
        d = pk.ops.token_logprobs_bwd(x, t, lse, dlogp)
        assert bool(torch.isnan(d[[0, 1, 4]]).all(1).all()) and not d[5].any() and not d[7].any()
        assert bool(torch.isfinite(d[3]).all()) and float(d[3, 40]) == 1.0 and bool(torch.isfinite(d[6]).all())
        want, _ = pk.ops.token_logprobs_fwd(fine, t)
        assert torch.equal(logp[6:], want[6:])


@pytest.mark.parametrize("scale", [2.0 ** -64, 1e-6, 1.0, 1.4426951, 300.0, 2.0 ** 64])
def test_token_logprobs_over_scales(pk, scale):
    """The exponent's factor in two parts, both numbers over the whole range; words without probability stay so at each."""
    x, t, _ = loss_inputs(6, 3001, FP32, 12)
    x[:, 5::11] = -math.inf
    t = torch.where(torch.isinf(x.gather(1, t.long()[:, None])[:, 0]), t - 1, t).clamp(min=0).to(torch.int32)
    s = float(np.float32(scale))
    z, wl, wp, _ = softmax64(x, t, s)
    logp, lse = pk.ops.token_logprobs_fwd(x, t, scale)
    within("lse", lse, wl, U * wl.abs() + logp_slack(z, 3001))
    within("logp", logp, wp, U * wp.abs() + logp_slack(z, 3001))


@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("rows,vocab,pitch", [(7, 61, 0), (3, 3001, 0), (200, 777, 784), (2, 150001, 0), (130, 66000, 0)])
@pytest.mark.parametrize("base", [-2e3, 5e5, -3e38])
def test_losses_of_far_logits(pk, base, rows, vocab, pitch, dtype):
    """Logits far from zero: their differences alone count, and the log of the sum in 32 bits tells too little for a gradient. A difference is exact where it is
    of use; an exponent past 104 gives nothing; so an exponent is within 2 u of 104, its log2 of the sum within u of 20, and the rest as for other logits."""
    x, t, g = loss_inputs(rows, vocab, dtype, 17, pitch)
    x.copy_(x.float().mul_(max(1.0, abs(base) * 2.0 ** -21) / 3.0).add_(base).clamp_(min=torch.finfo(dtype).min))
    dlogp = torch.randn(rows, generator=g, device="cuda")
    t[::2] = x[::2].argmax(1).to(torch.int32)
    top = x.double().amax(1, keepdim=True)
    _, wl, wp, p = softmax64(x.double() - top, t, 1.0)
    near = (wp > -100.0).float()   # the others' ratio is that of two roundings
    slack = (3 * 104 + 12 + 2 * 20 + vocab / 64) * U
    logp, lse = pk.ops.token_logprobs_fwd(x, t)
    within("lse", lse, wl + top[:, 0], U * (wl + top[:, 0]).abs() + slack)
    within("logp", logp, wp, U * wp.abs() + slack)
    hot = torch.zeros_like(p).scatter_(1, t.long()[:, None], 1.0)
    for coef, d in ((dlogp, pk.ops.token_logprobs_bwd(x, t, lse, dlogp)), (dlogp, pk.ops.token_logprobs_bwd(x, t, lse, dlogp, out=x.new_empty((rows, vocab + 5))[:, 2:2 + vocab])),
                    (dlogp, pk.ops.token_logprobs_bwd(x.clone(), t, lse, dlogp)),
                    (-dlogp.abs() * near, pk.blockops.policy_loss(x, t, logp, dlogp.abs(), near)[1])):
        want = coef.double()[:, None] * (hot - p)
        within("dlogits", d, want, HALF[dtype] * want.abs() + coef.double().abs()[:, None] * 2 * slack + 1e-37)
    over = x.clone()
    pk.ops.token_logprobs_bwd(over, t, lse, dlogp, out=over)
    assert torch.equal(over, pk.ops.token_logprobs_bwd(x.clone(), t, lse, dlogp))


@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("rows,vocab", [(5, 700), (9, 5003), (300, 32000), (3, 40001), (2, 150001), (130, 70000)])
def test_losses_of_rows_with_one_likely_word(pk, rows, vocab, dtype):
    """The log-probability of a word that has nearly all is the others' sum, a hundredth to a millionth: that sum's own error counts, not the rounding of 1 beside
    it. An exponent is within 3 u of its size, an exponential within 4 u, log and the last rounding 4 u."""
    x, t, g = loss_inputs(rows, vocab, dtype, 71)
    x.mul_(1.0 / 3.0)
    x.scatter_(1, t.long()[:, None], (math.log(vocab) + 5.0 + 9.0 * torch.rand(rows, 1, generator=g, device="cuda")).to(dtype))
    z, _, wp, _ = softmax64(x, t, 1.0)
    size = (z.amax(1) - z.amin(1)) / math.log(2)
    tol = (3 * size + 12) * U * wp.abs()
    assert float(wp.min()) > -0.02 and float(tol.max()) < 0.02 * 200 * U
    within("logp", pk.ops.token_logprobs_fwd(x, t)[0], wp, tol)
    one = torch.ones(rows, device="cuda")
    within("policy's logp", pk.blockops.policy_loss(x, t, 0 * one, one, one)[2], wp, tol)


def likely_rows(rows, vocab, dtype, base):
    """Rows of which one word, the target, has all but a hundredth to a millionth, their logits around `base`; in 64 bits the softmax and what the others come to."""
    x, t, g = loss_inputs(rows, vocab, dtype, 73)
    x.mul_(1.0 / 3.0)
    x.scatter_(1, t.long()[:, None], (math.log(vocab) + 5.0 + 9.0 * torch.rand(rows, 1, generator=g, device="cuda")).to(dtype))
    x = (x.float() + base).to(dtype)
    z = x.double() - x.double().amax(1, keepdim=True)
    e = torch.exp(z)
    rest = e.scatter(1, t.long()[:, None], 0.0).sum(1)
    p = e / (1.0 + rest)[:, None]   # the target is the largest, its e is 1
    return x, t, g, -torch.log1p(rest), p.scatter(1, t.long()[:, None], (-rest / (1.0 + rest))[:, None]).neg(), (z.amin(1) / -math.log(2)).clamp(min=1.0)


def likely_within(name, d, want, coef, size, dtype):
    """Every element relative to its own value, the target's too: exponents within 3 u of their size, an exponential 4 u, the sum's log and the token's log-probability 4 u, coefficient and
    products 8 u."""
    want = coef.double()[:, None] * want
    within(name, d, want, want.abs() * (HALF[dtype] + (3 * size[:, None] + 16) * U) + 1e-37)


LIKELY = [(5, 700), (9, 5003), (300, 32000), (3, 40001), (2, 150001), (40, 70000), (600, 3001)]


@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("base", [0.0, 300.0, -900.0, 5e4])
@pytest.mark.parametrize("rows,vocab", LIKELY)
def test_policy_loss_gradient_of_rows_with_one_likely_word(pk, rows, vocab, base, dtype):
    """Few long rows, which are dealt out, and others alike."""
    x, t, g, logp, want, size = likely_rows(rows, vocab, dtype, base)
    old, adv, w = (logp + 0.05).float(), torch.randn(rows, generator=g, device="cuda"), torch.rand(rows, generator=g, device="cuda") + 0.5
    loss, d, got = pk.blockops.policy_loss(x, t, old, adv, w, 0.5, 0.5)
    likely_within("dlogits", d, want, -w.double() * torch.exp(logp - old.double()) * adv.double(), size, dtype)


@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("base", [0.0, 300.0, -900.0, 5e4])
@pytest.mark.parametrize("rows,vocab", LIKELY)
def test_preference_loss_gradient_of_rows_with_one_likely_word(pk, rows, vocab, base, dtype):
    """Pairs formed by the gradient's wavefronts and by a launch of their own; a margin moves by no more than its log-probabilities' own error."""
    x, t, g, logp, want, size = likely_rows(rows, vocab, dtype, base)
    half = rows // 2
    starts, ref = torch.tensor([0, half, rows], dtype=torch.int32, device="cuda"), (logp - 0.5 * torch.rand(rows, generator=g, device="cuda")).float()
    loss, d, margins, got = pk.blockops.preference_loss(x, t, starts, ref, 0.0625, 0.25)
    gain = logp - ref.double()
    u = 0.0625 * (gain[:half].sum() - gain[half:].sum())
    slope = (0.25 * torch.sigmoid(u) - 0.75 * torch.sigmoid(-u)) * 0.0625
    assert abs(float(slope)) > 2.0 ** -10
    coef = torch.where(torch.arange(rows, device="cuda") < half, slope, -slope)
    likely_within("dlogits", d, want, coef, size, dtype)


ALLOWED = {FP32: 2.0 ** -17, BF16: 2.0 ** -14}   # what a log of the sum in 32 bits may turn an element by


@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("base", [0.0, 300.0, -900.0, 5e4])
@pytest.mark.parametrize("rows,vocab", LIKELY)
def test_token_logprobs_gradient_of_rows_with_one_likely_word(pk, rows, vocab, base, dtype):
    """Direct, over the logits, into rows at another pitch and through the node: the log of the sum that the backward pass is given counts with what it is allowed to."""
    x, t, g, logp, want, size = likely_rows(rows, vocab, dtype, base)
    dlogp = torch.randn(rows, generator=g, device="cuda")
    lse = pk.ops.token_logprobs_fwd(x, t)[1]
    want = dlogp.double()[:, None] * want
    tol = want.abs() * (HALF[dtype] + 1.01 * ALLOWED[dtype] + (3 * size[:, None] + 16) * U) + 1e-37
    d = pk.ops.token_logprobs_bwd(x, t, lse, dlogp)
    within("dlogits", d, want, tol)
    wide = x.new_full((rows, vocab + 5), 7.0)
    pk.ops.token_logprobs_bwd(x, t, lse, dlogp, out=wide[:, 2:2 + vocab])
    over, leaf = x.clone(), x.clone().requires_grad_()
    pk.ops.token_logprobs_bwd(over, t, lse, dlogp, out=over)
    pk.ops.token_logprobs(leaf, t).backward(dlogp)
    assert torch.equal(leaf.grad, d) and bool((wide[:, :2] == 7.0).all()) and bool((wide[:, 2 + vocab:] == 7.0).all())
    within("dlogits over the logits", over, want, tol)
    within("dlogits at another pitch", wide[:, 2:2 + vocab], want, tol)


@pytest.mark.parametrize("rows,vocab", [(5, 700), (300, 5003), (3, 40001), (64, 33001)])
@pytest.mark.parametrize("base", [40.0, 120.0, -900.0])
def test_token_logprobs_gradient_at_logits_of_hundreds(pk, rows, vocab, base):
    """Every element in 32 bits relative to its own value; the sum's own chain of additions counts too, as in logp_slack."""
    x, t, g = loss_inputs(rows, vocab, FP32, 19)
    x.add_(base)
    dlogp = torch.randn(rows, generator=g, device="cuda")
    z = x.double() - x.double().amax(1, keepdim=True)
    p = torch.softmax(z, 1)
    want = dlogp.double()[:, None] * (torch.zeros_like(p).scatter_(1, t.long()[:, None], 1.0) - p)
    size = z.amin(1, keepdim=True) / -math.log(2)
    lse = pk.ops.token_logprobs_fwd(x, t)[1]
    for out in (None, x):
        d = pk.ops.token_logprobs_bwd(x, t, lse, dlogp, out=out)
        within("dlogits", d, want, want.abs() * (1.01 * ALLOWED[FP32] + (3 * size + 16 + vocab / 64) * U) + 1e-37)


def test_token_logprobs_dealt_out_and_whole(pk):
    """A few rows past what a workgroup holds: dealt to several with a workspace, whole without one, each within the count of the other test; rows that hold no number,
    are not read or have one word only, among them."""
    import ctypes as C
    L = pk.lib.lib()
    for dtype, code in ((FP32, pk.lib.PK_F32), (BF16, pk.lib.PK_BF16)):
        x, t, _ = loss_inputs(7, 150001, dtype, 9)
        x[0] = -math.inf
        x[1], x[1, 77000] = -math.inf, 2.0
        x[2, 149999], t[3], t[4], t[1], t[0] = math.nan, -1, 150001, 77000, 5
        z, wl, wp, _ = softmax64(x, t, 1.0)
        wl[3], wp[3], wp[4] = 0.0, 0.0, math.nan
        slack = logp_slack(z, 150001)
        need = L.pk_token_logprobs_workspace_bytes(7, 150001, code)
        assert need > 0
        for ws in (torch.full((need,), 255, dtype=torch.uint8, device="cuda"), None):   # a workspace holds anything before
            logp, lse = torch.full((7,), 3.0, device="cuda"), torch.full((7,), 3.0, device="cuda")
            p = lambda y: C.c_void_p(y.data_ptr() if y is not None else None)  # noqa: E731
            pk.lib.check(L.pk_token_logprobs_fwd(p(x), x.stride(0), p(t), 7, 150001, 1.0, p(logp), p(lse), p(ws), need if ws is not None else 0, code,
                                                 C.c_void_p(torch.cuda.current_stream().cuda_stream)))
            within("lse", lse, wl, U * wl.abs().nan_to_num() + slack)
            within("logp", logp, wp, U * wp.abs().nan_to_num() + slack)


def test_token_logprobs_under_autograd_and_empty(pk):
    x, t, g = loss_inputs(6, 300, FP32, 8)
    leaf = x.clone().requires_grad_()
    y = pk.ops.token_logprobs(leaf, t, 0.9)
    got = torch.autograd.grad(y.sum(), leaf)[0]   # a gradient that is one value broadcast
    lse = pk.ops.token_logprobs_fwd(x, t, 0.9)[1]
    assert torch.equal(got, pk.ops.token_logprobs_bwd(x, t, lse, torch.ones(6, device="cuda"), 0.9))
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(pk.ops.token_logprobs(leaf, t).sum(), leaf, create_graph=True)
    logp, lse = pk.ops.token_logprobs_fwd(x[:0], t[:0])
    assert logp.numel() == 0 and pk.ops.token_logprobs_bwd(x[:0], t[:0], lse, logp).shape == (0, 300)
    row = x[:1].expand(5, 300)                    # one row of logits for five tokens
    assert torch.equal(pk.ops.token_logprobs_fwd(row, t[:5])[0], pk.ops.token_logprobs_fwd(row.contiguous(), t[:5])[0])


def plain_policy(logp, old, ref, adv, w, lo, hi, kl):
    ratio = torch.exp(logp - old.double())
    lo, hi = float(np.float32(lo)), float(np.float32(hi))
    free, held = ratio * adv.double(), ratio.clamp(1 - lo, 1 + hi) * adv.double()
    each, slope = -torch.minimum(free, held), torch.where(free > held, 0.0, -free)   # what is no number stays none
    if kl:
        kl = float(np.float32(kl))
        d = ref.double() - logp
        each, slope = each + kl * (torch.exp(d) - d - 1), slope + kl * (1 - torch.exp(d))
    return each, slope


@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("kl", [0.0, 0.05])
@pytest.mark.parametrize("case", [c for c in ROWS if c[0] > 1], ids=lambda c: "-".join(map(str, c)))
def test_policy_loss_against_64_bits(pk, case, kl, dtype):
    """A row's loss moves by |slope| times logp's error (slack) and twice that for the exponentials' curvature; no ratio lies within 2^-10 of a clip."""
    rows, vocab, pitch, offset, forbidden = case
    x, t, g = loss_inputs(rows, vocab, dtype, 31, pitch, offset, forbidden)
    if forbidden:
        t = torch.where(torch.isinf(x.gather(1, t.long()[:, None])[:, 0]), (t + 1) % vocab, t).to(torch.int32)
    scale, lo, hi, upstream = 1.25, 0.2, 0.3, 0.5
    z, _, logp, p = softmax64(x, t, scale)
    drift = (0.3 * torch.randn(rows, generator=g, device="cuda")).double()
    for edge in (math.log(1 - lo), math.log(1 + hi)):
        drift = torch.where((drift - edge).abs() < 2 ** -10, drift + 2 ** -8, drift)
    old, ref = (logp - drift).float(), (logp + 0.2 * torch.randn(rows, generator=g, device="cuda")).float()
    adv, w = torch.randn(rows, generator=g, device="cuda"), torch.rand(rows, generator=g, device="cuda")
    w[0] = 0.0
    t[rows - 1] = -1
    x[0] = math.nan   # a row that does not count is not read
    loss, d, got = pk.blockops.policy_loss(x, t, old, adv, w, lo, hi, ref if kl else None, kl, scale, upstream)
    used = (t >= 0) & (w != 0)
    each, slope = plain_policy(logp, old, ref, adv, w, lo, hi, kl)
    wd = torch.where(used, w.double(), 0.0)
    slack = logp_slack(z, vocab) + U * (logp.abs() + 1)
    slack = torch.where(used, slack, 0.0)
    within("logp", got, torch.where(used, logp, 0.0), slack + 1e-37)
    steep = slope.abs() + adv.double().abs() * 2 + (1.0 if kl else 0.0)
    within("loss", loss, (wd * each)[used].sum(), (wd * (4 * steep * slack + 4 * U * each.abs()))[used].sum() + 1e-37)
    coef = torch.where(used, wd * slope * scale * upstream, 0.0)[:, None]
    hot = torch.zeros_like(p).scatter_(1, t.clamp(min=0).long()[:, None], 1.0)
    want = torch.where(used[:, None] & (coef != 0), coef * (hot - p), 0.0)
    tol = HALF[dtype] * want.abs() + (wd[:, None] * scale * upstream * 4 * steep[:, None] * (slack + 2 * U * sizes(torch.nan_to_num(z)))[:, None])
    within("dlogits", d, want, tol + 1e-37)
    over = x.clone()
    same = pk.blockops.policy_loss(x.clone(), t, old, adv, w, lo, hi, ref if kl else None, kl, scale, upstream)
    res = pk.blockops.policy_loss(over, t, old, adv, w, lo, hi, ref if kl else None, kl, scale, upstream, out=over)
    assert res[1] is over and same_bits(over, same[1]) and same_bits(res[0], same[0])


@pytest.mark.parametrize("rows,vocab,dtype", [(1, 33001, BF16), (32, 33001, BF16), (33, 66001, BF16), (64, 34007, FP32), (2, 200001, FP32)])
def test_policy_loss_dealt_out_and_whole(pk, rows, vocab, dtype):
    """A few long rows, dealt to several workgroups with a workspace and whole without one: each within the count of the other test, in place too; rows that do not
    count and one that is clipped among them."""
    import ctypes as C
    x, t, g = loss_inputs(rows, vocab, dtype, 61)
    z, _, lp, p = softmax64(x, t, 1.25)
    old, ref, adv, w = lp.float() - 0.1, lp.float() + 0.2, torch.randn(rows, generator=g, device="cuda"), torch.rand(rows, generator=g, device="cuda") + 0.1
    if rows > 4:
        w[1], t[2], old[3], adv[3] = 0.0, -1, old[3] - 3.0, 1.0
        x[1:3] = math.nan
    used = ((t >= 0) & (w != 0))
    each, slope = plain_policy(lp, old, ref, adv, w, 0.2, 0.3, 0.05)
    wd = torch.where(used, w.double(), 0.0)
    slack = torch.where(used, logp_slack(z, vocab) + U * (lp.abs() + 1), 0.0)
    steep = slope.abs() + adv.double().abs() * 2 + 1.0
    coef = torch.where(used, wd * slope * 1.25 * 0.5, 0.0)[:, None]
    want = torch.where(used[:, None] & (coef != 0), coef * (torch.zeros_like(p).scatter_(1, t.clamp(min=0).long()[:, None], 1.0) - p), 0.0)
    tol = HALF[dtype] * want.abs() + (wd[:, None] * 1.25 * 0.5 * 4 * steep[:, None] * (slack + 2 * U * sizes(z))[:, None]) + 1e-37
    L, code = pk.lib.lib(), pk.lib.PK_F32 if dtype == FP32 else pk.lib.PK_BF16
    need = L.pk_policy_loss_workspace_bytes(rows, vocab, code)
    assert need > 0
    c = pk.lib.PolicyConfig(0.2, 0.3, 0.05, 1.25, 0.5)
    for ws in (torch.full((need,), 255, dtype=torch.uint8, device="cuda"), None):
        for over in (False, True):
            a = x.clone()
            d = a if over else torch.full_like(x, 3.0)
            logp, loss, row_loss = torch.full((rows,), 3.0, device="cuda"), torch.zeros((), device="cuda"), torch.full((rows,), 3.0, dtype=F64, device="cuda")
            q = lambda y: C.c_void_p(y.data_ptr() if y is not None else None)  # noqa: E731
            pk.lib.check(L.pk_policy_loss(C.byref(c), q(a), vocab, q(t), q(old), q(ref), q(adv), q(w), rows, vocab, q(d), vocab, q(logp), q(row_loss), q(loss),
                                          q(ws), need if ws is not None else 0, code, C.c_void_p(torch.cuda.current_stream().cuda_stream)))
            within("logp", logp, torch.where(used, lp, 0.0), slack + 1e-37)
            within("loss", loss, (wd * each)[used].sum(), (wd * (4 * steep * slack + 4 * U * each.abs()))[used].sum() + 1e-37)
            within("dlogits", d, want, tol)


def test_policy_loss_gradient_against_differences(pk):
    """Along a direction in the logits; the loss is smooth between the clips. Two losses of fp32, each within 64 u of its terms, over a step of 2^-7; the
    third-order term of the step below 2^-11."""
    x, t, g = loss_inputs(12, 500, FP32, 41)
    logp = softmax64(x, t, 1.0)[2]
    old, ref = (logp - 0.05).float(), (logp + 0.1).float()
    adv, w = torch.randn(12, generator=g, device="cuda"), torch.full((12,), 1 / 12, device="cuda")
    way = 0.1 * torch.randn(x.shape, generator=g, device="cuda")
    f = lambda y: pk.blockops.policy_loss(y, t, old, adv, w, 0.5, 0.5, ref, 0.1)  # noqa: E731
    step = 2.0 ** -7
    slope = float((f(x)[1].double() * way.double()).sum())
    there = (float(f(x + step * way)[0]) - float(f(x - step * way)[0])) / (2 * step)
    size = float((w * (2 * adv.abs() + 0.3)).sum())
    assert abs(there - slope) <= (64 * U / step + 2.0 ** -11) * size


def test_policy_loss_of_nothing(pk):
    """No rows, and rows of which none counts: a loss of zero and a gradient of zeros."""
    x, t, g = loss_inputs(4, 100, FP32, 2)
    v = lambda n: torch.ones(n, device="cuda")  # noqa: E731
    loss, d, _ = pk.blockops.policy_loss(x[:0], t[:0], v(0), v(0), v(0))
    assert float(loss) == 0.0 and d.shape == (0, 100)
    loss, d, logp = pk.blockops.policy_loss(x * math.nan, t, v(4), v(4), v(4) * 0)
    assert float(loss) == 0.0 and not d.any() and not logp.any()


PAIRS = [  # lengths of chosen, lengths of rejected, rows behind, vocab, smoothing
    ([1], [1], 0, 50, 0.0), ([5, 0, 33], [7, 4, 0], 3, 1000, 0.1), ([300, 20], [17, 290], 0, 130, 0.0), ([9, 8, 7, 6], [1, 2, 3, 4], 1, 10007, 0.25),
    ([3], [4], 0, 32000, 1.0), ([0], [0], 2, 64, 0.3), ([40], [41], 0, 4096, 0.5),
    ([32] * 8, [32] * 8, 0, 700, 0.0), ([32] * 8, [32] * 8, 1, 700, 0.2), ([3] * 9, [4] * 9, 2, 3001, 0.1), ([255], [256], 1, 2000, 0.0), ([2000, 1, 0], [0, 900, 33], 9, 257, 0.1)]


@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("case", PAIRS, ids=str)
def test_preference_loss_against_64_bits(pk, case, dtype):
    """A margin is beta times a sum of differences of 32-bit values: slack + 2 u (|logp| + |ref|) of each; the loss's slope is at most 1."""
    chosen, rejected, behind, vocab, e = case
    lens, P = chosen + rejected, len(chosen)
    rows, beta, upstream, scale = sum(lens) + behind, 0.2, 2.0, 0.9
    x, t, g = loss_inputs(rows, vocab, dtype, 51)
    starts = torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device="cuda")
    t[torch.rand(rows, generator=g, device="cuda") < 0.25] = -1
    s32 = lambda v: float(np.float32(v))  # noqa: E731
    z, _, logp, p = softmax64(x, t, s32(scale))
    ref = (logp + 0.4 * torch.randn(rows, generator=g, device="cuda")).float()
    loss, d, margins, got = pk.blockops.preference_loss(x, t, starts, ref, beta, e, scale, upstream)
    used = t >= 0
    gain = torch.where(used, logp - ref.double(), 0.0)
    off = torch.where(used, logp_slack(z, vocab) + 2 * U * (logp.abs() + ref.double().abs()), 0.0)
    ends = starts.tolist()
    add = lambda v: torch.stack([v[a:b].sum() for a, b in zip(ends, ends[1:])])  # noqa: E731
    sums, offs = add(gain), add(off)
    u, du = s32(beta) * (sums[:P] - sums[P:]), s32(beta) * (offs[:P] + offs[P:])
    within("margins", margins, u, du + U * u.abs() + 1e-37)
    e32 = s32(e)
    want = (1 - e32) * torch.nn.functional.softplus(-u) + e32 * torch.nn.functional.softplus(u)
    within("loss", loss, want.mean(), (du + 4 * U * (want + 1)).mean())
    within("logp", got, torch.where(used, logp, 0.0), torch.where(used, logp_slack(z, vocab) + U * logp.abs(), 0.0) + 1e-37)
    slope = (e32 * torch.sigmoid(u) - (1 - e32) * torch.sigmoid(-u)) * s32(beta) * upstream / P
    of = torch.bucketize(torch.arange(rows, device="cuda"), starts[1:].long(), right=True)
    coef = torch.where(used & (of < 2 * P), torch.cat([slope, -slope, slope.new_zeros(1)])[of], 0.0) * s32(scale)
    hot = torch.zeros_like(p).scatter_(1, t.clamp(min=0).long()[:, None], 1.0)
    want = torch.where(coef[:, None] != 0, coef[:, None] * (hot - p), 0.0)
    wobble = torch.cat([du, du, du.new_zeros(1)])[of] * s32(beta) * upstream / P
    tol = HALF[dtype] * want.abs() + ((logp_slack(z, vocab) + 4 * U * sizes(z)) * coef.abs() + wobble + 4 * U * coef.abs())[:, None] + 1e-37
    within("dlogits", d, want, tol)
    over = x.clone()
    res = pk.blockops.preference_loss(over, t, starts, ref, beta, e, scale, upstream, out=over)
    assert torch.equal(over, d) and torch.equal(res[0], loss)


@pytest.mark.parametrize("ends", [(0, 60, 100, 160, 200), (5, 5, 5, 5, 5), (-9, 40, 190, 2 ** 31 - 1, -2 ** 31), (150, 100, 50, 0, 250)], ids=str)
def test_preference_loss_a_launch_less_or_not(pk, ends):
    """Two pairs formed by the gradient's wavefronts and, with rows behind that count nothing, by a launch of their own: sums in 64 bits in another order, so a step
    of 32 bits in the margins, and offsets that lie held to the rows alike."""
    x, t, g = loss_inputs(200, 900, FP32, 5)
    t[::7] = -1
    starts, ref = torch.tensor(ends, dtype=torch.int32, device="cuda"), -8 * torch.rand(200, generator=g, device="cuda")
    a = pk.blockops.preference_loss(x, t, starts, ref, 0.3, 0.1)
    more = lambda y, v: torch.cat([y, y.new_full((400, *y.shape[1:]), v)])  # noqa: E731
    b = pk.blockops.preference_loss(more(x, 0), more(t, -1), starts, more(ref, 0), 0.3, 0.1, out=x.new_empty(600, 903)[:, 2:902])
    assert torch.equal(a[3], b[3][:200]) and not b[3][200:].any() and not b[1][200:].any()
    within("margins", a[2], b[2], 2 * U * b[2].abs() + 1e-37)
    within("loss", a[0], b[0], 2 * U * (b[0].abs() + b[2].abs().sum()))
    within("dlogits", a[1], b[1][:200], 8 * U * b[1][:200].abs() + 1e-37)   # a step or two in the pair's slope, a rounding
    if sorted(ends) == list(ends):   # rows of no sequence
        assert not a[1][ends[-1]:].any() and not a[1][:ends[0]].any()


def test_preference_loss_of_thousands_of_pairs(pk):
    """More pairs than the small workgroups of short rows add up: margins are exact in their two log-probabilities, the loss their mean."""
    P = 5000
    x, t, g = loss_inputs(2 * P, 60, FP32, 5)
    starts, ref = torch.arange(2 * P + 1, device="cuda", dtype=torch.int32), -8 * torch.rand(2 * P, generator=g, device="cuda")
    loss, d, margins, logp = pk.blockops.preference_loss(x, t, starts, ref, 0.5)
    z, _, wp, p = softmax64(x, t, 1.0)
    u, off = 0.5 * (wp - ref.double()), 0.5 * (logp_slack(z, 60) + U * (wp.abs() + ref.double().abs()))
    u, off = u[:P] - u[P:], off[:P] + off[P:]
    within("margins", margins, u, off + U * u.abs())
    each = torch.nn.functional.softplus(-u)
    within("loss", loss, each.mean(), (off + 4 * U * (each + 1)).mean())
    slope = -torch.sigmoid(-u) * 0.5 / P
    coef = torch.cat([slope, -slope])[:, None]
    want = coef * (torch.zeros_like(p).scatter_(1, t.long()[:, None], 1.0) - p)
    within("dlogits", d, want, U * want.abs() + coef.abs() * (logp_slack(z, 60) + 4 * U * sizes(z) + torch.cat([off, off]) + 4 * U)[:, None])


def test_preference_loss_far_margins_and_lying_offsets(pk):
    """Margins of hundreds: loss and slope stay finite and right. Offsets outside the rows are held to them; nothing outside is read or written."""
    x, t, _ = loss_inputs(6, 200, FP32, 3)
    starts = torch.tensor([0, 3, 6], dtype=torch.int32, device="cuda")
    logp = pk.ops.token_logprobs_fwd(x, t)[0]
    for shift, want in ((-400.0, 0.0), (400.0, 3 * 400.0 * 0.5)):
        ref = logp.clone()
        ref[:3] += shift
        loss, d, margins, _ = pk.blockops.preference_loss(x, t, starts, ref, beta=0.5)
        assert abs(float(margins) + 1.5 * shift) < 1e-2 and abs(float(loss) - want) < 1e-2 and bool(torch.isfinite(d).all())
        assert (shift < 0) == (float(d.abs().max()) < 1e-30)
    wild = torch.tensor([-5, 3, 900], dtype=torch.int32, device="cuda")
    ref = logp - 0.25
    assert all(torch.equal(a, b) for a, b in zip(pk.blockops.preference_loss(x, t, wild, ref), pk.blockops.preference_loss(x, t, starts, ref)))


def test_preference_loss_of_an_answer_without_probability(pk):
    """A forbidden word in one answer: the margin is infinite, the loss 0 or infinite, and the gradient finite wherever the softmax is."""
    x, t, _ = loss_inputs(6, 200, FP32, 3)
    starts, ref = torch.tensor([0, 3, 6], dtype=torch.int32, device="cuda"), torch.full((6,), -5.0, device="cuda")
    for row, margin, loss in ((4, math.inf, 0.0), (1, -math.inf, math.inf)):
        y = x.clone()
        y[row, int(t[row])] = -math.inf
        got, d, margins, logp = pk.blockops.preference_loss(y, t, starts, ref)
        assert float(margins) == margin and float(got) == loss and float(logp[row]) == -math.inf and bool(torch.isfinite(d).all())
        assert bool(d.any()) == (margin < 0)


# ---- AdamW over many tensors --------------------------------------------------------------------------------------------


def mix32(x):
    x = np.asarray(x, np.uint64) & 0xFFFFFFFF
    x ^= x >> 16
    x = (x * 0xBB67AE85) & 0xFFFFFFFF
    x ^= x >> 15
    x = (x * 0x6A09E667) & 0xFFFFFFFF
    return x ^ (x >> 16)


@functools.lru_cache(None)
def powers_of_two():
    """2^-126 .. 2^127 as torch.ldexp forms them on the device: for some exponents one step of fp32 below the power."""
    e = torch.arange(-126, 128, device="cuda", dtype=torch.int32)
    return torch.ldexp(torch.ones(e.numel(), device="cuda"), e).cpu().numpy()


def pack8(x, chance, square):
    """numpy restatement of the 8-bit states: codes and scales of a flat fp32 array."""
    x = np.asarray(x, np.float32)
    n, top, drop, bias = x.size, *((15, 21, 112) if square else (8, 20, 120))
    rows = np.pad(x, (0, -n % 256)).reshape(-1, 256)
    scale, codes = np.empty(rows.shape[0], np.float32), np.empty(rows.shape, np.uint8)
    chance = np.pad(chance, (0, -n % 256)).reshape(-1, 256).astype(np.uint64)
    for i, row in enumerate(rows):
        most = np.abs(row).max()
        if not np.isfinite(most):
            scale[i], codes[i] = np.nan, 0x7F
            continue
        part, power = np.frexp(most)
        e = max(-126, int(power) - 1 - top + (part > 0.875)) if most > 0 else -126
        scale[i] = powers_of_two()[e + 126]
        y = row * powers_of_two()[126 - e]
        bits = (np.abs(y) * np.float32(2.0) ** np.float32(-bias)).astype(np.float32).view(np.uint32).astype(np.uint64)
        bits = (bits + (chance[i] << np.uint64(drop - 16)) + np.uint64(1 << (drop - 17))) >> np.uint64(drop)
        codes[i] = np.maximum(bits, row > 0) if square else bits | (np.signbit(y).astype(np.uint64) << np.uint64(7))
    return codes.reshape(-1)[:n], scale


def plain_adamw(p, g, m, v, lr, b1, b2, eps, wd, t, factor):
    """m and v bit for bit in 32 bits, p in 64 from them."""
    f = np.float32
    with np.errstate(all="ignore"):
        g = (g * f(factor)).astype(f)
        m2 = f(b1) * m + f(f(1) - f(b1)) * g
        v2 = f(b2) * v + (f(f(1) - f(b2)) * g) * g
        c1, c2 = 1 - float(f(b1)) ** t, 1 - float(f(b2)) ** t
        d = lambda x: x.astype(np.float64)  # noqa: E731
        upd = d(m2) / c1 / (np.sqrt(d(v2) / c2) + float(f(eps)))
        p2 = d(p) - float(f(lr)) * (upd + float(f(wd)) * d(p))
    return p2, m2, v2, upd


SIZES = [[1], [255, 256, 257], [4096, 1, 4097, 3], [70001, 512], [5] * 130 + [3000], [0, 7, 0]]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("grads", [FP32, BF16], ids=["g32", "g16"])
@pytest.mark.parametrize("clip", [0.0, 0.7])
@pytest.mark.parametrize("ns", SIZES, ids=lambda s: f"{len(s)}x{max(s)}")
@pytest.mark.parametrize("apart", [False, True], ids=["aligned", "unaligned"])
def test_adamw_many_against_plain(pk, bits, grads, clip, ns, apart):
    """Three steps. m, v and their codes are those of the formula in 32 bits, bit for bit; the norm is a sum in 64; p is rounded once and its update carries 16
    u (the two corrections, a root, two quotients, sums)."""
    rng = np.random.default_rng(17)
    lr, b1, b2, eps, wd = 0.01, 0.9, 0.99, 1e-8, 0.1

    def on(x, dt=FP32):   # one element past an aligned address where asked
        flat = torch.empty(x.size + 1, dtype=dt, device="cuda")
        t = flat[1:] if apart else flat[:-1]
        t.copy_(torch.from_numpy(x).to(dt))
        return t

    P = [rng.standard_normal(n).astype(np.float32) for n in ns]
    ps = [on(p) for p in P]
    copies = [on(p, BF16) for p in P]
    if bits == 32:
        state = pk.blockops.AdamWState([on(np.zeros(n, np.float32)) for n in ns], [on(np.zeros(n, np.float32)) for n in ns])
    else:
        def codes(dt):
            return [torch.zeros(n + 1, dtype=torch.uint8, device="cuda")[int(apart):n + int(apart)].view(dt) for n in ns]
        fresh = pk.blockops.adamw_state(ps, 8)
        state = pk.blockops.AdamWState(codes(torch.float8_e4m3fn), codes(torch.float8_e5m2), fresh.m_scale, fresh.v_scale)
    M = [np.zeros(n, np.float32) for n in ns]
    V = [np.zeros(n, np.float32) for n in ns]
    for t in (1, 2, 3):
        seed = 1000 + t
        G = [torch.from_numpy((rng.standard_normal(n) * np.exp(2 * rng.standard_normal(n))).astype(np.float32)).to(grads) for n in ns]
        gs = [on(g.float().numpy(), grads) for g in G]
        norm = pk.blockops.adamw_many_(ps, gs, state, lr, b1, b2, eps, wd, t=t, max_norm=clip, copies=copies, seed=seed)
        total = math.sqrt(sum(float((g.double() ** 2).sum()) for g in G))
        factor = np.float32(1.0)
        if clip:
            assert abs(float(norm) - total) <= 2 * U * total
            # the factor is a quotient of 64-bit numbers rounded once: the device's, from its norm, may be the neighbour
            factor = np.float32(float(np.float32(clip)) / total) if total > clip else np.float32(1.0)
        else:
            assert norm is None
        for i, n in enumerate(ns):
            if not n:
                continue
            p2, m2, v2, upd = plain_adamw(P[i], G[i].float().numpy(), M[i], V[i], lr, b1, b2, eps, wd, t, factor)
            got = ps[i].cpu().numpy()
            tol = U * np.abs(p2) + 16 * U * lr * (np.abs(upd) + wd * np.abs(P[i]) + np.abs(P[i])) + 1e-37
            assert (np.abs(got - p2) <= tol).all(), f"p of {n} at step {t}"
            assert torch.equal(copies[i], ps[i].to(BF16)) and torch.equal(gs[i].cpu(), G[i])
            P[i] = got
            if bits == 32:
                assert np.array_equal(state.m[i].cpu().numpy(), m2) and np.array_equal(state.v[i].cpu().numpy(), v2)
                M[i], V[i] = m2, v2
                continue
            key = mix32(seed * 0x9E3779B9 + int(mix32(i + 0x3C6EF373)))
            h = mix32(np.arange(n, dtype=np.uint64) ^ key)
            for x, chance, codes_, scales, square in ((m2, h & 0xFFFF, state.m[i], state.m_scale[i], False), (v2, h >> 16, state.v[i], state.v_scale[i], True)):
                want, ws = pack8(x, chance, square)
                assert np.array_equal(scales.cpu().numpy(), ws) and np.array_equal(codes_.view(torch.uint8).cpu().numpy(), want), f"codes of {n} at step {t}"
            up = lambda c, s, n=n: (c.float().cpu() * s.cpu().repeat_interleave(256)[:n]).numpy()  # noqa: E731
            M[i], V[i] = up(state.m[i], state.m_scale[i]), up(state.v[i], state.v_scale[i])


@pytest.mark.parametrize("grads", [FP32, BF16], ids=["g32", "g16"])
@pytest.mark.parametrize("wd", [0.0, 0.1])
def test_adamw_many_parameters_bit_for_bit(pk, grads, wd):
    """With moments in 32 bits a step is the formula's own roundings, the parameter's too: products and sums by themselves, a root and a quotient to half a step. Whole blocks and what is
    behind them, gradients of 2^-40 to 2^20, zeros."""
    f, rng = np.float32, np.random.default_rng(5)
    lr, b1, b2, eps, w = f(0.01), f(0.9), f(0.99), f(1e-8), f(wd)
    p = rng.standard_normal(300001).astype(f)
    m, v = np.zeros_like(p), np.zeros_like(p)
    got = torch.from_numpy(p).cuda()
    state = pk.blockops.adamw_state([got])
    for t in (1, 2, 1000):
        g = torch.from_numpy((rng.standard_normal(p.size) * 2.0 ** rng.integers(-40, 20, p.size)).astype(f)).to(grads)
        g[::97] = 0.0
        pk.blockops.adamw_many_([got], [g.cuda()], state, float(lr), float(b1), float(b2), float(eps), wd, t=t)
        g = g.float().numpy()
        m, v = b1 * m + (f(1) - b1) * g, b2 * v + ((f(1) - b2) * g) * g
        per1, per2 = (f(1 / (1 - float(b) ** t)) for b in (b1, b2))
        p = p - lr * ((m * per1) / (np.sqrt(v * per2) + eps) + w * p)
        assert p.dtype == m.dtype == f and np.array_equal(state.m[0].cpu().numpy(), m) and np.array_equal(state.v[0].cpu().numpy(), v)
        assert np.array_equal(got.cpu().numpy(), p), t


def test_adamw_many_states_in_8_bits_do_not_stall(pk):
    """v under a constant gradient: each step moves it by (1 - b2)(g^2 - v), under 1/16 of a step of its format, so rounded to nearest it would stay where it is.
    Over 4096 elements its mean follows the formula: after 200 steps within 5 standard errors of draws whose spread is at most a step (1/4 of the
    value) each, as the last 1 / (1 - b2) of them count: 0.25 * sqrt((1 - b2) / 2 + 1) / 64 * 5 relative."""
    n, b2 = 4096, 0.99
    p, g = torch.zeros(n, device="cuda"), torch.ones(n, device="cuda")
    state = pk.blockops.adamw_state([p], 8)
    for t in range(1, 201):
        pk.blockops.adamw_many_([p], [g], state, 0.0, 0.9, b2, t=t, seed=t)
    v = state.v[0].float() * state.v_scale[0].repeat_interleave(256)
    want = 1 - b2 ** 200
    assert abs(float(v.mean()) - want) <= 0.25 * math.sqrt(1 + (1 - b2) / 2) / 64 * 5 * want


def test_adamw_many_what_is_not_finite_stays_in_its_block(pk):
    """A NaN and an infinity in the gradients: their own parameter and, in 8 bits, their own block's state; nothing else."""
    for bits in (8, 32):
        n = 1024
        g = torch.randn(n, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
        runs = []
        for bad in (False, True):
            p, gg = torch.ones(n, device="cuda"), g.clone()
            if bad:
                gg[300], gg[700] = math.nan, math.inf
            state = pk.blockops.adamw_state([p], bits)
            pk.blockops.adamw_many_([p], [gg], state, 0.1, seed=4)
            value = [x[0].float() * (s[0].repeat_interleave(256) if s else 1.0) for x, s in ((state.m, state.m_scale), (state.v, state.v_scale))]
            runs.append([p, *value])
        (p0, m0, v0), (p1, m1, v1) = runs
        ok = torch.ones(n, dtype=torch.bool, device="cuda")
        ok[300] = ok[700] = False
        assert torch.equal(p0[ok], p1[ok]) and bool(torch.isnan(p1[~ok]).all())
        if bits == 8:
            ok[256:512] = ok[512:768] = False
            assert bool(torch.isnan(m1[~ok]).all()) and bool(torch.isnan(v1[~ok]).all())
        assert torch.equal(m0[ok], m1[ok]) and torch.equal(v0[ok], v1[ok])


def test_adamw_many_extremes(pk):
    """Gradients from the smallest numbers there are to 1e18, zeros, blocks of one kind and mixed: codes as restated, a v that is not zero never zero, zero blocks
    stay zero."""
    n = 256 * 6
    g = torch.zeros(n)
    g[0:256] = 1e-45
    g[256:512] = 1e18 * torch.linspace(-1, 1, 256)
    g[512:768] = torch.logspace(-30, 15, 256)
    g[768:1024] = 0.0
    g[1024:1280] = torch.logspace(-20, -10, 256) * torch.tensor([1.0, -1.0]).repeat(128)
    g[1280] = 3.0
    p = torch.zeros(n, device="cuda")
    state = pk.blockops.adamw_state([p], 8)
    pk.blockops.adamw_many_([p], [g.cuda()], state, 1e-3, 0.9, 0.99, seed=77)
    _, m2, v2, _ = plain_adamw(np.zeros(n, np.float32), g.numpy(), np.zeros(n, np.float32), np.zeros(n, np.float32), 1e-3, 0.9, 0.99, 1e-8, 0.01, 1, 1.0)
    h = mix32(np.arange(n, dtype=np.uint64) ^ mix32(77 * 0x9E3779B9 + int(mix32(0x3C6EF373))))
    for x, chance, got, scales, square in ((m2, h & 0xFFFF, state.m[0], state.m_scale[0], False), (v2, h >> 16, state.v[0], state.v_scale[0], True)):
        want, ws = pack8(x, chance, square)
        assert np.array_equal(got.view(torch.uint8).cpu().numpy(), want) and np.array_equal(scales.cpu().numpy(), ws)
    codes = state.v[0].view(torch.uint8).cpu().numpy()
    assert ((v2 > 0) == (codes > 0)).all() and not state.m[0].view(torch.uint8)[768:1024].any() and bool(torch.isfinite(p).all())


def test_adamw_many_skips_what_has_no_gradient(pk):
    """A None gradient leaves parameter and state as they are, and the other tensors' draws where they were."""
    g = torch.Generator(device="cuda").manual_seed(6)
    mk = lambda n: torch.randn(n, generator=g, device="cuda")  # noqa: E731
    P, G = [mk(500), mk(600), mk(700)], [mk(500), mk(600), mk(700)]
    runs = []
    for hole in (False, True):
        ps = [p.clone() for p in P]
        state = pk.blockops.adamw_state(ps, 8)
        pk.blockops.adamw_many_(ps, [G[0], None if hole else G[1], G[2]], state, 0.01, seed=9)
        runs.append((ps, state))
    (a, sa), (b, sb) = runs
    assert torch.equal(b[1], P[1]) and not sb.m[1].view(torch.uint8).any() and not sb.m_scale[1].any()
    for i in (0, 2):
        assert torch.equal(a[i], b[i]) and torch.equal(sa.m[i].view(torch.uint8), sb.m[i].view(torch.uint8)) and torch.equal(sa.v_scale[i], sb.v_scale[i])


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_many_writes_over_its_own_gradients(pk, bits):
    """bf16 copies in the place of the bf16 gradients, whole blocks and what is behind them, with a clip: the bits of a call with copies of their own."""
    g = torch.Generator(device="cuda").manual_seed(4)
    ps = [torch.randn(n, generator=g, device="cuda") for n in (70001, 5, 256, 40000)]
    gs = [torch.randn(p.shape, generator=g, device="cuda").to(BF16) for p in ps]
    runs = []
    for over in (False, True):
        p, grads = [x.clone() for x in ps], [x.clone() for x in gs]
        state, copies = pk.blockops.adamw_state(p, bits), grads if over else [torch.empty_like(x) for x in grads]
        norm = pk.blockops.adamw_many_(p, grads, state, 0.01, max_norm=1.0, copies=copies, seed=3)
        assert all(torch.equal(a, b.to(BF16)) for a, b in zip(copies, p))
        runs.append([y.view(torch.uint8) for y in (*p, *state.m, *state.v, norm.view(1))])
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    two = [torch.zeros(300, device="cuda") for _ in range(2)]   # each the other one's gradient; each other's copies in the gradients' places
    with pytest.raises(RuntimeError, match="element for element"):
        pk.blockops.adamw_many_(two, two[::-1], pk.blockops.adamw_state(two, bits), 0.01)
    halves = [y.to(BF16) for y in two]
    with pytest.raises(RuntimeError, match="element for element"):
        pk.blockops.adamw_many_(two, halves, pk.blockops.adamw_state(two, bits), 0.01, copies=halves[::-1])
    assert not any(y.any() for y in (*two, *halves))


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_many_does_not_depend_on_how_a_list_is_dealt(pk, bits):
    """A tensor's bits beside others of any number and size, in one launch or several, with bf16 copies or without."""
    g = torch.Generator(device="cuda").manual_seed(9)
    grads = [torch.randn(n, generator=g, device="cuda") for n in [70000] + [1 + 37 * k for k in range(260)]]

    def run(n_more, large, copies):
        gs = grads[:1 + n_more] + ([torch.ones(large, device="cuda")] if large else [])
        ps = [torch.zeros_like(y) for y in gs]
        state = pk.blockops.adamw_state(ps, bits)
        out = [torch.empty_like(y, dtype=BF16) for y in ps] if copies else None
        for t in (1, 2):
            norm = pk.blockops.adamw_many_(ps, gs, state, 0.01, t=t, max_norm=1e9, copies=out, seed=t)
        assert abs(float(norm) - math.sqrt(sum(float((y.double() ** 2).sum()) for y in gs))) <= 2 * U * float(norm)
        if copies:
            assert all(torch.equal(a, b.to(BF16)) for a, b in zip(out, ps))
        return [[y.view(torch.uint8) for y in x[:1 + n_more]] for x in (ps, state.m, state.v)]

    want = run(0, 0, False)
    for n_more, large, copies in ((0, 0, True), (260, 0, False), (260, 0, True), (3, 5 * 10 ** 6, False), (3, 9 * 10 ** 6, True)):
        got = run(n_more, large, copies)
        assert all(torch.equal(a[0], b[0]) for a, b in zip(got, want)), (n_more, large, copies)
        if (n_more, copies) == (260, False):
            long = got
        elif n_more:
            assert all(torch.equal(a, b) for x, y in zip(got, long) for a, b in zip(x, y))


def test_adamw_many_is_adamw_and_clip(pk):
    """32-bit states against `clip_grad_norm_` and `adamw_` one tensor at a time: the formula is the same, its roundings differ (16 u of the update)."""
    g = torch.Generator(device="cuda").manual_seed(8)
    mk = lambda n: torch.randn(n, generator=g, device="cuda")  # noqa: E731
    ps, gs = [mk(3000), mk(17)], [mk(3000), mk(17)]
    qs, hs = [p.clone() for p in ps], [x.clone() for x in gs]
    state, ms, vs = pk.blockops.adamw_state(ps), [torch.zeros_like(p) for p in ps], [torch.zeros_like(p) for p in ps]
    for t in (1, 2):
        norm = pk.blockops.adamw_many_(ps, gs, state, 0.01, t=t, max_norm=1.0)
        copy = [h.clone() for h in hs]
        total = pk.blockops.clip_grad_norm_(copy, 1.0)
        assert abs(float(norm) - total) <= 4 * U * total
        for q, x, m, v in zip(qs, copy, ms, vs):
            pk.blockops.adamw_(q, x, m, v, 0.01, t=t)
        # c2 = 1 - b2^t is formed in 32 bits there: 2^-24 / (1 - 0.999^t) of it, half of that of the update
        slack = (16 * U + U / (1 - 0.999 ** t)) * 0.01 * 40
        assert all(float((p - q).abs().max()) <= slack + 4 * U * float(q.abs().max()) for p, q in zip(ps, qs))


# ---- past 32 bits ---------------------------------------------------------------------------------------------------------


def test_qk_norm_rope_past_2_to_the_31(pk):
    """Heads whose offsets pass 32 bits, in elements: the last tokens' bits are those of a call on them alone, forward and backward."""
    T, Hq, Hkv, dk = 35000, 480, 2, 128
    g = torch.Generator(device="cuda").manual_seed(2)
    qkv = torch.empty(1, T, Hq + Hkv, dk, dtype=BF16, device="cuda")
    assert qkv.numel() > 2 ** 31
    qkv[:, :8].normal_(generator=g)
    qkv[:, -8:].normal_(generator=g)
    qkv[:, 8:-8].zero_()
    q, k = qkv[:, :, :Hq], qkv[:, :, Hq:]
    w, pos = 1 + 0.2 * torch.randn(dk, generator=g, device="cuda"), torch.arange(T, device="cuda", dtype=torch.int32)
    yq, yk = pk.ops.qk_norm_rope_fwd(q, k, w, w, pos, 1e4)
    last = slice(T - 8, T)
    a, b = pk.ops.qk_norm_rope_fwd(q[:, last], k[:, last], w, w, pos[last], 1e4)
    assert torch.equal(a, yq[:, last]) and torch.equal(b, yk[:, last]) and not yq[:, 8:64].any()
    dq, dk_, *_ = pk.ops.qk_norm_rope_bwd(yq, yk, q, k, w, w, pos, 1e4)
    c, d, *_ = pk.ops.qk_norm_rope_bwd(a, b, q[:, last], k[:, last], w, w, pos[last], 1e4)
    assert torch.equal(c, dq[:, last]) and torch.equal(d, dk_[:, last])


def test_losses_past_2_to_the_31(pk):
    """Logits whose rows begin past 2^31 elements, in place: the last rows' bits are those of a call on them alone."""
    rows, vocab, tail = 68000, 32000, 7
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.zeros(rows, vocab, dtype=BF16, device="cuda")
    x[-tail:].normal_(generator=g)
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda").to(torch.int32)
    t[:-tail] = -1
    old, adv, w = torch.full((rows,), -11.0, device="cuda"), torch.ones(rows, device="cuda"), torch.ones(rows, device="cuda")
    last = x[-tail:].clone()
    cut = lambda *v: tuple(y[-tail:].contiguous() for y in v)  # noqa: E731
    want = pk.blockops.policy_loss(last, *cut(t, old, adv, w))
    lp = pk.ops.token_logprobs_fwd(last, *cut(t))
    logp, lse = pk.ops.token_logprobs_fwd(x, t)
    assert torch.equal(logp[-tail:], lp[0]) and torch.equal(lse[-tail:], lp[1]) and not logp[:-tail].any()
    loss, d, logp = pk.blockops.policy_loss(x, t, old, adv, w, out=x)
    assert torch.equal(d[-tail:], want[1]) and torch.equal(logp[-tail:], want[2]) and torch.equal(loss, want[0]) and not d[:16].any() and not d[-tail - 9:-tail].any()
    d[-tail:] = last
    assert torch.equal(pk.ops.token_logprobs_bwd(d, t, lse, w, out=d)[-tail:], pk.ops.token_logprobs_bwd(last, *cut(t, lse, w)))


def test_losses_of_more_rows_than_a_launch_has_threads_for(pk):
    """2^26 rows and three: each entry's rows are those of calls on a few of them, at both ends, around every 2^22 and between; every other row's against 64 bits."""
    rows, vocab = 2 ** 26 + 3, 3
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(rows, vocab, generator=g, device="cuda", dtype=FP32).to(BF16)
    t = torch.randint(-1, vocab, (rows,), generator=g, device="cuda").to(torch.int32)
    old, adv, w = torch.full((rows,), -1.0, device="cuda"), torch.randn(rows, generator=g, device="cuda"), torch.rand(rows, generator=g, device="cuda") / rows
    some = sorted({min(max(k * 2 ** 22 + o, 0), rows - 8) for k in range(17) for o in range(-40, 41, 8)} | {12345678})
    part = torch.cat([torch.arange(r, r + 8, device="cuda") for r in some])
    few = [y[part] for y in (x, t, old, adv, w)]
    logp, lse = pk.ops.token_logprobs_fwd(x, t)
    want = pk.ops.token_logprobs_fwd(few[0], few[1])
    assert torch.equal(logp[part], want[0]) and torch.equal(lse[part], want[1])
    for r in range(0, rows, 2 ** 24):
        z = x[r:r + 2 ** 24].double()
        used = t[r:r + 2 ** 24] >= 0
        wl = torch.where(used, torch.logsumexp(z, 1), 0.0)
        wp = torch.where(used, z.gather(1, t[r:r + 2 ** 24].clamp(min=0).long()[:, None])[:, 0] - wl, 0.0)
        within("logp", logp[r:r + 2 ** 24], wp, U * wp.abs() + logp_slack(z, vocab))
    d = pk.ops.token_logprobs_bwd(x, t, lse, adv)
    assert torch.equal(d[part], pk.ops.token_logprobs_bwd(few[0], few[1], want[1], few[3]))
    loss, d, logp = pk.blockops.policy_loss(x, t, old, adv, w)
    want = pk.blockops.policy_loss(*few)
    assert torch.equal(d[part], want[1]) and torch.equal(logp[part], want[2])
    each = torch.where(t >= 0, -torch.minimum(torch.exp(logp.double() + 1) * adv, torch.exp(logp.double() + 1).clamp(0.8, 1.2) * adv) * w, 0.0)
    within("loss", loss, each.sum(), U * each.abs().sum() * 8)
    starts = torch.tensor([0, rows // 4, rows // 2, 3 * (rows // 4), rows], dtype=torch.int32, device="cuda")
    loss, d, margins, logp = pk.blockops.preference_loss(x, t, starts, old, beta=2.0 ** -12)
    within("margins", margins, torch.stack([sum((1 - 2 * k) * ((logp.double() + 1) * (t >= 0))[starts[i + 2 * k]:starts[i + 2 * k + 1]].sum() for k in range(2)) for i in range(2)]) * 2.0 ** -12,
           rows / 4 * 2.0 ** -12 * 4 * U)
    want = pk.ops.token_logprobs_bwd(*few[:2], pk.ops.token_logprobs_fwd(*few[:2])[1], torch.where(part < rows // 2, 1.0, -1.0).contiguous())
    slope = [torch.sigmoid(-margins[i].double()) * 2.0 ** -13 for i in range(2)]
    which = sum((part >= int(s)).long() for s in starts[1:4]) % 2
    want = -want.double() * torch.where(which == 0, slope[0], slope[1])[:, None]
    within("dlogits", d[part], want, want.abs() * 3 * HALF[BF16] + 1e-37)
    assert bool(torch.isfinite(loss))


def test_adamw_many_past_2_to_the_31(pk):
    """One tensor of more than 2^31 elements with 8-bit moments: the last block's values and codes, whose draws come from the element's place."""
    n, tail = 2 ** 31 + 700, 700
    p, g = torch.zeros(n, device="cuda"), torch.zeros(n, dtype=BF16, device="cuda")
    g[-tail:] = torch.randn(tail, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda").to(BF16)
    state = pk.blockops.adamw_state([p], 8)
    norm = pk.blockops.adamw_many_([p], [g], state, 0.01, max_norm=1.0, seed=21)
    gl = g[-tail:].float().cpu()
    total = math.sqrt(float((gl.double() ** 2).sum()))
    assert abs(float(norm) - total) <= 2 * U * total
    z = np.zeros(tail, np.float32)
    p2, m2, v2, upd = plain_adamw(z, gl.numpy(), z, z, 0.01, 0.9, 0.999, 1e-8, 0.01, 1, np.float32(1.0 / total) if total > 1 else np.float32(1))
    assert (np.abs(p[-tail:].cpu().numpy() - p2) <= U * np.abs(p2) + 16 * U * 0.01 * np.abs(upd) + 1e-37).all() and not p[:4096].any()
    h = mix32((np.arange(n - tail, n, dtype=np.uint64) & 0xFFFFFFFF) ^ mix32(21 * 0x9E3779B9 + int(mix32(0x3C6EF373))))
    for x, chance, got, scales, square in ((m2, h & 0xFFFF, state.m[0], state.m_scale[0], False), (v2, h >> 16, state.v[0], state.v_scale[0], True)):
        want, ws = pack8(x, chance, square)   # 2^31 is a whole number of blocks: the tail's blocks are the tensor's last three
        assert np.array_equal(got[-tail:].view(torch.uint8).cpu().numpy(), want) and np.array_equal(scales[-3:].cpu().numpy(), ws)


# ---- together, captured, on other streams ---------------------------------------------------------------------------------


def graph_of(fn):
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        fn()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fn()
    return graph, out


def test_operators_under_graph_capture(pk):
    """Every call recorded and replayed three times on new inputs, with eager calls of the same between the replays: each replay has the eager bits."""
    q, k, wq, wk, pos, dyq, dyk = qk_inputs(2, 40, 4, 2, 64, BF16, 3)
    q, k = q.contiguous(), k.contiguous()
    x, t, g = loss_inputs(50, 5000, BF16, 4)
    v = lambda: torch.rand(50, generator=g, device="cuda")  # noqa: E731
    old, ref, adv, w = -8 * v(), -8 * v(), v() - 0.5, v()
    starts = torch.tensor([0, 10, 20, 40, 50], dtype=torch.int32, device="cuda")
    p0 = [torch.randn(n, generator=g, device="cuda") for n in (700, 5000)]
    grads = [torch.randn(n, generator=g, device="cuda") for n in (700, 5000)]
    ps, state = [p.clone() for p in p0], pk.blockops.adamw_state(p0, 8)

    def losses():
        return (*pk.ops.qk_norm_rope_fwd(q, k, wq, wk, pos, 1e4), *pk.ops.qk_norm_rope_bwd(dyq, dyk, q, k, wq, wk, pos, 1e4),
                *pk.ops.token_logprobs_fwd(x, t), *pk.blockops.policy_loss(x, t, old, adv, w, ref_logp=ref, kl_coef=0.1),
                *pk.blockops.preference_loss(x, t, starts, ref))

    def step(ps, state):
        return pk.blockops.adamw_many_(ps, grads, state, 0.01, t=3, max_norm=1.0, seed=5)

    graph, out = graph_of(losses)
    fresh = lambda: (  # noqa: E731
        [p.clone() for p in p0], pk.blockops.adamw_state(p0, 8))
    graph2, norm = graph_of(lambda: step(ps, state))
    for again in range(3):
        for y in (q, k, dyq, dyk, x):
            y.copy_(torch.randn(y.shape, generator=g, device="cuda").to(y.dtype))
        for y in grads:
            y.normal_(generator=g)
        want = [y.clone() for y in losses()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), again
        for a, b in zip(ps, p0):
            a.copy_(b)
        for a in (*state.m, *state.v):
            a.view(torch.uint8).zero_()
        for a in (*state.m_scale, *state.v_scale):
            a.zero_()
        eps, estate = fresh()
        enorm = step(eps, estate)
        graph2.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, enorm) and all(torch.equal(a, b) for a, b in zip(ps, eps))
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip((*state.m, *state.v), (*estate.m, *estate.v)))


def test_larger_calls_under_graph_capture(pk):
    """What takes more launches than the calls above: a preference loss over many rows, dealt-out rows, gradients of long logs, lists of several tables."""
    x, t, g = loss_inputs(700, 3001, BF16, 4)
    y, u, _ = loss_inputs(3, 150001, FP32, 5)
    starts, ref = torch.tensor([0, 300, 700], dtype=torch.int32, device="cuda"), torch.full((700,), -8.0, device="cuda")
    dlogp = torch.ones(3, device="cuda")
    ps, gs = ([torch.zeros(n, device="cuda") for n in [3000] + [40] * 300] for _ in range(2))
    state = pk.blockops.adamw_state(ps, 32)

    def calls():
        logp, lse = pk.ops.token_logprobs_fwd(y, u)
        return (*pk.blockops.preference_loss(x, t, starts, ref), logp, lse, pk.ops.token_logprobs_bwd(y, u, lse, dlogp),
                *pk.blockops.policy_loss(y, u, ref[:3], dlogp, dlogp))

    def step(ps, state):
        return pk.blockops.adamw_many_(ps, gs, state, 0.01, t=2, max_norm=1.0)

    graph, out = graph_of(calls)
    graph2, norm = graph_of(lambda: step(ps, state))
    for again in range(3):
        x.copy_(torch.randn(x.shape, generator=g, device="cuda").to(BF16))
        y.copy_(torch.randn(y.shape, generator=g, device="cuda") + 3000 * (again == 1))
        for v in gs:
            v.normal_(generator=g)
        for v in (*ps, *state.m, *state.v):
            v.fill_(0.5)
        eager = [v.clone() for v in ps]
        estate = pk.blockops.AdamWState([v.clone() for v in state.m], [v.clone() for v in state.v])
        enorm = step(eager, estate)
        want = [v.clone() for v in calls()]
        graph.replay()
        graph2.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), again
        assert torch.equal(norm, enorm) and all(torch.equal(a, b) for a, b in zip((*ps, *state.m, *state.v), (*eager, *estate.m, *estate.v))), again


def test_a_backward_pass_under_graph_capture(pk):
    """Both nodes recorded with the passes around them and replayed between eager calls. While an eager graph of the same leaves lives, their gradients belong
    to its stream, which must not wait for a recording: refused, and the next recording stands."""
    q, k, wq, wk, pos, dyq, dyk = qk_inputs(2, 24, 4, 2, 64, FP32, 3)
    x, t, g = loss_inputs(48, 700, FP32, 4)
    q, k, x = (y.contiguous().requires_grad_() for y in (q, k, x))
    wq, wk = wq.requires_grad_(), wk.requires_grad_()

    def norms():
        yq, yk = pk.ops.qk_norm_rope(q, k, wq, wk, pos, 1e4)
        return torch.autograd.grad((yq * dyq).sum() + (yk * dyk).sum(), (q, k, wq, wk))

    def logp():
        return torch.autograd.grad((pk.ops.token_logprobs(x, t) * 0.5).sum(), x)

    for fn, graph_that_lives in ((norms, lambda: pk.ops.qk_norm_rope(q, k, wq, wk, pos, 1e4)), (logp, lambda: pk.ops.token_logprobs(x, t))):
        alive = graph_that_lives()
        with pytest.raises(RuntimeError, match="outside of the recording"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                fn()
        del alive
        graph, out = graph_of(fn)
        for _ in range(3):
            with torch.no_grad():
                for y in (q, k, x):
                    y.copy_(torch.randn(y.shape, generator=g, device="cuda"))
            want = fn()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_operators_on_two_streams_at_once(pk):
    """The same calls queued on two streams over different inputs: the results of one after the other."""
    sets = []
    for seed in (1, 2):
        x, t, g = loss_inputs(400, 8000, BF16, seed)
        sets.append((x, t, torch.full((400,), -9.0, device="cuda"), torch.randn(400, generator=g, device="cuda"), torch.rand(400, generator=g, device="cuda"),
                     torch.tensor([0, 200, 400], dtype=torch.int32, device="cuda"), qk_inputs(2, 300, 4, 4, 128, BF16, seed)))

    def work(s):
        x, t, old, adv, w, starts, (q, k, wq, wk, pos, dyq, dyk) = s
        return (*pk.blockops.policy_loss(x, t, old, adv, w), *pk.blockops.preference_loss(x, t, starts, old), *pk.ops.qk_norm_rope_bwd(dyq, dyk, q, k, wq, wk, pos, 1e4))

    want = [work(s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [None, None]
    for _ in range(3):
        for i, (st, s) in enumerate(zip(streams, sets)):
            with torch.cuda.stream(st):
                got[i] = work(s)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for u, v in zip(got, want) for a, b in zip(u, v))


def test_a_policy_step_through_all_operators(pk):
    """One layer with per-head norms, attention, a head, the policy loss on log-probabilities of an older model, and the optimiser, in fp32: loss, the gradients of
    all seven parameters and the parameters after the step against the same model in 64 bits. The longest chain is about 10 operators of sums over at
    most 64 terms: 2^-15 of the largest gradient of a tensor."""
    B, T, Hq, Hkv, dk, V = 2, 24, 4, 2, 16, 97
    d = Hq * dk
    g = torch.Generator().manual_seed(13)
    randn = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    params = {"emb": randn(V, d), "qkv": randn(d, (Hq + 2 * Hkv) * dk) / 8, "wq": 1 + 0.2 * randn(dk), "wk": 1 + 0.2 * randn(dk), "o": randn(d, d) / 8,
              "head": randn(d, V) / 8, "gain": 1 + 0.1 * randn(d)}
    ids, t = torch.randint(0, V, (B, T), generator=g), torch.randint(0, V, (B * T,), generator=g)
    pos = torch.arange(T)
    adv, w = randn(B * T), (torch.rand(B * T, generator=g) > 0.3).float() / 30
    drift = 0.1 * randn(B * T)

    def plain(P):
        x = P["emb"][ids]
        q, k, v = (x @ P["qkv"]).view(B, T, -1, dk).split([Hq, Hkv, Hkv], 2)
        q, k = plain_qk(q, P["wq"], pos, 1e4, 1e-5, 0, False), plain_qk(k, P["wk"], pos, 1e4, 1e-5, 0, False)
        k, v = (y.repeat_interleave(Hq // Hkv, 2) for y in (k, v))
        s = (q[:, :, None] * k[:, None]).sum(-1) * dk ** -0.5   # [B, T, T, H]
        s = s.masked_fill(~torch.ones(T, T, dtype=torch.bool).tril()[None, :, :, None], -math.inf)
        a = (torch.softmax(s, 2)[..., None] * v[:, None]).sum(2)
        h = x + a.reshape(B, T, d) @ P["o"]
        return (h.view(B * T, d) * P["gain"]) @ P["head"]

    P64 = {n: p.double().requires_grad_() for n, p in params.items()}
    logits = plain(P64)
    logp = torch.log_softmax(logits, 1).gather(1, t[:, None])[:, 0]
    old = (logp.detach() - drift).float()
    each, _ = plain_policy(logp, old, None, adv, w, 0.2, 0.2, 0.0)
    want_loss = (w.double() * each).sum()
    want = torch.autograd.grad(want_loss, list(P64.values()))

    leaves = {n: p.cuda().requires_grad_() for n, p in params.items()}
    x = leaves["emb"][ids.cuda()]
    q, k, v = (x @ leaves["qkv"]).view(B, T, -1, dk).split([Hq, Hkv, Hkv], 2)
    q, k = pk.ops.qk_norm_rope(q, k, leaves["wq"], leaves["wk"], pos.to(torch.int32).cuda(), 1e4)
    a = pk.ops.attention(q, k, v, dk ** -0.5)
    h = x + a.reshape(B, T, d) @ leaves["o"]
    out = (h.view(B * T, d) * leaves["gain"]) @ leaves["head"]
    loss, dlogits, _ = pk.blockops.policy_loss(out.detach(), t.to(torch.int32).cuda(), old.cuda(), adv.cuda(), w.cuda())
    out.backward(dlogits)
    want_loss = float(want_loss.detach())
    assert abs(float(loss) - want_loss) <= 2.0 ** -15 * float((w * adv.abs()).sum())
    for (n, leaf), ref in zip(leaves.items(), want):
        assert float((leaf.grad.double().cpu() - ref).abs().max()) <= 2.0 ** -15 * float(ref.abs().max()), n
    ps, gs = [leaf.detach() for leaf in leaves.values()], [leaf.grad for leaf in leaves.values()]
    before = leaves["head"]._version
    norm = pk.blockops.adamw_many_(ps, gs, pk.blockops.adamw_state(ps), 0.01, eps=1e-3, max_norm=0.05)
    total = math.sqrt(sum(float((r ** 2).sum()) for r in want))
    assert abs(float(norm) - total) <= 2.0 ** -15 * total and leaves["head"]._version > before
    f = min(1.0, 0.05 / total)
    for (n, leaf), ref, p in zip(leaves.items(), want, params.values()):
        step = (ref * f) / ((ref * f).abs() + 1e-3)   # m / c1 = g and sqrt(v / c2) = |g| at the first step
        slack = 0.01 * (2.0 ** -15 * f * float(ref.abs().max()) / 1e-3 + 2.0 ** -18) + 2.0 ** -22 * float(p.abs().max())
        assert float((leaf.detach().double().cpu() - (p.double() - 0.01 * (step + 0.01 * p.double()))).abs().max()) <= slack, n
