"""The operators of a student model on the GPU against plain implementations in 64 bits: the gated delta rule, layer norm with the residual addition, distillation
from a teacher's top logits.

Tolerances are counted as in test_post_ops_gpu.py: u = 2^-24 is half a step of fp32 relative to a value, h half a step of the output's type (u, or 2^-8 for bf16). An
output carries one rounding to its type, h * |value|, and what the 32-bit arithmetic before it adds up to, in u times the largest term that enters it."""
from __future__ import annotations

import math

import pytest
import torch

from test_post_ops_gpu import BF16, F64, FP32, HALF, U, graph_of, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pk():
    from paperkiln_amd import _lib, blockops, ops
    _lib.check(_lib.lib().pk_init(0, None, 0))

    class Both:
        pass
    b = Both()
    b.ops, b.blockops, b.lib = ops, blockops, _lib
    return b


def bits(x):
    return x.contiguous().view({2: torch.int16, 4: torch.int32, 8: torch.int64}[x.element_size()])


def same(a, b):
    return len(a) == len(b) and all(torch.equal(bits(x), bits(y)) for x, y in zip(a, b))


# ---- gated delta rule ----------------------------------------------------------------------------------------------------


def plain_delta(q, k, v, g, beta, scale, state=None, do=None, dstate=None):
    """Token by token in 64 bits; with do the gradients (dq, dk, dv, dg, dbeta, dstate) too, walking back."""
    B, T, Hk, dk = q.shape
    Hv, dv = v.shape[2:]
    rep = Hv // Hk
    q, k = (x.double().repeat_interleave(rep, 2) for x in (q, k))
    v, a, b = v.double(), g.double().exp(), beta.double()
    S = torch.zeros(B, Hv, dk, dv, dtype=F64, device=q.device) if state is None else state.double()
    outs, steps = [], []
    for t in range(T):
        kept = a[:, t, :, None, None] * S
        e = v[:, t] - (k[:, t, :, :, None] * kept).sum(2)
        u = b[:, t, :, None] * e
        after = kept + k[:, t, :, :, None] * u[:, :, None]
        outs.append(scale * (q[:, t, :, :, None] * after).sum(2))
        steps.append((S, kept, e, u, after))
        S = after
    o = torch.stack(outs, 1) if T else torch.zeros(B, 0, Hv, dv, dtype=F64, device=q.device)
    if do is None:
        return o, S
    D = torch.zeros_like(S) if dstate is None else dstate.double()
    dq, dk_, dv_, dg, db = (torch.zeros_like(x) for x in (q, k, v, a, b))
    for t in reversed(range(T)):
        before, kept, e, u, after = steps[t]
        d = do[:, t].double()
        dq[:, t] = scale * (after * d[:, :, None]).sum(-1)
        D = D + scale * q[:, t, :, :, None] * d[:, :, None]
        du = (D * k[:, t, :, :, None]).sum(2)
        dw = b[:, t, :, None] * du
        dv_[:, t], db[:, t] = dw, (du * e).sum(-1)
        dk_[:, t] = (D * u[:, :, None]).sum(-1) - (kept * dw[:, :, None]).sum(-1)
        D = D - k[:, t, :, :, None] * dw[:, :, None]
        dg[:, t] = (D * kept).sum((-1, -2))
        D = a[:, t, :, None, None] * D
    dq, dk_ = (x.unflatten(2, (Hk, rep)).sum(3) for x in (dq, dk_))
    return (o, S), (dq, dk_, dv_, dg, db, D)


def delta_inputs(B, T, Hk, Hv, dk, dv, dtype, seed=1, layout="plain", state=True):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    unit = lambda x: x / x.square().sum(-1, keepdim=True).sqrt().clamp(min=1e-6)  # noqa: E731
    q, k, v, do = unit(randn(B, T, Hk, dk)).to(dtype), unit(randn(B, T, Hk, dk) + 0.5).to(dtype), randn(B, T, Hv, dv).to(dtype), randn(B, T, Hv, dv).to(dtype)

    def lay(x):
        if layout == "heads":       # [B, H, T, d] memory
            return x.transpose(1, 2).contiguous().transpose(1, 2)
        if layout == "offset":      # one element past an aligned address, odd pitches
            return torch.nn.functional.pad(x, (1, 2))[..., 1:-2]
        if layout == "fused":       # between the columns of a projection
            return torch.nn.functional.pad(x.flatten(2), (8, 24))[..., 8:-24].unflatten(2, x.shape[2:])
        return x
    q, k, v, do = map(lay, (q, k, v, do))
    beta = torch.sigmoid(randn(B, T, Hv))
    g = -torch.nn.functional.softplus(randn(B, T, Hv)) * torch.exp(-6.0 * torch.rand((1, 1, Hv), generator=gen, device="cuda"))
    first = randn(B, Hv, dk, dv) * dk ** -0.5 if state else None
    return q, k, v, g, beta, first, do, randn(B, Hv, dk, dv)


NAMES = ("o", "state", "dq", "dk", "dv", "dg", "dbeta", "dstate")


def close(name, got, want, dtype, times=1.0, dk=128, pair=0.0):
    """The matrix cores add up 32 products at a time, six rounds of them for each 32 of a sum of values in three parts: at most 24 roundings in a row of u each, in either
    direction: 5 u of a result's root mean square. Three such products follow one another in a chunk (K S, T R, K^T U), and what is wrong in a state shrinks as
    the state does (unit keys, beta to 1): 9 u. Over all of an output 16 u then, times 2 for a gradient, which goes both ways, and 4 for dg, a sum of differences of terms up to four times its
    size. dg_t is besides a sum over the chunk's pairs of tokens on either side of t, at most 32 x 32 of them, whose terms are of one size where all keys are the same and nothing decays
    (dk = 1), while what they come to is the nearest ones': steps with beta of a half forget in two. 1024 independent roundings are 32 of one pair's. Keys of dk random
    columns overlap by dk^-1/2, twice in a term: 32 / dk. And the pairs on one side of t go out in 64 bits: 4096 terms of `pair` at most leave 4096 * 2^-53 of it. One element: that times 16 (the largest of a million is 5 times their root mean square, and they are of different sizes), of the largest of its head and
    sequence. The rounding to the output's type is counted by itself."""
    got, want = got.double(), want.double()
    assert got.shape == want.shape, name
    if not want.numel():
        return
    n = 16 * times * {"o": 1, "state": 1, "dg": 4 + 32 / dk}.get(name, 2) * U
    h = HALF[got_type(got, dtype, name)]
    over = [i for i in range(want.dim()) if i not in (0, head_axis(name))]
    top = want.abs().amax(over, keepdim=True)
    within(name, got, want, h * want.abs() + 16 * n * top + 1e-30 + (2.0 ** -41 * pair if name == "dg" else 0.0))
    if h == U:
        far, size = float((got - want).norm()), float(want.norm())
        assert far <= (n + U) * size + 1e-30 + (2.0 ** -41 * pair * want.numel() ** 0.5 if name == "dg" else 0.0), (name, far / max(size, 1e-300) / U)


def got_type(got, dtype, name):
    return FP32 if name in ("state", "dstate", "dg", "dbeta") else dtype


def head_axis(name):
    return 1 if name in ("state", "dstate") else 2


def check_delta(pk, q, k, v, g, beta, first, do, dlast, scale, times=1.0):
    dtype = q.dtype
    kept = [t.clone() for t in (q, k, v, g, beta, do, dlast)]
    o, state = pk.ops.gated_delta_rule_fwd(q, k, v, g, beta, scale, first)
    grads = pk.ops.gated_delta_rule_bwd(do, q, k, v, g, beta, scale, first, dlast)
    assert same(kept, (q, k, v, g, beta, do, dlast))
    assert o.dtype == dtype and state.dtype == FP32 and [t.dtype for t in grads[:5]] == [dtype] * 3 + [FP32] * 2 and (grads[5] is None) == (first is None)
    held = g.clamp(min=-1000.0)
    (wo, ws), want = plain_delta(q, k, v, held, beta, scale, first, do, dlast)
    want = list(want)
    want[3] = torch.where(g < -1000.0, 0.0, want[3])
    for n, a, b in zip(NAMES, (o, state, *grads), (wo, ws, *want)):
        if a is not None:
            close(n, a, b, dtype, times, q.shape[3], 2 * abs(scale) * v.shape[3] * float(do.double().abs().max() * v.double().abs().max()))
    return (o, state, *grads), (wo, ws, *want)


DELTAS = [  # B, T, Hk, Hv, dk, dv, layout, state
    (1, 1, 1, 1, 1, 1, "plain", True), (2, 1, 2, 4, 64, 64, "plain", True), (1, 2, 1, 1, 3, 5, "plain", False), (2, 15, 2, 2, 32, 32, "fused", True), (3, 16, 1, 3, 40, 72, "heads", False), (2, 7, 2, 2, 32, 32, "fused", True), (3, 8, 1, 3, 40, 72, "heads", False), (1, 9, 1, 2, 128, 100, "offset", True),
    (2, 17, 2, 2, 64, 64, "plain", True), (1, 63, 1, 1, 128, 128, "plain", True), (2, 64, 3, 3, 64, 128, "heads", True), (1, 65, 2, 6, 48, 80, "offset", True),
    (2, 130, 1, 7, 64, 64, "fused", False), (1, 200, 2, 2, 128, 256, "plain", True), (1, 257, 1, 2, 127, 33, "offset", False), (3, 100, 2, 2, 16, 8, "plain", True),
    (1, 300, 3, 3, 33, 31, "heads", True), (9, 70, 1, 1, 96, 96, "fused", True), (1, 500, 1, 1, 31, 1, "plain", True), (1, 129, 1, 2, 1, 255, "offset", True),
    # heads enough for workgroups of 32 columns: whole blocks, rows of whole pieces, any
    (32, 100, 4, 8, 32, 64, "fused", True), (16, 130, 16, 16, 64, 32, "heads", False), (9, 70, 8, 32, 128, 32, "plain", True), (40, 75, 2, 8, 24, 40, "plain", True),
    (70, 66, 1, 4, 96, 16, "fused", False), (64, 90, 2, 4, 31, 17, "offset", True), (64, 65, 2, 4, 101, 9, "plain", False)]


@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("case", DELTAS, ids=lambda c: "-".join(map(str, c)))
def test_gated_delta_rule_against_64_bits(pk, case, dtype):
    B, T, Hk, Hv, dk, dv, layout, state = case
    check_delta(pk, *delta_inputs(B, T, Hk, Hv, dk, dv, dtype, 3, layout, state), dk ** -0.5)


@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("T", [8, 9, 190])
@pytest.mark.parametrize("which", ["no decay", "no beta", "documents", "strong", "mixed", "same keys", "reflections", "padding"])
def test_gated_delta_rule_extremes(pk, which, T, dtype):
    """Decays of 1, of 0 and of nearly 0 among others, and sums of them that go far; keys that repeat with beta 1 (T's rows go back and forth) and beta 2, whose steps are
    reflections: nothing shrinks what is wrong there, so over 190 tokens it adds up, 3 chunks to a fourfold count."""
    q, k, v, g, beta, first, do, dlast = delta_inputs(2, T, 2, 4, 64, 48, dtype, 5)
    times = 1.0
    if which == "no decay":
        g, times = torch.zeros_like(g), 4.0
    elif which == "no beta":
        beta = torch.zeros_like(beta)
    elif which == "documents":
        g[:, 5], g[0, T // 2], g[1, T - 1, 1], g[:, 0, 2] = -math.inf, -math.inf, -math.inf, -math.inf
    elif which == "strong":
        g = g * 40 - 30
    elif which == "mixed":
        g[:, ::7], g[:, 3::11], g[:, 4] = -50.0, -1e30, -999.0
    elif which == "same keys":
        k, beta, g, times = k[:, :1].expand(k.shape), torch.ones_like(beta), g * 0.01, 4.0
        k = k.contiguous()
    elif which == "reflections":
        beta, g, times = torch.full_like(beta, 2.0), torch.zeros_like(g), 4.0
        k = (k.double() / k.double().norm(dim=-1, keepdim=True)).to(dtype)
    else:
        beta[0, T - 6:], g[0, T - 6:] = 0.0, 0.0
    out, _ = check_delta(pk, q, k, v, g, beta, first, do, dlast, 0.125, times)
    if which == "padding":   # the state is the one before it, to the bit where the chunks are the same
        close("state", out[1][:1], plain_delta(*(x[:1, :T - 6] for x in (q, k, v, g, beta)), 0.125, first[:1])[1], dtype)
    if which == "no beta":
        assert not out[4].any()


def test_gated_delta_rule_goes_on_from_a_state(pk):
    """A sequence in pieces, each from the state that the one before has left, by tokens and by chunks: the whole one's values. Steps move their state on in place."""
    for dtype in (FP32, BF16):
        q, k, v, g, beta, first, _, _ = delta_inputs(2, 150, 2, 4, 64, 64, dtype, 6)
        wo, ws = plain_delta(q, k, v, g, beta, 0.125, first)
        state, parts, at = first, [], 0
        for n in (1, 70, 3, 64, 12):
            o, state = pk.ops.gated_delta_rule_fwd(*(x[:, at:at + n] .contiguous() if x.dim() == 3 else x[:, at:at + n] for x in (q, k, v, g, beta)), 0.125, state)
            parts.append(o)
            at += n
        close("o", torch.cat(parts, 1), wo, dtype)
        close("state", state, ws, dtype)
        moved, parts, version = first.clone(), [], None
        place = moved.data_ptr()
        for a, n in ((0, 1), (1, 5), (6, 100), (106, 44)):   # more than a few tokens at once too
            parts.append(pk.ops.gated_delta_step_(*(x[:, a:a + n].contiguous() if x.dim() == 3 else x[:, a:a + n] for x in (q, k, v, g, beta)), 0.125, moved))
        assert moved.data_ptr() == place
        close("o", torch.cat(parts, 1), wo, dtype)
        close("state", moved, ws, dtype)


def test_gated_delta_rule_of_nothing(pk):
    q, k, v, g, beta, first, do, dlast = delta_inputs(2, 5, 1, 2, 16, 24, FP32, 7)
    e = lambda x: x[:, :0]  # noqa: E731
    o, state = pk.ops.gated_delta_rule_fwd(e(q), e(k), e(v), e(g), e(beta), 1.0, first)
    assert o.shape == (2, 0, 2, 24) and torch.equal(state, first)
    assert not pk.ops.gated_delta_rule_fwd(e(q), e(k), e(v), e(g), e(beta), 1.0)[1].any()
    grads = pk.ops.gated_delta_rule_bwd(e(do), e(q), e(k), e(v), e(g), e(beta), 1.0, first, dlast)
    assert torch.equal(grads[5], dlast) and grads[0].shape == (2, 0, 1, 16)
    assert not pk.ops.gated_delta_rule_bwd(e(do), e(q), e(k), e(v), e(g), e(beta), 1.0, first)[5].any()
    o, state = pk.ops.gated_delta_rule_fwd(q[:0], k[:0], v[:0], g[:0], beta[:0], 1.0)
    assert o.shape == (0, 5, 2, 24) and state.shape == (0, 2, 16, 24)
    moved = first.clone()
    pk.ops.gated_delta_step_(e(q), e(k), e(v), e(g), e(beta), 1.0, moved)
    assert torch.equal(moved, first)


@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
def test_gated_delta_rule_keeps_a_bad_value_to_its_head(pk, dtype):
    """What is not finite spoils its head of its sequence from its chunk on, and nothing else: other heads, other sequences, chunks before it (forward) and after it (backward)."""
    q, k, v, g, beta, first, do, dlast = delta_inputs(2, 200, 2, 4, 32, 40, dtype, 8)
    fwd = lambda: pk.ops.gated_delta_rule_fwd(q, k, v, g, beta, 1.0, first)  # noqa: E731
    bwd = lambda: pk.ops.gated_delta_rule_bwd(do, q, k, v, g, beta, 1.0, first, dlast)  # noqa: E731
    (o, state), grads = fwd(), bwd()
    v = v.clone()
    v[1, 130, 2, 7] = math.nan
    o2, state2 = fwd()
    good = torch.ones_like(o, dtype=torch.bool)
    good[1, 128:, 2] = False
    assert torch.equal(o2[good], o[good]) and bool(torch.isnan(o2[1, 130:, 2, 7].float()).all())
    assert torch.equal(state2[0], state[0]) and torch.equal(state2[1, [0, 1, 3]], state[1, [0, 1, 3]]) and torch.equal(state2[1, 2, :, :7], state[1, 2, :, :7])
    for a, b in zip(grads, bwd()):
        assert torch.equal(a[0], b[0])
    v = v.nan_to_num()
    k = k.clone()
    k[0, 3, 1, 0] = math.inf
    o2, _ = fwd()
    assert torch.equal(o2[1, :, 0], o[1, :, 0]) and torch.equal(o2[0, :, :2], o[0, :, :2]) and not bool(torch.isfinite(o2[0, 3:, 2:].float()).any())


def test_gated_delta_rule_repeats_its_bits(pk):
    """The same call twice, and a batch's sequences by themselves: the same bits."""
    q, k, v, g, beta, first, do, dlast = delta_inputs(3, 150, 2, 6, 64, 64, BF16, 9)
    run = lambda i: [*pk.ops.gated_delta_rule_fwd(*(x[i] for x in (q, k, v, g, beta)), 0.125, first[i]),  # noqa: E731
                     *pk.ops.gated_delta_rule_bwd(do[i], *(x[i] for x in (q, k, v, g, beta)), 0.125, first[i], dlast[i])]
    whole = run(slice(None))
    assert same(whole, run(slice(None)))
    for i in range(3):
        assert same([x[i:i + 1] for x in whole], run(slice(i, i + 1)))


def test_gated_delta_rule_gradient_against_differences(pk):
    """The derivative of sum(o do) + sum(S dS) along a direction against a central difference of the operator in fp32: two sums whose terms carry 64 u of their size, over a
    step of 2^-6; the third-order term, of a product of at most five inputs' changes, is below 2^-10 of the terms."""
    q, k, v, g, beta, first, do, dlast = delta_inputs(1, 70, 1, 2, 24, 20, FP32, 10)
    grads = pk.ops.gated_delta_rule_bwd(do, q, k, v, g, beta, 0.3, first, dlast)
    gen = torch.Generator(device="cuda").manual_seed(4)
    inputs = (q, k, v, g, beta, first)
    sizes = (0.1, 0.1, 0.5, 0.05, 0.1, 0.1)
    dirs = [s * torch.randn(x.shape, generator=gen, device="cuda") for s, x in zip(sizes, inputs)]
    step = 2.0 ** -6

    def value(e):
        o, s = pk.ops.gated_delta_rule_fwd(*(x + e * d for x, d in zip(inputs[:5], dirs)), 0.3, first + e * dirs[5])
        return float((o.double() * do).sum() + (s.double() * dlast).sum())
    o, s = pk.ops.gated_delta_rule_fwd(*inputs[:5], 0.3, first)
    terms = float((o.double() * do).abs().sum() + (s.double() * dlast).abs().sum())
    slope = float(sum((a.double() * d).sum() for a, d in zip(grads, dirs)))
    assert abs((value(step) - value(-step)) / (2 * step) - slope) <= (64 * U / step + 2.0 ** -10) * terms


def test_gated_delta_rule_under_autograd(pk):
    """The node gives what the direct backward gives, of one output alone too, for gradients that are not dense."""
    q, k, v, g, beta, first, do, dlast = delta_inputs(2, 80, 2, 4, 32, 32, BF16, 11, "fused")
    leaves = [x.detach().clone().requires_grad_() for x in (q, k, v, g, beta, first)]
    o, state = pk.ops.gated_delta_rule(*leaves[:5], 0.2, leaves[5])
    plain = [x.detach() for x in leaves]
    assert same(torch.autograd.grad([o, state], leaves, [do, dlast], retain_graph=True), pk.ops.gated_delta_rule_bwd(do, *plain[:5], 0.2, plain[5], dlast))
    assert same(torch.autograd.grad(o.sum(), leaves, retain_graph=True), pk.ops.gated_delta_rule_bwd(torch.ones_like(o), *plain[:5], 0.2, plain[5]))
    sideways = do.transpose(2, 3).contiguous().transpose(2, 3)
    assert torch.equal(torch.autograd.grad(o, leaves[0], sideways, retain_graph=True)[0], pk.ops.gated_delta_rule_bwd(do, *plain[:5], 0.2, plain[5])[0])
    far = dlast.transpose(2, 3).contiguous().transpose(2, 3)
    assert same(torch.autograd.grad(state, leaves, far, retain_graph=True), pk.ops.gated_delta_rule_bwd(torch.zeros_like(do), *plain[:5], 0.2, plain[5], dlast))
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(o.sum(), leaves[0], create_graph=True)
    o, _ = pk.ops.gated_delta_rule(*plain[:2], leaves[2], *plain[3:5], 0.2)
    assert torch.equal(torch.autograd.grad(o, leaves[2], do)[0], pk.ops.gated_delta_rule_bwd(do, *plain[:5], 0.2)[2])
    with torch.no_grad():
        assert not pk.ops.gated_delta_rule(*leaves[:5], 0.2)[0].requires_grad
    moved = plain[5].clone()
    kept = (moved.requires_grad_() * 1.0)
    z = kept * kept
    pk.ops.gated_delta_step_(*plain[:5], 0.2, kept.detach())   # a tensor that another node has saved
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.sum().backward()


def test_gated_delta_rule_past_2_to_the_31(pk):
    """Tokens 2^25 elements apart, the last of them past 2^31 elements of its tensor: what dense copies give, to the bit."""
    q, k, v, g, beta, first, do, dlast = delta_inputs(1, 70, 1, 1, 32, 32, BF16, 12)
    pitch = 1 << 25
    far = torch.zeros(70 * pitch, dtype=BF16, device="cuda")
    views = [far[64 * i:].as_strided(x.shape, (0, pitch, 0, 1)) for i, x in enumerate((q, k, v, do))]
    for y, x in zip(views, (q, k, v, do)):
        y.copy_(x)
    for T in (70, 7):   # by chunks; by tokens, the far ones
        part = lambda x: x[:, 70 - T:]  # noqa: E731
        near = [part(x).contiguous() for x in (q, k, v, g, beta, do)]
        away = [part(x) for x in views]
        scalars = (near[3], near[4], 0.2, first)
        assert same(pk.ops.gated_delta_rule_fwd(*away[:3], *scalars), pk.ops.gated_delta_rule_fwd(*near[:3], *scalars))
        assert same(pk.ops.gated_delta_rule_bwd(away[3], *away[:3], *scalars, dlast), pk.ops.gated_delta_rule_bwd(near[5], *near[:3], *scalars, dlast))


def test_gated_delta_step_of_states_past_2_to_the_31(pk):
    """140000 heads of states of 128 x 128, more than 2^31 elements: the last ones as by themselves."""
    B, H = 8750, 16
    q, k, v, g, beta, _, _, _ = delta_inputs(B, 1, 1, H, 128, 128, BF16, 13, state=False)
    state = torch.zeros(B, H, 128, 128, device="cuda")
    state[-1], state[0] = 0.1, -0.2
    want = [state[i:i + 1].clone() if i >= 0 else state[-1:].clone() for i in (0, -1)]
    o = pk.ops.gated_delta_step_(q, k, v, g, beta, 0.1, state)
    for i, w in zip((0, -1), want):
        at = slice(i, i + 1 if i >= 0 else None)
        assert torch.equal(o[at], pk.ops.gated_delta_step_(*(x[at] for x in (q, k, v, g, beta)), 0.1, w)) and torch.equal(state[at], w)


# ---- layer norm ----------------------------------------------------------------------------------------------------------

NORMS = [  # rows, cols, columns between rows, elements in front of the first
    (1, 1, 0, 0), (3, 2, 0, 0), (5, 7, 0, 0), (2, 8, 0, 0), (17, 64, 0, 0), (9, 511, 0, 0), (6, 512, 0, 0), (5, 513, 520, 0), (7, 1000, 1001, 1), (4, 1024, 0, 0), (3, 1025, 0, 0),
    (700, 300, 0, 0), (3100, 40, 0, 0), (5000, 2048, 0, 0), (2, 2049, 0, 0), (3, 4096, 4104, 3), (2, 5003, 0, 0), (2, 8192, 0, 0), (3, 8195, 0, 0), (2, 16384, 0, 0), (3, 16390, 0, 0),
    (400, 16400, 0, 0), (2, 32768, 0, 0), (2, 40001, 40007, 1), (1, 100000, 0, 0)]


def norm_inputs(rows, cols, pitch, front, dtype, seed=3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    wide = max(pitch, cols + front)
    part = lambda s=1.0: (torch.randn((rows, wide), generator=g, device="cuda") * s).to(dtype)[:, front:front + cols]  # noqa: E731
    x, r, dy, dh = part() + 0.5, part(2.0), part(), part()
    x = (x * torch.exp(torch.randn((rows, 1), generator=g, device="cuda"))).to(dtype)
    x = torch.nn.functional.pad(x, (front, wide - cols - front))[:, front:front + cols]
    w, b = 1 + 0.3 * torch.randn(cols, generator=g, device="cuda"), 0.5 * torch.randn(cols, generator=g, device="cuda")
    return x, r, w, b, dy, dh


def plain_norm(h, w, b, eps):
    """y, mean, rstd in 64 bits."""
    h = h.double()
    mean = h.mean(1, keepdim=True)
    rstd = torch.rsqrt((h - mean).square().mean(1, keepdim=True) + eps)
    y = (h - mean) * rstd * w.double()
    return y if b is None else y + b.double(), mean, rstd


def chain(cols):
    """Additions that a term of a row's sum goes through: 64 in a lane at most (a 1024th of a row past 65536), 6 in the wavefront, 16 over wavefronts."""
    return max(64, cols / 1024) + 22


@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("residual,bias", [(True, True), (False, False)], ids=["residual", "plain"])
@pytest.mark.parametrize("case", NORMS, ids=lambda c: "-".join(map(str, c)))
def test_layernorm_against_64_bits(pk, case, residual, bias, dtype):
    """mean: the chain's u times the mean size, dm. rstd: the squares' chain and 8 more u, relative, plus what the mean's error does to them, (dm rstd)^2. y: rstd's error and
    4 u of |xhat w|, dm rstd |w|, u of |b|.
    dx, from the kernel's own statistics: with A the largest |dy w| and X the largest |xhat| of the row (at least 1), du, xhat and the two means carry (chain + 8) u of
    A X at most, times |xhat| once more: 2 (chain + 8) u rstd A X^2. dw, db: a term goes through a step's addition for each of its walk's rows (a 256th of all and one, at most),
    2 or 4 walks, a 16th of 768 workgroups' sums, 16 of those; 4 u of each term besides."""
    rows, cols, pitch, front = case
    x, r, w, b, dy, dh = norm_inputs(rows, cols, pitch, front, dtype)
    b, r, eps, h = b if bias else None, r if residual else None, 1e-5, HALF[dtype]
    kept = [t.clone() for t in (x, dy, dh)]
    y, held, mean, rstd = pk.ops.layernorm_fwd(x, w, b, eps, r)
    if residual:
        assert torch.equal(held, (x.float() + r.float()).to(dtype))
    else:
        assert held.data_ptr() == x.data_ptr()
    assert y.dtype == dtype and mean.dtype == rstd.dtype == FP32
    want, wm, wr = plain_norm(held, w, b, eps)
    n, size = chain(cols), held.double().abs().mean(1, keepdim=True)
    dm = (n * U * size + U * wm.abs())
    dr = ((n + 8) * U + (dm * wr) ** 2)
    unit = (held.double() - wm) * wr
    within("mean", mean, wm[:, 0], dm[:, 0])
    within("rstd", rstd, wr[:, 0], (wr * dr)[:, 0])
    within("y", y, want, h * want.abs() + (dr + 4 * U) * (unit * w).abs() + 2 * dm * wr * w.abs() + (U * b.abs() if bias else 0.0))
    dx, dw, db = pk.ops.layernorm_bwd(dy, held, w, mean, rstd, dh if residual else None)
    assert same(kept, (x, dy, dh)) and dx.dtype == dtype and dw.dtype == db.dtype == FP32
    m, s, d = mean.double()[:, None], rstd.double()[:, None], dy.double()
    unit = (held.double() - m) * s
    du = d * w
    gx = s * (du - du.mean(1, keepdim=True) - unit * (du * unit).mean(1, keepdim=True))
    if residual:
        gx = gx + dh.double()
    A, X = du.abs().amax(1, keepdim=True), unit.abs().amax(1, keepdim=True).clamp(min=1.0)
    within("dx", dx, gx, h * gx.abs() + 2 * (n + 8) * U * s * A * X * X + (2 * U * dh.double().abs() if residual else 0.0))
    terms = rows / 256 + 1 + 4 + 48 + 16 + 4
    within("dw", dw, (d * unit).sum(0), terms * U * (d * unit).abs().sum(0))
    within("db", db, d.sum(0), terms * U * d.abs().sum(0))


def test_layernorm_gradient_against_differences(pk):
    """The derivative of sum(y dy) + sum(h dh) along a direction against a central difference of the operator itself in fp32: two sums of n values, each within 100 u of its
    terms' largest, over a step of 2^-6; the third-order term of the step is below 2^-12 of the sum."""
    x, r, w, b, dy, dh = norm_inputs(7, 129, 0, 0, FP32)
    y, h, mean, rstd = pk.ops.layernorm_fwd(x, w, b, 1e-5, r)
    dx, dw, db = pk.ops.layernorm_bwd(dy, h, w, mean, rstd, dh)
    g = torch.Generator(device="cuda").manual_seed(8)
    dirs = [torch.randn(t.shape, generator=g, device="cuda") for t in (x, r, w, b)]
    step = 2.0 ** -6

    def value(e):
        y, h, _, _ = pk.ops.layernorm_fwd(x + e * dirs[0], w + e * dirs[2], b + e * dirs[3], 1e-5, r + e * dirs[1])
        return float((y.double() * dy).sum() + (h.double() * dh).sum())
    slope = float(sum((a.double() * d).sum() for a, d in zip((dx, dx, dw, db), dirs)))
    terms = float((y.double() * dy).abs().sum() + (h.double() * dh).abs().sum())
    assert abs((value(step) - value(-step)) / (2 * step) - slope) <= 100 * U * terms / step + 2.0 ** -12 * terms


def test_layernorm_extremes(pk):
    """Rows of one value (variance 0), of values far from zero, of numbers that are none: each row by itself. No rows at all: sums of nothing."""
    for dtype in (FP32, BF16):
        x, _, w, b, dy, _ = norm_inputs(8, 777, 0, 0, dtype)
        x = x.clone()
        want, _, _, _ = pk.ops.layernorm_fwd(x, w, b)
        x[1], x[2, 5], x[3, 0], x[4] = 3.0, math.nan, math.inf, 1e4 + x[4]
        y, _, mean, rstd = pk.ops.layernorm_fwd(x, w, b)
        assert torch.equal(y[[0, 5, 6, 7]], want[[0, 5, 6, 7]])
        assert bool(torch.isnan(y[2:4].float()).all())
        within("flat", y[1:2], b[None].double(), HALF[dtype] * b[None].double().abs())
        assert float(mean[1]) == 3.0 and abs(float(rstd[1]) - 1e-5 ** -0.5) < 1e-4
        far, wm, wr = plain_norm(x[4:5], w, b, 1e-5)
        dm = chain(777) * U * wm.abs()
        within("far", y[4:5], far, HALF[dtype] * far.abs() + 2 * dm * wr * w.abs() + (chain(777) + 12) * U * far.abs().amax() + (dm * wr) ** 2 * far.abs().amax())
        dx, dw, db = pk.ops.layernorm_bwd(dy, x, w, mean, rstd)
        assert bool(torch.isfinite(dx[[0, 1, 4, 5, 6, 7]].float()).all()) and bool(torch.isnan(dx[2:4].float()).all()) and bool(torch.isfinite(db).all())
        e = x[:0]
        y, h, mean, rstd = pk.ops.layernorm_fwd(e, w, b, residual=e)
        dx, dw, db = pk.ops.layernorm_bwd(e, h, w, mean, rstd, e)
        assert y.shape == h.shape == dx.shape == (0, 777) and not dw.any() and not db.any() and dw.shape == (777,)


def test_layernorm_rows_do_not_depend_on_the_batch(pk):
    for dtype in (FP32, BF16):
        x, r, w, b, _, _ = norm_inputs(300, 512, 0, 0, dtype)
        y, h, mean, rstd = pk.ops.layernorm_fwd(x, w, b, 1e-5, r)
        for i in (0, 77, 299):
            assert same([t[i:i + 1] for t in (y, h, mean, rstd)], pk.ops.layernorm_fwd(x[i:i + 1], w, b, 1e-5, r[i:i + 1]))
    one = x[:1].expand(5, 512)   # one row for all
    y = pk.ops.layernorm_fwd(one, w, b)[0]
    assert torch.equal(y, pk.ops.layernorm_fwd(one.contiguous(), w, b)[0])


def test_layernorm_under_autograd(pk):
    """The node gives what the direct backward gives, with and without a residual, of one output alone, for gradients that are not dense."""
    x, r, w, b, dy, dh = norm_inputs(19, 136, 0, 0, BF16)
    leaves = [t.detach().clone().requires_grad_() for t in (x, w, b, r)]
    y, h = pk.ops.layernorm(leaves[0], leaves[1], leaves[2], 1e-5, leaves[3])
    _, held, mean, rstd = pk.ops.layernorm_fwd(x, w, b, 1e-5, r)
    dx, dw, db = pk.ops.layernorm_bwd(dy, held, w, mean, rstd, dh)
    assert same(torch.autograd.grad([y, h], leaves, [dy, dh], retain_graph=True), (dx, dw, db, dx))
    assert torch.equal(torch.autograd.grad(h, leaves[0], dh, retain_graph=True)[0], dh)
    dx, dw, _ = pk.ops.layernorm_bwd(torch.ones_like(dy), held, w, mean, rstd)
    assert same(torch.autograd.grad(y.sum(), leaves[:2], retain_graph=True), (dx, dw))
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(y.sum(), leaves[0], create_graph=True)
    only = pk.ops.layernorm(x, leaves[1])
    _, _, mean, rstd = pk.ops.layernorm_fwd(x, w)
    assert torch.equal(torch.autograd.grad(only, leaves[1], dy.t().contiguous().t())[0], pk.ops.layernorm_bwd(dy, x, w, mean, rstd)[1])
    with torch.no_grad():
        assert not pk.ops.layernorm(*leaves[:3]).requires_grad
    h.detach().add_(1.0)   # what the backward needs is no longer what it was
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


# ---- distillation --------------------------------------------------------------------------------------------------------


TOPS = [  # rows, vocab, words, columns between rows, elements in front of the first
    (1, 1, 1, 0, 0), (3, 2, 2, 0, 0), (5, 7, 3, 0, 0), (9, 64, 9, 0, 0), (4, 511, 20, 512, 1), (33, 1000, 5, 0, 0), (2, 2048, 64, 0, 0), (3, 4097, 65, 0, 0), (2, 8200, 130, 0, 0),
    (3, 10007, 200, 10016, 3), (2, 17000, 64, 0, 0), (3, 32003, 20, 0, 0), (2, 65536, 1024, 0, 0), (2, 70001, 64, 0, 0), (1, 150001, 7, 0, 0), (700, 333, 12, 0, 0)]


def distill_inputs(rows, vocab, top, dtype, seed=5, pitch=0, front=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = torch.randn((rows, vocab), generator=g, device="cuda") * 2.5
    best = t.topk(top, 1)
    x = torch.nn.functional.pad((0.8 * t + torch.randn((rows, vocab), generator=g, device="cuda")).to(dtype), (front, max(0, pitch - vocab - front)))[:, front:front + vocab]
    w = torch.rand(rows, generator=g, device="cuda") / rows
    return x, best.indices.to(torch.int32).contiguous(), best.values.contiguous(), w, torch.logsumexp(t.double(), 1).float()


def plain_distill(x, idx, t, w, tau, lse, upstream):
    """loss, gradient, KL, and beside them P q and p word by word, in 64 bits."""
    rows, vocab = x.shape
    logq = torch.log_softmax(x.double() / tau, 1)
    slot = idx >= 0
    t = torch.where(slot, t.double() / tau, -math.inf)
    logp = t - (torch.logsumexp(t, 1, keepdim=True) if lse is None else lse.double()[:, None])
    p = torch.where(slot, torch.exp(logp), 0.0)
    at = idx.clamp(min=0).long()
    kl = torch.where(p == 0, torch.zeros_like(p), p * (logp - logq.gather(1, at))).sum(1)
    counts = (w != 0) & slot.any(1)
    kl = torch.where(counts, kl, 0.0)
    spread = torch.zeros_like(logq).scatter_add_(1, at, p)
    mass = p.sum(1, keepdim=True) * torch.exp(logq)
    coef = torch.where(counts, w.double() * tau * upstream, 0.0)[:, None]
    grad = torch.where(coef != 0, coef * (mass - spread), 0.0)
    return tau * tau * torch.where(counts, w.double() * kl, 0.0).sum(), grad, kl, coef, mass, spread, logq


def check_distill(pk, x, idx, t, w, tau, lse=None, upstream=1.0):
    """q in 32-bit arithmetic: the exponent's difference from the largest logit and its product carry 2 u of their size S, the exponential 2 u, a sum's chain vocab/64 and
    8 more additions: e = (3 S + 14 + vocab / 64) u of q, and of a log-probability. KL is formed and added up in 64 bits from that one sum and rounded: P e + u |KL|.
    The gradient: coef (P q e + 4 u P q + 4 u p), and its rounding."""
    dtype, vocab = x.dtype, x.shape[1]
    kept = x.clone()
    loss, d, kl = pk.blockops.distill_loss(x, idx, t, w, tau, lse, upstream)
    assert torch.equal(bits(x), bits(kept)) and d.dtype == dtype and kl.dtype == loss.dtype == FP32
    wl, wg, wk, coef, mass, spread, logq = plain_distill(x, idx, t, w, tau, lse, upstream)
    S = torch.where(torch.isfinite(x), x.double() / tau, 0.0)
    S = (S.amax(1) - S.amin(1)).clamp(min=1.0)
    e = (3 * S + 14 + vocab / 64) * U
    P = spread.sum(1)
    within("kl", kl, wk, P * e + U * wk.abs())
    within("loss", loss, wl, U * wl.abs() + tau * tau * (w.double() * (P * e)).nansum())
    within("dlogits", d, wg, HALF[dtype] * wg.abs() + coef.abs() * (mass * (e[:, None] + 4 * U) + 4 * U * spread) + 1e-37)
    alone, none, kl1 = pk.blockops.distill_loss(x, idx, t, w, tau, lse, upstream, grad=False)
    assert none is None and same((alone, kl1), (loss, kl))
    over = x.clone()
    got = pk.blockops.distill_loss(over, idx, t, w, tau, lse, upstream, out=over)
    assert got[1].data_ptr() == over.data_ptr()
    # a row that begins elsewhere is taken apart elsewhere: the same values within the counts
    within("over", over, wg, HALF[dtype] * wg.abs() + coef.abs() * (mass * (e[:, None] + 4 * U) + 4 * U * spread) + 1e-37)
    return loss, d, kl


@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("tail,tau", [(False, 1.0), (True, 1.0), (False, 2.5), (False, 0.7)], ids=["top", "tail", "warm", "cool"])
@pytest.mark.parametrize("case", TOPS, ids=lambda c: "-".join(map(str, c)))
def test_distill_loss_against_64_bits(pk, case, tail, tau, dtype):
    rows, vocab, top, pitch, front = case
    x, idx, t, w, lse = distill_inputs(rows, vocab, top, dtype, 5, pitch, front)
    if rows > 2:
        w[1] = 0.0
    if rows > 3 and top > 2:
        idx[2, 1::2], idx[0, :-1] = -1, -1
        idx[3] = -1                       # a row that nothing is learned from
    check_distill(pk, x, idx, t, w, tau, lse if tail else None, 0.5 if tail else 1.0)


@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("vocab", [50, 5000, 80001])
def test_distill_loss_of_a_word_in_several_slots(pk, vocab, dtype):
    x, idx, t, w, _ = distill_inputs(6, vocab, 12, dtype, 6)
    idx[0] = idx[0, 0]
    idx[1, 6:] = idx[1, :6]
    idx[2, ::3] = vocab - 1
    idx[3, 4:9] = 0
    check_distill(pk, x, idx, t, w, 1.0)


@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("vocab", [60, 3001, 70001])
def test_distill_loss_of_ruled_out_words(pk, vocab, dtype):
    """Logits of -inf: the student's, which make a KL infinite only where the teacher gives such a word something; the teacher's, which add nothing. Rows that hold no number,
    words past the vocabulary and teachers without a probability make their own row's results none."""
    x, idx, t, w, lse = distill_inputs(8, vocab, 6, dtype, 7)
    x = x.clone()
    low = x[:, :].topk(3, 1, largest=False).indices
    for r in range(8):
        x[r, [i for i in low[r].tolist() if i not in idx[r].tolist()]] = -math.inf
    t[1, 2], t[2, :5] = -math.inf, -math.inf
    x[1, int(idx[1, 2])] = -math.inf      # nobody wants it
    check_distill(pk, x, idx, t, w, 1.0)
    want = pk.blockops.distill_loss(x, idx, t, w)
    x[3, int(idx[3, 0])] = -math.inf      # the teacher does
    idx[4, 1] = vocab
    t[5] = -math.inf
    x[6, 3] = math.nan
    x[7] = -math.inf
    loss, d, kl = pk.blockops.distill_loss(x, idx, t, w)
    assert float(kl[3]) == math.inf and bool(torch.isfinite(d[3].float()).all()) and bool(torch.isnan(kl[4:]).all()) and bool(torch.isnan(loss))
    assert torch.equal(kl[:3], want[2][:3]) and torch.equal(bits(d[:3]), bits(want[1][:3])) and bool(torch.isnan(d[5:].float()).all())
    p3 = torch.softmax(t[3].double(), 0)[0]
    assert abs(float(d[3, int(idx[3, 0])]) + float(w[3] * p3)) <= 2 * HALF[dtype] * float(w[3] * p3)
    w2 = w.clone()
    w2[3:] = 0.0                          # rows that do not count are not read
    loss, d, kl = pk.blockops.distill_loss(x, idx, t, w2)
    assert not kl[3:].any() and not d[3:].any() and bool(torch.isfinite(loss))


def test_distill_loss_of_far_logits_and_likely_words(pk):
    """Logits far from zero, and a student that gives one word nearly everything: KL to what the counts of 64-bit sums allow."""
    for dtype in (FP32, BF16):
        for base in (0.0, 3e4, -3e4):
            x, idx, t, w, _ = distill_inputs(5, 9000, 8, FP32, 9)
            x, t = (x + base).to(dtype), t + base / 2
            x[2, int(idx[2, 0])] += 512.0 if base else 60.0
            check_distill(pk, x.contiguous(), idx, t.contiguous(), w, 1.0)


def test_distill_loss_of_nothing(pk):
    x, idx, t, w, _ = distill_inputs(4, 100, 3, BF16)
    loss, d, kl = pk.blockops.distill_loss(x[:0], idx[:0], t[:0], w[:0])
    assert float(loss) == 0.0 and d.shape == (0, 100) and kl.shape == (0,)
    loss, d, kl = pk.blockops.distill_loss(x, idx, t, torch.zeros_like(w))
    assert float(loss) == 0.0 and not d.any() and not kl.any()


def test_distill_loss_gradient_against_differences(pk):
    """A central difference of the loss alone along a direction, in fp32 logits: the loss carries 100 u of its terms, over a step of 2^-5; the third-order term is below
    2^-12 of sum |coef| times the direction's largest cubed (5 sigma at most: 125)."""
    x, idx, t, w, lse = distill_inputs(6, 300, 10, FP32, 11)
    g = torch.Generator(device="cuda").manual_seed(12)
    v = torch.randn(x.shape, generator=g, device="cuda").clamp(-2, 2)
    step = 2.0 ** -5
    for extra in (None, lse):
        _, d, _ = pk.blockops.distill_loss(x, idx, t, w, 2.0, extra)
        up, down = (float(pk.blockops.distill_loss(x + s * v, idx, t, w, 2.0, extra, grad=False)[0]) for s in (step, -step))
        assert abs((up - down) / (2 * step) - float((d.double() * v).sum())) <= (100 * U / step + step ** 2 * 8) * float(w.sum()) * 4


# ---- all of them -----------------------------------------------------------------------------------------------------------


def test_norm_and_distill_under_graph_capture(pk):
    """Recorded and replayed three times on new inputs, with eager calls of the same between the replays: each replay has the eager bits."""
    x, r, w, b, dy, dh = norm_inputs(300, 512, 0, 0, BF16)
    z, idx, t, weights, _ = distill_inputs(40, 5003, 16, BF16)

    def calls():
        y, h, mean, rstd = pk.ops.layernorm_fwd(x, w, b, 1e-5, r)
        return [y, h, *pk.ops.layernorm_bwd(dy, h, w, mean, rstd, dh), *pk.blockops.distill_loss(z, idx, t, weights, 2.0)]
    graph, out = graph_of(calls)
    for k in range(3):
        g = torch.Generator(device="cuda").manual_seed(50 + k)
        for tensor in (x, r, dy, dh, z):
            tensor.copy_(torch.randn(tensor.shape, generator=g, device="cuda"))
        want = [o.clone() for o in calls()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert same(out, want), k


@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
def test_gated_delta_rule_under_graph_capture(pk, dtype):
    """By chunks, back, and a token that moves a state on, recorded and replayed on new inputs between eager calls: each replay has the eager bits."""
    q, k, v, g, beta, first, do, dlast = delta_inputs(2, 150, 2, 4, 64, 48, dtype, 20)
    token = [x[:, 5:6].contiguous() for x in (q, k, v, g, beta)]
    moved = torch.empty_like(first)

    def calls():
        torch.add(first, 0.0, out=moved)
        o = pk.ops.gated_delta_step_(*token, 0.2, moved)
        return [o, moved + 0.0, *pk.ops.gated_delta_rule_fwd(q, k, v, g, beta, 0.2, first), *pk.ops.gated_delta_rule_bwd(do, q, k, v, g, beta, 0.2, first, dlast)]
    graph, out = graph_of(calls)
    for seed in range(3):
        for old, new in zip((q, k, v, g, beta, first, do, dlast), delta_inputs(2, 150, 2, 4, 64, 48, dtype, 30 + seed)):
            old.copy_(new)
        for old, new in zip(token, (q, k, v, g, beta)):
            old.copy_(new[:, seed:seed + 1])
        want = [x.clone() for x in calls()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert same(out, want), seed


def test_backward_passes_under_graph_capture(pk):
    """Both nodes recorded with their forwards and replayed between eager calls. While an eager graph of the same leaves lives, their gradients belong to its stream, which must
    not wait for a recording: refused, and the next recording stands."""
    *rule, do, dlast = delta_inputs(2, 90, 2, 4, 32, 32, BF16, 21)
    x, r, w, b, dy, dh = norm_inputs(64, 96, 0, 0, FP32)
    rule, norm = [y.detach().clone().requires_grad_() for y in rule], [y.detach().clone().requires_grad_() for y in (x, w, b, r)]

    def mixed():
        return torch.autograd.grad(pk.ops.gated_delta_rule(*rule[:5], 0.2, rule[5]), rule, [do, dlast])

    def normed():
        return torch.autograd.grad(pk.ops.layernorm(norm[0], norm[1], norm[2], 1e-5, norm[3]), norm, [dy, dh])

    for leaves, fn, alive in ((rule, mixed, lambda: pk.ops.gated_delta_rule(*rule[:5], 0.2, rule[5])), (norm, normed, lambda: pk.ops.layernorm(*norm[:3], 1e-5, norm[3]))):
        lives = alive()
        with pytest.raises(RuntimeError, match="outside of the recording"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                fn()
        del lives
        graph, out = graph_of(fn)
        gen = torch.Generator(device="cuda").manual_seed(2)
        for _ in range(3):
            with torch.no_grad():
                for y in leaves[:3]:
                    y.copy_(torch.nn.functional.normalize(torch.randn(y.shape, generator=gen, device="cuda"), dim=-1))
            want = fn()
            graph.replay()
            torch.cuda.synchronize()
            assert same(out, want)


def test_student_operators_on_two_streams_at_once(pk):
    """The same calls queued on two streams over different inputs: the results of one after the other."""
    sets = [(delta_inputs(2, 500, 2, 4, 64, 64, BF16, seed), norm_inputs(700, 512, 0, 0, BF16, seed), distill_inputs(100, 9000, 20, BF16, seed)) for seed in (1, 2)]

    def work(s):
        (q, k, v, g, beta, first, do, dlast), (x, r, w, b, dy, dh), (z, idx, t, weights, _) = s
        y, h, mean, rstd = pk.ops.layernorm_fwd(x, w, b, 1e-5, r)
        return [*pk.ops.gated_delta_rule_fwd(q, k, v, g, beta, 0.2, first), *pk.ops.gated_delta_rule_bwd(do, q, k, v, g, beta, 0.2, first, dlast), y, h,
                *pk.ops.layernorm_bwd(dy, h, w, mean, rstd, dh), *pk.blockops.distill_loss(z, idx, t, weights, 2.0)]
    want = [work(s) for s in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], [None, None]
    for _ in range(3):
        for i, (st, s) in enumerate(zip(streams, sets)):
            with torch.cuda.stream(st):
                got[i] = work(s)
    torch.cuda.synchronize()
    assert all(same(a, b) for a, b in zip(got, want))


def test_student_operators_refuse(pk):
    """What the C entries cannot see: types, devices, shapes of tensors that belong together, strides."""
    q, k, v, g, beta, first, do, dlast = delta_inputs(2, 20, 2, 4, 32, 32, BF16, 22)
    rule = pk.ops.gated_delta_rule_fwd
    for bad in ((q.float(), k, v, g, beta, 1.0), (q, k[:, :9], v, g, beta, 1.0), (q, k, v[:1], g, beta, 1.0), (q, k, v[:, :, :3], g[..., :3], beta[..., :3], 1.0), (q, k, v, g.double(), beta, 1.0),
                (q, k, v, g[:, :9], beta, 1.0), (q, k, v, g, beta.transpose(0, 1), 1.0), (q.transpose(2, 3), k.transpose(2, 3), v, g, beta, 1.0), (q.cpu(), k.cpu(), v.cpu(), g, beta, 1.0),
                (q, k, v, g, beta, math.inf), (q, k, v, g, beta, 1.0, first.double()), (q, k, v, g, beta, 1.0, first[:1]), (q, k, v, g, beta, 1.0, first.transpose(2, 3)),
                (q.half(), k.half(), v.half(), g, beta, 1.0), (q, k, v.cpu(), g, beta, 1.0), (q, k, v, g.cpu(), beta, 1.0)):
        with pytest.raises(RuntimeError):
            rule(*bad)
    for bad in (dict(d_o=do[:, :9]), dict(d_o=do.float()), dict(d_state=dlast[:1]), dict(d_state=dlast.transpose(2, 3)), dict(initial_state=first.to(BF16))):
        with pytest.raises(RuntimeError):
            pk.ops.gated_delta_rule_bwd(**{**dict(d_o=do, q=q, k=k, v=v, g=g, beta=beta, scale=1.0, initial_state=first, d_state=dlast), **bad})
    kept = first.clone()
    for state in (first.clone().requires_grad_(), first[:1].expand(2, -1, -1, -1), first.cpu()):
        with pytest.raises(RuntimeError):
            pk.ops.gated_delta_step_(q, k, v, g, beta, 1.0, state)
    assert torch.equal(first, kept)
    x, r, w, b, dy, dh = norm_inputs(6, 32, 0, 0, BF16)
    for bad in ((x, w[:9], b), (x, w.to(BF16), b), (x, w, b[:9]), (x, w, b, -1.0), (x, w, b, 1e-5, r[:3]), (x, w, b, 1e-5, r.float()), (x.t(), w[:6], b[:6]), (x.cpu(), w, b), (x[0], w, b)):
        with pytest.raises(RuntimeError):
            pk.ops.layernorm_fwd(*bad)
    z, idx, t, weights, lse = distill_inputs(6, 50, 4, FP32)
    for bad in (dict(indices=idx.long()), dict(indices=idx[:3]), dict(teacher_logits=t.double()), dict(teacher_logits=t[:, :2]), dict(weights=weights[:3]), dict(temperature=0.0),
                dict(teacher_lse=lse[:3]), dict(out=z.to(BF16)), dict(out=z[:3]), dict(logits=z.t()), dict(logits=z.half()), dict(logits=z.cpu()), dict(upstream=math.nan)):
        with pytest.raises(RuntimeError):
            pk.blockops.distill_loss(**{**dict(logits=z, indices=idx, teacher_logits=t, weights=weights), **bad})


def test_a_student_step_through_all_operators(pk):
    """A layer of norm, gated delta rule and residual norm, a head, the loss against a teacher's top logits, and the optimiser, in fp32: loss, gradients of all eight
    parameters and the parameters after the step against the same model in 64 bits; then the stepped model token by token against itself over the whole sequence. The longest
    chain is twelve operators, each 64 u of its result's largest at most: 2^-14."""
    B, T, Hk, Hv, dk, dv, V, top, d = 2, 70, 2, 4, 16, 24, 211, 12, 64
    near = 2.0 ** -14
    gen = torch.Generator().manual_seed(14)
    randn = lambda *s: torch.randn(s, generator=gen)  # noqa: E731
    cut = [Hk * dk, Hk * dk, Hv * dv, Hv, Hv]
    params = {"emb": randn(V, d), "w1": 1 + 0.2 * randn(d), "b1": 0.2 * randn(d), "in": randn(d, sum(cut)) / 8, "out": randn(Hv * dv, d) / 10, "w2": 1 + 0.2 * randn(d), "b2": 0.2 * randn(d),
              "head": randn(d, V) / 8}
    ids = torch.randint(0, V, (B, T), generator=gen)
    best = (2.5 * randn(B * T, V)).topk(top, 1)
    weights = (torch.rand(B * T, generator=gen) > 0.2).float() / 100

    def model(P, ids, norm, rule):
        x = P["emb"][ids]
        n = x.shape[1]
        z = norm(x.view(-1, d), P["w1"], P["b1"], None).view(B, n, -1)
        q, k, v, g, beta = z.matmul(P["in"]).split(cut, 2)
        q, k = (torch.nn.functional.normalize(y.unflatten(2, (Hk, dk)), dim=-1) for y in (q, k))
        o = rule(q, k, v.unflatten(2, (Hv, dv)), -torch.nn.functional.softplus(g), torch.sigmoid(beta))
        return norm(o.reshape(B * n, -1) @ P["out"], P["w2"], P["b2"], x.view(-1, d)) @ P["head"]

    def plain_normed(x, w, b, residual):
        x = x if residual is None else x + residual
        return torch.nn.functional.layer_norm(x, (d,), w, b, 1e-5)

    P64 = {n: p.double().requires_grad_() for n, p in params.items()}
    logits = model(P64, ids, plain_normed, lambda q, k, v, g, beta: plain_delta(q, k, v, g, beta, 0.25)[0])
    logp, logq = torch.log_softmax(best.values.double() / 2, 1), torch.log_softmax(logits / 2, 1).gather(1, best.indices)
    want_loss = 4 * (weights.double() * (logp.exp() * (logp - logq)).sum(1)).sum()
    want = torch.autograd.grad(want_loss, list(P64.values()))

    def normed(x, w, b, residual):
        y = pk.ops.layernorm(x, w, b, 1e-5, residual)
        return y if residual is None else y[0]
    leaves = {n: p.cuda().requires_grad_() for n, p in params.items()}
    out = model(leaves, ids.cuda(), normed, lambda *a: pk.ops.gated_delta_rule(*a, 0.25)[0])
    loss, dlogits, _ = pk.blockops.distill_loss(out.detach(), best.indices.to(torch.int32).cuda(), best.values.cuda(), weights.cuda(), 2.0)
    out.backward(dlogits)
    assert abs(float(loss) - float(want_loss.detach())) <= near * float((4 * weights).sum())
    for (n, leaf), ref in zip(leaves.items(), want):
        assert float((leaf.grad.double().cpu() - ref).abs().max()) <= near * float(ref.abs().max()), n
    ps, gs = [leaf.detach() for leaf in leaves.values()], [leaf.grad for leaf in leaves.values()]
    pk.blockops.adamw_many_(ps, gs, pk.blockops.adamw_state(ps), 0.01, eps=1e-3)
    for (n, leaf), ref, p in zip(leaves.items(), want, params.values()):
        step = ref / (ref.abs() + 1e-3)   # m / c1 = g and sqrt(v / c2) = |g| at the first step
        slack = 0.01 * (near * float(ref.abs().max()) / 1e-3 + 2.0 ** -18) + 2.0 ** -22 * float(p.abs().max())
        assert float((leaf.detach().double().cpu() - (p.double() - 0.01 * (step + 0.01 * p.double()))).abs().max()) <= slack, n
    with torch.no_grad():
        whole = model(leaves, ids.cuda(), normed, lambda *a: pk.ops.gated_delta_rule(*a, 0.25)[0]).view(B, T, V)
        state = torch.zeros(B, Hv, dk, dv, device="cuda")
        tokens = [model(leaves, ids[:, t:t + 1].cuda(), normed, lambda *a: pk.ops.gated_delta_step_(*a, 0.25, state)) for t in range(T)]
        assert float((torch.stack(tokens, 1) - whole).abs().max()) <= near * float(whole.abs().max())
