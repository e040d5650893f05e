"""The operators of a student model on the GPU against plain implementations in 64 bits: layer norm with the residual addition, distillation from a teacher's top
logits.

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
