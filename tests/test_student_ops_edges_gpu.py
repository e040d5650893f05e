"""The operators of a student model at the edges of what they promise, on the GPU against 64 bits: bf16 tensors whose sums nearly cancel, words that are none, tall and far
inputs. Tolerances are counted as in test_student_ops_gpu.py: u = 2^-24, h half a step of the output's type."""
from __future__ import annotations

import math

import pytest
import torch

from test_post_ops_gpu import BF16, F64, FP32, HALF, U, within
from test_student_ops_gpu import bits, close, delta_inputs, distill_inputs, pk, plain_delta  # noqa: F401  (pk: a fixture)

pytestmark = pytest.mark.gpu


# ---- gated delta rule ----------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("heads", [2, 256], ids=["few", "many"])   # workgroups of 16 and of 32 columns
@pytest.mark.parametrize("T,dk,dv", [(32, 32, 32), (50, 64, 64), (64, 128, 96), (60, 100, 40), (64, 67, 33)])
def test_gated_delta_rule_of_bf16_where_sums_cancel(pk, T, dk, dv, heads):
    """Every token's key is a unit vector of its own and beta is 1, so the row of the state that a key names becomes the token's v: o is scale * v for a query that names the
    same row, as the difference of what the state before the chunk gives and what the chunk takes from it, both 2^10 times as large. dq likewise. With queries and gradients of
    one element every product of a state has one term: scale and the product's three parts 4 u, those of A 3 u, of U 1 u, what the parts leave out 3 u, six additions and the two
    sums' 8 u: 16 u of either term, and the rounding to bf16. (Two parts of a state would be 2^-17 of it off, 128 u.)"""
    gen = torch.Generator(device="cuda").manual_seed(T + dk)
    randn = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    one = lambda i, n: torch.nn.functional.one_hot(i, n).to(BF16)    # noqa: E731
    rows = torch.stack([torch.randperm(dk, generator=gen, device="cuda")[:T] for _ in range(heads)], 1)   # [T, heads]
    pick = torch.gather(rows, 0, (torch.rand((T, heads), generator=gen, device="cuda") * (torch.arange(T, device="cuda")[:, None] + 1)).long())   # a row that is v by then
    q, k = one(pick, dk)[None], one(rows, dk)[None]
    v, first = (randn(1, T, heads, dv) * 2.0 ** -10).to(BF16), randn(1, heads, dk, dv)
    do = one(torch.randint(dv, (T, heads), generator=gen, device="cuda"), dv)[None]
    beta, g = torch.ones(1, T, heads, device="cuda"), torch.zeros(1, T, heads, device="cuda")
    scale = 0.1
    (wo, ws), want = plain_delta(q, k, v, g, beta, scale, first, do)
    o, state = pk.ops.gated_delta_rule_fwd(q, k, v, g, beta, scale, first)
    dq = pk.ops.gated_delta_rule_bwd(do, q, k, v, g, beta, scale, first)[0]
    before = scale * torch.einsum("bthk,bhkv->bthv", q.double(), first.double()).abs()   # what the state gives; the chunk's part is as large
    within("o", o, wo, HALF[BF16] * wo.abs() + 16 * U * (2 * before + wo.abs()))
    given = scale * torch.einsum("bhkv,bthv->bthk", first.double(), do.double()).abs()
    within("dq", dq, want[0], HALF[BF16] * want[0].abs() + 16 * U * (2 * given + want[0].abs()))
    assert float(wo.abs().max()) < 2.0 ** -7 * float(before.max())


@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("T,n", [(190, 184), (100, 65), (72, 64), (200, 64), (64, 9), (8, 5), (3, 1)])
def test_gated_delta_rule_padding_leaves_the_state_to_the_bit(pk, T, n, dtype):
    """Tokens of g 0 and beta 0 behind the last of n, whatever finite q, k and v they have: o and the state of the n alone, where both go by chunks or both by tokens."""
    q, k, v, g, beta, first, do, dlast = delta_inputs(2, T, 2, 4, 48, 40, dtype, 19)
    g[:, n:], beta[:, n:] = 0.0, 0.0
    v[:, n:] = 1e3
    o, state = pk.ops.gated_delta_rule_fwd(q, k, v, g, beta, 0.2, first)
    part = [x[:, :n].contiguous() for x in (q, k, v, g, beta)]
    want = pk.ops.gated_delta_rule_fwd(*part, 0.2, first)
    assert torch.equal(bits(o[:, :n]), bits(want[0])) and torch.equal(bits(state), bits(want[1]))
    do[:, n:] = 0.0
    grads = pk.ops.gated_delta_rule_bwd(do, q, k, v, g, beta, 0.2, first, dlast)
    alone = pk.ops.gated_delta_rule_bwd(do[:, :n].contiguous(), *part, 0.2, first, dlast)
    assert not grads[0][:, n:].any() and not grads[1][:, n:].any() and not grads[2][:, n:].any()
    for name, a, b in zip(("dq", "dk", "dv", "dg", "dbeta"), grads, alone):
        close(name, a[:, :n], b, dtype, 1.0, 48, 2.0 ** 8)
    close("dstate", grads[5], alone[5], dtype)


def test_gated_delta_rule_between_the_columns_of_one_buffer(pk):
    """The C entries with every tensor of heads between the others' columns, sequences in reverse order in memory: what dense tensors give, to the bit."""
    B, T, Hk, Hv, dk, dv = 3, 80, 2, 4, 32, 40
    q, k, v, g, beta, first, do, dlast = delta_inputs(B, T, Hk, Hv, dk, dv, BF16, 16)
    C, L, shape = pk.lib.C, pk.lib.lib(), pk.lib.DeltaShape(B, T, Hk, Hv, dk, dv, pk.lib.PK_BF16, 0.25)
    widths = [Hk * dk, Hk * dk, Hv * dv, Hv * dv, Hv * dv, Hk * dk, Hk * dk, Hv * dv]   # q, k, v, o, d_o, dq, dk, dv
    whole, row = torch.zeros(B, T, sum(widths), dtype=BF16, device="cuda"), sum(widths)
    parts = [x.unflatten(2, (-1, d)) for x, d in zip(whole.split(widths, 2), (dk, dk, dv, dv, dv, dk, dk, dv))]
    for part, x in zip(parts, (q, k, v, None, do)):
        if x is not None:
            part.copy_(x.flip(0))
    place = lambda p: C.byref(pk.lib.Tensor4(p[B - 1].data_ptr(), -T * row, row, p.shape[3]))  # noqa: E731
    tq, tk, tv, to, td, tdq, tdk, tdv = map(place, parts)
    at = lambda t: C.c_void_p(t.data_ptr())  # noqa: E731
    room = lambda n: torch.empty(n, dtype=torch.uint8, device="cuda")  # noqa: E731
    last, dfirst, dg, dbeta = (torch.empty_like(x) for x in (first, first, g, beta))
    ws, wb = room(L.pk_delta_rule_fwd_workspace_bytes(C.byref(shape))), room(L.pk_delta_rule_bwd_workspace_bytes(C.byref(shape)))
    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    pk.lib.check(L.pk_delta_rule_fwd(C.byref(shape), tq, tk, tv, at(g), at(beta), at(first), to, at(last), at(ws), ws.numel(), stream))
    pk.lib.check(L.pk_delta_rule_bwd(C.byref(shape), td, at(dlast), tq, tk, tv, at(g), at(beta), at(first), tdq, tdk, tdv, at(dg), at(dbeta), at(dfirst), at(wb), wb.numel(), stream))
    want = [*pk.ops.gated_delta_rule_fwd(q, k, v, g, beta, 0.25, first), *pk.ops.gated_delta_rule_bwd(do, q, k, v, g, beta, 0.25, first, dlast)]
    o, dq, dk_, dv_ = (parts[i].flip(0) for i in (3, 5, 6, 7))
    assert all(torch.equal(bits(a), bits(b)) for a, b in zip((o, last, dq, dk_, dv_, dg, dbeta, dfirst), want))
    assert all(torch.equal(parts[i].flip(0), x) for i, x in ((0, q), (1, k), (2, v), (4, do)))


def test_gated_delta_step_refuses_what_wants_a_gradient(pk):
    """With gradients kept, a step that one of its tensors wants a gradient of, or that has a tangent, is refused before it moves the state; without, it is what it is."""
    *rule, first, _, _ = delta_inputs(2, 3, 1, 2, 16, 24, BF16, 15)
    kept = first.clone()
    for i, x in enumerate((*rule, first)):
        leaf = x.detach().clone().requires_grad_()
        args = [leaf if i == j else y for j, y in enumerate(rule)]
        with pytest.raises(RuntimeError, match="not differentiable"):
            pk.ops.gated_delta_step_(*args, 0.5, leaf if i == 5 else first)
        with torch.no_grad():
            moved = (leaf if i == 5 else first).clone()
            o = pk.ops.gated_delta_step_(*args, 0.5, moved)
        assert not o.requires_grad and torch.equal(first, kept) and not torch.equal(moved, kept)
        with torch.autograd.forward_ad.dual_level():
            dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
            with pytest.raises(RuntimeError, match="forward-mode"):
                pk.ops.gated_delta_step_(*(dual if i == j else y for j, y in enumerate(rule)), 0.5, dual if i == 5 else first)
    assert torch.equal(first, kept)


# ---- layer norm ----------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("rows,cols,dtype", [(5000, 16400, FP32), (70000, 16385, BF16), (1 << 18, 16400, BF16)], ids=str)
def test_layernorm_weights_gradients_of_tall_inputs_of_long_rows(pk, rows, cols, dtype):
    """dw and db past the rows that are held: 64 workgroups for a column, 64 of their rows added up at a time, those sums one behind the other (a 4096th of the rows), then 4
    workgroups' and 16 of those; the term itself is the kernel's own statistics and 4 u. The same row every time, so that roundings of a long chain all go one way: a chain of a
    64th of the rows would be off by up to a third of its length, 1400 u for the tallest."""
    gen = torch.Generator(device="cuda").manual_seed(rows)
    h, dy = (torch.randn((1, cols), generator=gen, device="cuda").to(dtype) for _ in range(2))
    w = torch.ones(cols, device="cuda")
    _, _, mean, rstd = pk.ops.layernorm_fwd(h, w)
    _, dw, db = pk.ops.layernorm_bwd(dy.expand(rows, cols), h.expand(rows, cols), w, mean.expand(rows).contiguous(), rstd.expand(rows).contiguous())
    n = 64 + rows / 4096 + 1 + 4 + 16 + 4
    term = dy[0].double() * (h[0].double() - mean.double()) * rstd.double()
    within("dw", dw, rows * term, n * U * rows * term.abs())
    within("db", db, rows * dy[0].double(), n * U * rows * dy[0].double().abs())


@pytest.mark.parametrize("rows,cols,dtype", [(70000, 4100, BF16), (1 << 20, 2052, BF16), (1 << 21, 1030, BF16), ((1 << 22) - 3, 24, FP32)], ids=str)
def test_layernorm_weights_gradients_of_tall_inputs(pk, rows, cols, dtype):
    """The same of rows that are held: a walk adds up 256 rows at a time, and those sums one behind the other (at most a 2^16th of the rows), a workgroup's 4 walks, a 16th of 512
    workgroups, 16 of those; 4 u of the term. In a chain of a 256th of the rows, 4096 of the second case, up to a third of its length would be off."""
    gen = torch.Generator(device="cuda").manual_seed(rows)
    h, dy = (torch.randn((1, cols), generator=gen, device="cuda").to(dtype) for _ in range(2))
    w = torch.ones(cols, device="cuda")
    _, _, mean, rstd = pk.ops.layernorm_fwd(h, w)
    _, dw, db = pk.ops.layernorm_bwd(dy.expand(rows, cols), h.expand(rows, cols), w, mean.expand(rows).contiguous(), rstd.expand(rows).contiguous())
    n = 256 + rows / 2 ** 16 + 1 + 4 + 32 + 16 + 4
    term = dy[0].double() * (h[0].double() - mean.double()) * rstd.double()
    within("dw", dw, rows * term, n * U * rows * term.abs())
    within("db", db, rows * dy[0].double(), n * U * rows * dy[0].double().abs())


@pytest.mark.parametrize("cols", [520, 5000, 20000])   # rows of a wavefront, of a workgroup, read three times
def test_layernorm_past_2_to_the_31(pk, cols):
    """Rows 2^30 elements apart, read and with what goes through them; and dense results whose last rows lie past 2^31 elements: what near rows give, to the bit."""
    gen = torch.Generator(device="cuda").manual_seed(cols)
    x, r, dy, dh = (torch.randn((4, cols), generator=gen, device="cuda").to(BF16) for _ in range(4))
    w, b = torch.randn(cols, generator=gen, device="cuda"), torch.randn(cols, generator=gen, device="cuda")
    buffer = torch.zeros(3 * 2 ** 30 + 4 * cols, dtype=BF16, device="cuda")
    far = [buffer[i * cols:].as_strided((4, cols), (2 ** 30, 1)) for i in range(4)]
    for a, near in zip(far, (x, r, dy, dh)):
        a.copy_(near)
    want = pk.ops.layernorm_fwd(x, w, b, 1e-5, r)
    got = pk.ops.layernorm_fwd(far[0], w, b, 1e-5, far[1])
    assert all(torch.equal(bits(p), bits(q)) for p, q in zip(got, want))
    far[0].copy_(want[1])
    back = pk.ops.layernorm_bwd(dy, want[1], w, want[2], want[3], dh)
    assert all(torch.equal(bits(p), bits(q)) for p, q in zip(pk.ops.layernorm_bwd(far[2], far[0], w, want[2], want[3], far[3]), back))
    del buffer, far, got
    rows = 2 ** 31 // cols + 5
    many = lambda t: t[1:2].expand(rows, cols)  # noqa: E731
    y, h, mean, rstd = pk.ops.layernorm_fwd(many(x), w, b, 1e-5, many(r))
    for i in (0, rows - 5, rows - 1):
        assert all(torch.equal(bits(p[i]), bits(q[1])) for p, q in zip((y, h, mean, rstd), want))
    dx, _, _ = pk.ops.layernorm_bwd(many(dy), h, w, mean, rstd, many(dh))
    for i in (0, rows - 5, rows - 1):
        assert torch.equal(bits(dx[i]), bits(back[0][1]))


# ---- distillation --------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("vocab", [4097, 8192, 40000])   # rows of a few pieces to a thread, of more, rows read twice
def test_distill_loss_gradient_does_not_lean(pk, vocab):
    """Words of probability 2^-64 to 2^-120, one by one: the exponent is rounded to 24 bits, 2^-17 apart at these sizes, so each is off by up to 2^-18 ln 2 either way and the
    mean of n of them by 2^-17 ln 2 / sqrt(12 n), six times that here, besides 4 u of the exponential, the factor and the products. An exponent scale rounded to 32 bits before
    the product would turn all of them the same way: by up to 2^-24 of 64 to 120, 50 u at these temperatures."""
    worst = sorted((abs(float(torch.tensor(1 / (math.log(2) * k / 64), dtype=FP32)) * math.log(2) * k / 64 - 1), k / 64) for k in range(32, 257))[-3:]
    assert worst[0][0] > 0.8 * U
    gen = torch.Generator(device="cuda").manual_seed(vocab)
    for _, tau in worst:
        x = -tau * math.log(2) * (64 + 56 * torch.rand((2, vocab), generator=gen, device="cuda", dtype=F64)).to(FP32)
        x[:, 5] = 0.0
        idx, t, w = torch.full((2, 1), 5, dtype=torch.int32, device="cuda"), torch.ones(2, 1, device="cuda"), torch.tensor([0.5, 0.25], device="cuda")
        _, d, _ = pk.blockops.distill_loss(x, idx, t, w, tau)
        want = (w.double().cpu() * tau)[:, None] * torch.exp(x.double().cpu() / tau)   # the sum of the exponentials is 1 to 2^-48; torch's softmax of doubles on the GPU takes 32-bit exponentials
        off = (d.double().cpu() / want - 1)[:, torch.arange(vocab) != 5]
        assert float(off.abs().max()) <= 2.0 ** -18 * math.log(2) + 6 * U
        assert float(off.mean(1).abs().max()) <= 6 * 2.0 ** -17 * math.log(2) / math.sqrt(12 * (vocab - 1)) + 4 * U


@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("vocab", [60, 3001, 70001])
@pytest.mark.parametrize("tail", [False, True], ids=["top", "tail"])
def test_distill_loss_of_words_that_are_none(pk, vocab, tail, dtype):
    """A word past the vocabulary that the teacher gives something: its row has no loss and no gradient, and no other row knows. One that the teacher rules out adds nothing."""
    x, idx, t, w, lse = distill_inputs(6, vocab, 5, dtype, 13)
    lse = lse if tail else None
    idx[1, 4], idx[3, 0], idx[4, 2] = vocab, 2 ** 31 - 1, vocab + 7
    t[4, 2] = -math.inf
    loss, d, kl = pk.blockops.distill_loss(x, idx, t, w, 2.0, lse)
    _, none, alone = pk.blockops.distill_loss(x, idx, t, w, 2.0, lse, grad=False)
    bad = torch.tensor([1, 3], device="cuda")
    assert none is None and torch.equal(bits(alone), bits(kl)) and bool(torch.isnan(loss))
    assert bool(torch.isnan(kl[bad]).all()) and bool(torch.isnan(d[bad].float()).all())
    idx[1], idx[3], idx[4, 2] = -1, -1, -1
    want = pk.blockops.distill_loss(x, idx, t, w, 2.0, lse)
    good = torch.tensor([0, 2, 4, 5], device="cuda")
    assert torch.equal(bits(d[good]), bits(want[1][good])) and torch.equal(kl[good], want[2][good])


def test_distill_loss_past_2_to_the_31(pk):
    """Rows of logits and of their gradient 2^30 elements apart, and a row whose slots begin 2^31 values into the teacher's tensors: what near ones give, to the bit."""
    x, idx, t, w, lse = distill_inputs(4, 1000, 6, BF16, 17)
    far = torch.zeros(3 * 2 ** 30 + 2000, dtype=BF16, device="cuda").as_strided((4, 1000), (2 ** 30, 1))
    far.copy_(x)
    want = pk.blockops.distill_loss(x, idx, t, w, 2.0, lse)
    over = torch.zeros(3 * 2 ** 30 + 2000, dtype=BF16, device="cuda").as_strided((4, 1000), (2 ** 30, 1))
    for out in (None, over, far):
        got = pk.blockops.distill_loss(far, idx, t, w, 2.0, lse, out=out)
        assert out is None or got[1].data_ptr() == out.data_ptr()
        assert all(torch.equal(bits(a), bits(b)) for a, b in zip(got, want))
    del far, over, got
    rows, top = 2 ** 21 + 1, 1024
    x, idx, t, w, _ = distill_inputs(1, 2000, top, BF16, 18)
    many, given, weights = torch.full((rows, top), -1, dtype=torch.int32, device="cuda"), torch.zeros(rows, top, device="cuda"), torch.zeros(rows, device="cuda")
    many[-1], given[-1], weights[-1] = idx[0], t[0], w[0]
    loss, none, kl = pk.blockops.distill_loss(x.expand(rows, 2000), many, given, weights, grad=False)
    alone = pk.blockops.distill_loss(x, idx, t, w, grad=False)
    assert none is None and torch.equal(kl[-1:], alone[2]) and torch.equal(loss, alone[0]) and not kl[:-1].any()
