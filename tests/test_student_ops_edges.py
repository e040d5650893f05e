"""What the operators of a student model refuse beyond test_student_ops.py, asked of the C ABI with pointers that are never followed (no GPU needed)."""
import ctypes as C

import pytest

from paperkiln_amd import _lib
from test_student_ops import ARGUMENT, T4, at, delta, distill

past = lambda i, n: C.c_void_p(at(i).value + n)  # noqa: E731

# rows 4, vocab 100, 8 words for each row, fp32: logits 0, indices 1, teacher 2, its sums 3, weights 4, dlogits 5, kl 6, the rows' losses 7, the loss 8
IN_GRADIENT = [dict(d=at(6)), dict(d=at(7)), dict(d=at(8)), dict(kl=past(5, 1596)), dict(row=past(5, 1592)), dict(loss=past(5, 400))]
DISTILL_OVER = [dict(kl=at(0)), dict(row=at(0)), dict(loss=past(0, 1596)), dict(kl=at(1)), dict(row=past(2, 120)), dict(kl=at(3)), dict(kl=at(4)), dict(row=past(4, 8)), dict(loss=past(4, 12)),
                dict(loss=past(3, 4)), dict(kl=past(7, 28)), dict(row=at(6)), dict(loss=at(6)), dict(loss=past(7, 24))]
where = lambda c: "-".join(f"{n}_{hex(p.value)}" if p else f"no_{n}" for n, p in c.items())  # noqa: E731


@pytest.mark.parametrize("change", IN_GRADIENT + DISTILL_OVER + [dict(d=None, **c) for c in DISTILL_OVER], ids=where)
def test_distill_loss_refuses_results_on_top_of_others(change):
    assert distill(**change) == ARGUMENT and b"overlaps" in _lib.lib().pk_last_error()


def test_distill_loss_refuses_results_in_logits_that_are_overwritten():
    for change in (dict(kl=at(0)), dict(row=past(0, 800)), dict(loss=past(0, 1596))):
        assert distill(d=at(0), **change) == ARGUMENT and b"overlaps" in _lib.lib().pk_last_error()


def test_distill_loss_refuses_row_losses_between_words():
    for rows in (0, 4):
        assert distill(rows=rows, row=past(7, 4)) == ARGUMENT and b"8 bytes" in _lib.lib().pk_last_error()


# q, k, v, o, d_o, dq, dk, dv of 2 x 100 tokens of 64 in bf16, dense, at 1 to 8 << 24: 25600 bytes each
DELTA_PARTLY = [("fwd", dict(o=T4((3 << 24) + 128))), ("fwd", dict(o=T4((1 << 24) + 25598))), ("fwd", dict(o=T4((2 << 24) - 25598))), ("fwd", dict(o=T4((3 << 24) + 13000, -6400, 64, 64))),
                ("bwd", dict(dq=T4((1 << 24) + 128))), ("bwd", dict(dq=T4((7 << 24) - 128))), ("bwd", dict(dk_=T4((8 << 24) + 25598))), ("bwd", dict(dv_=T4((5 << 24) - 64)))]
DELTA_SHARED = [("fwd", dict(o=T4(4 << 24, 0, 64, 64))), ("fwd", dict(o=T4(4 << 24, 6400, 0, 64))), ("fwd", dict(o=T4(4 << 24, 12800, 64, 0), Hv=2)), ("bwd", dict(dq=T4(6 << 24, 0, 64, 64))),
                ("bwd", dict(dk_=T4(7 << 24, 64, 0, 64))), ("bwd", dict(dv_=T4(8 << 24, 12800, 64, 0), Hv=2))]


@pytest.mark.parametrize("entry,change", DELTA_PARTLY, ids=[f"{e}_{i}" for i, (e, _) in enumerate(DELTA_PARTLY)])
def test_gated_delta_rule_refuses_dense_results_partly_on_top_of_others(entry, change):
    assert delta(entry, **change) == ARGUMENT and b"clear of" in _lib.lib().pk_last_error()


@pytest.mark.parametrize("entry,change", DELTA_SHARED, ids=[f"{e}_{i}" for i, (e, _) in enumerate(DELTA_SHARED)])
def test_gated_delta_rule_refuses_results_that_share_their_elements(entry, change):
    assert delta(entry, **change) == ARGUMENT and b"share memory" in _lib.lib().pk_last_error()
