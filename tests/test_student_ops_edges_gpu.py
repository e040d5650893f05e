"""The operators of a student model at the edges of what they promise, on the GPU against 64 bits: bf16 tensors whose sums nearly cancel, words that are none, tall and far
inputs. Tolerances are counted as in test_student_ops_gpu.py: u = 2^-24, h half a step of the output's type."""
from __future__ import annotations

import pytest
import torch

from test_post_ops_gpu import BF16, F64, FP32, HALF, U, within
from test_student_ops_gpu import pk, plain_delta  # noqa: F401  (pk: a fixture)

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
