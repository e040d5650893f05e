"""What the operators of a student model refuse, asked of the C ABI with pointers that are never followed (no GPU needed): every refusal comes before the first
launch and leaves a message."""
import ctypes as C
import math
import os
import re
import shutil
import subprocess

import pytest

from paperkiln_amd import _lib

SHAPE, ARGUMENT, WORKSPACE = 1, 2, 3
at = lambda i: C.c_void_p((1 + i) << 24)  # noqa: E731  (stands for a device pointer)


def norm(entry, **kw):
    d = dict(rows=4, cols=100, dtype=_lib.PK_F32, x=at(0), ldx=100, r=at(1), ldr=100, w=at(2), b=at(3), eps=1e-5, y=at(4), h=at(5), mean=at(6), rstd=at(7), dy=at(8), lddy=100,
             dh=at(9), lddh=100, dx=at(10), dw=at(11), db=at(12), ws=at(13), ws_bytes=1 << 20)
    d.update(kw)
    L, s = _lib.lib(), _lib.NormShape(d["rows"], d["cols"], d["dtype"])
    if entry == "fwd":
        return L.pk_layernorm_fwd(C.byref(s), d["x"], d["ldx"], d["r"], d["ldr"], d["w"], d["b"], d["eps"], d["y"], d["h"], d["mean"], d["rstd"], None)
    return L.pk_layernorm_bwd(C.byref(s), d["dy"], d["lddy"], d["h"], d["ldx"], d["dh"], d["lddh"], d["w"], d["mean"], d["rstd"], d["dx"], d["dw"], d["db"], d["ws"], d["ws_bytes"], None)


BOTH = [(dict(rows=-1), SHAPE), (dict(rows=1 << 22), SHAPE), (dict(cols=0), SHAPE), (dict(cols=(1 << 24) + 1), SHAPE), (dict(dtype=2), ARGUMENT), (dict(ldx=-1), SHAPE), (dict(w=None), ARGUMENT),
        (dict(mean=None), ARGUMENT), (dict(rstd=None), ARGUMENT)]
FWD = BOTH + [(dict(x=None), ARGUMENT), (dict(y=None), ARGUMENT), (dict(h=None), ARGUMENT), (dict(r=None), ARGUMENT), (dict(ldr=-1), SHAPE), (dict(eps=-1.0), ARGUMENT), (dict(eps=math.nan), ARGUMENT),
              (dict(eps=math.inf), ARGUMENT), (dict(y=at(0)), ARGUMENT), (dict(y=at(1)), ARGUMENT), (dict(h=at(0)), ARGUMENT), (dict(h=at(4)), ARGUMENT), (dict(y=C.c_void_p((3 << 24) + 40)), ARGUMENT),
              (dict(mean=C.c_void_p((5 << 24) + 1596)), ARGUMENT), (dict(rstd=at(6)), ARGUMENT), (dict(y=at(3)), ARGUMENT)]
BWD = BOTH + [(dict(dy=None), ARGUMENT), (dict(h=None), ARGUMENT), (dict(dx=None), ARGUMENT), (dict(dw=None), ARGUMENT), (dict(db=None), ARGUMENT), (dict(lddy=-1), SHAPE), (dict(lddh=-1), SHAPE),
              (dict(ws=None), WORKSPACE), (dict(ws_bytes=15), WORKSPACE), (dict(ws=C.c_void_p((14 << 24) + 2)), WORKSPACE), (dict(dx=at(8)), ARGUMENT), (dict(dx=at(5)), ARGUMENT),
              (dict(dx=at(9)), ARGUMENT), (dict(dw=at(12)), ARGUMENT), (dict(db=at(2)), ARGUMENT), (dict(ws=at(8)), ARGUMENT), (dict(dw=at(13)), ARGUMENT)]


@pytest.mark.parametrize("change,code", FWD, ids=str)
def test_layernorm_forward_refuses(change, code):
    assert norm("fwd", **change) == code and _lib.lib().pk_last_error()


@pytest.mark.parametrize("change,code", BWD, ids=str)
def test_layernorm_backward_refuses(change, code):
    assert norm("bwd", **change) == code and _lib.lib().pk_last_error()


def test_layernorm_of_no_rows():
    assert norm("fwd", rows=0, x=None, y=None, w=None, mean=None, rstd=None) == 0
    L = _lib.lib()
    for shape in ((-1, 8, 0), (1 << 22, 8, 0), (4, 0, 0)):
        assert L.pk_layernorm_bwd_workspace_bytes(C.byref(_lib.NormShape(*shape))) == 0
    assert L.pk_layernorm_bwd_workspace_bytes(C.byref(_lib.NormShape(0, 8, 0))) == 0 and L.pk_layernorm_bwd_workspace_bytes(C.byref(_lib.NormShape(5, 8, 0))) > 0


def distill(**kw):
    d = dict(tau=1.0, upstream=1.0, x=at(0), ld=100, idx=at(1), t=at(2), lse=at(3), w=at(4), rows=4, vocab=100, top=8, d=at(5), dld=100, kl=at(6), row=at(7), loss=at(8), dtype=_lib.PK_F32)
    d.update(kw)
    c = _lib.DistillConfig(d["tau"], d["upstream"])
    return _lib.lib().pk_distill_loss(C.byref(c), d["x"], d["ld"], d["idx"], d["t"], d["lse"], d["w"], d["rows"], d["vocab"], d["top"], d["d"], d["dld"], d["kl"], d["row"], d["loss"],
                                      d["dtype"], None)


DISTILL = [(dict(tau=0.0), ARGUMENT), (dict(tau=-1.0), ARGUMENT), (dict(tau=math.nan), ARGUMENT), (dict(tau=1e-9), ARGUMENT), (dict(tau=math.inf), ARGUMENT), (dict(upstream=math.inf), ARGUMENT),
           (dict(rows=-1), SHAPE), (dict(rows=1 << 22), SHAPE), (dict(vocab=0), SHAPE), (dict(vocab=(1 << 30) + 1), SHAPE), (dict(top=0), SHAPE), (dict(top=1025), SHAPE), (dict(ld=-1), SHAPE),
           (dict(dld=99), SHAPE), (dict(dtype=3), ARGUMENT), (dict(d=C.c_void_p((1 << 24) + 64)), ARGUMENT), (dict(d=at(0), dld=200), ARGUMENT), (dict(d=at(1)), ARGUMENT), (dict(d=at(2)), ARGUMENT),
           (dict(d=at(3)), ARGUMENT), (dict(d=at(4)), ARGUMENT)] + [({n: None}, ARGUMENT) for n in ("x", "idx", "t", "w", "kl", "row", "loss")]


@pytest.mark.parametrize("change,code", DISTILL, ids=str)
def test_distill_loss_refuses(change, code):
    assert distill(**change) == code and _lib.lib().pk_last_error()
    if change.keys() <= {"tau", "upstream", "loss"}:
        assert distill(rows=0, **change) == code


def T4(p, *strides):
    return C.byref(_lib.Tensor4(p, *(strides or (6400, 64, 64)))) if p else None


def delta(entry, **kw):
    place = dict(q=0, k=1, v=2, o=3, d_o=4, dq=5, dk_=6, dv_=7)
    d = dict(B=2, T=100, Hk=1, Hv=1, dk=64, dv=64, dtype=_lib.PK_BF16, scale=0.125, g=at(8), beta=at(9), s0=at(10), s1=at(11), ds1=at(12), ds0=at(13), dg=at(14), dbeta=at(15), ws=at(16),
             ws_bytes=1 << 40, **{n: T4((1 + i) << 24) for n, i in place.items()})
    d.update(kw)
    L, s = _lib.lib(), _lib.DeltaShape(d["B"], d["T"], d["Hk"], d["Hv"], d["dk"], d["dv"], d["dtype"], d["scale"])
    if entry == "fwd":
        return L.pk_delta_rule_fwd(C.byref(s), d["q"], d["k"], d["v"], d["g"], d["beta"], d["s0"], d["o"], d["s1"], d["ws"], d["ws_bytes"], None)
    return L.pk_delta_rule_bwd(C.byref(s), d["d_o"], d["ds1"], d["q"], d["k"], d["v"], d["g"], d["beta"], d["s0"], d["dq"], d["dk_"], d["dv_"], d["dg"], d["dbeta"], d["ds0"], d["ws"],
                               d["ws_bytes"], None)


DELTA = [(dict(B=-1), SHAPE), (dict(T=-1), SHAPE), (dict(Hk=0), SHAPE), (dict(Hv=0), SHAPE), (dict(Hk=2, Hv=3), SHAPE), (dict(dk=0), SHAPE), (dict(dk=129), SHAPE), (dict(dv=0), SHAPE),
         (dict(dv=257), SHAPE), (dict(dtype=2), ARGUMENT), (dict(scale=math.nan), ARGUMENT), (dict(scale=math.inf), ARGUMENT), (dict(B=1 << 20, Hv=2), SHAPE), (dict(B=(1 << 19) + 1, T=1), SHAPE), (dict(T=(1 << 26) + 1), SHAPE), (dict(B=1, T=(1 << 22) * 64), SHAPE), (dict(B=1 << 16, T=63 * 64 + 1), SHAPE),
         (dict(B=1 << 18, T=1 << 14), SHAPE), (dict(ws=None), WORKSPACE), (dict(ws_bytes=100), WORKSPACE), (dict(ws=C.c_void_p((17 << 24) + 8)), WORKSPACE)]
# results on top of what is read or of one another; a step of 6400 elements between tensors of heads of 2 x 100 tokens of 64
DELTA_OVER = {"fwd": [dict(o=T4(2 << 24)), dict(o=T4((9 << 24) + 64)), dict(s1=C.c_void_p((11 << 24) + 64)), dict(s1=at(0)), dict(s1=C.c_void_p((2 << 24) + 25000)), dict(s1=at(8)), dict(ws=at(1)),
                      dict(ws=C.c_void_p((4 << 24) - 64)), dict(s1=at(3)), dict(ws=at(11)), dict(o=T4((9 << 24) + 13200, -6400, 64, 64))],
              "bwd": [dict(dq=T4(1 << 24)), dict(dv_=T4(5 << 24)), dict(dq=T4(7 << 24)), dict(dg=at(8)), dict(dg=at(15)), dict(dbeta=at(9)), dict(ds0=at(10)), dict(ds0=at(12)), dict(ds0=at(7)),
                      dict(ws=at(4)), dict(ws=at(14)), dict(ws=C.c_void_p((13 << 24) - 64)), dict(dk_=T4((16 << 24) + 396))]}


@pytest.mark.parametrize("entry,change", [(e, c) for e, l in DELTA_OVER.items() for c in l], ids="-".join)
def test_gated_delta_rule_refuses_results_on_top_of_others(entry, change):
    assert delta(entry, **change) == ARGUMENT and b"clear of" in _lib.lib().pk_last_error()


DELTA_NULL = {"fwd": ("q", "k", "v", "g", "beta", "o"), "bwd": ("d_o", "q", "k", "v", "g", "beta", "dq", "dk_", "dv_", "dg", "dbeta")}


@pytest.mark.parametrize("entry", ["fwd", "bwd"])
@pytest.mark.parametrize("change,code", DELTA, ids=str)
def test_gated_delta_rule_refuses(entry, change, code):
    assert delta(entry, **change) == code and _lib.lib().pk_last_error()


@pytest.mark.parametrize("entry", ["fwd", "bwd"])
def test_gated_delta_rule_refuses_null(entry):
    for n in DELTA_NULL[entry]:
        assert delta(entry, **{n: None}) == ARGUMENT, n
    assert delta(entry, B=0, **{n: None for n in DELTA_NULL[entry]}) == 0    # nothing to do
    L = _lib.lib()
    for T, none in ((1, True), (8, True), (9, False)):
        assert (L.pk_delta_rule_fwd_workspace_bytes(C.byref(_lib.DeltaShape(2, T, 1, 1, 64, 64, 1, 1.0))) == 0) == none
    assert L.pk_delta_rule_bwd_workspace_bytes(C.byref(_lib.DeltaShape(2, 1, 1, 1, 64, 64, 1, 1.0))) > 0
    assert L.pk_delta_rule_bwd_workspace_bytes(C.byref(_lib.DeltaShape(2, 1, 1, 1, 640, 64, 1, 1.0))) == 0


SOURCES = ("layernorm.hip", "distill_loss.hip", "delta_rule.hip", "delta_rule_bwd.hip")


@pytest.fixture(scope="module")
def assembly(tmp_path_factory):
    from test_asm_hazards import CSRC, FLAGS
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not found")
    out = tmp_path_factory.mktemp("student")
    jobs = {src: str(out / (src + ".s")) for src in SOURCES}
    running = [subprocess.Popen([hipcc, *FLAGS, os.path.join(CSRC, src), "-o", to], stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL) for src, to in jobs.items()]
    assert [p.wait() for p in running] == [0] * len(running)
    return jobs


def test_kernels_stay_in_registers(assembly):
    """Nothing spilled to memory, and no array kept in LDS by an offset from the launch's packet."""
    for src, path in assembly.items():
        text = open(path).read()
        assert len(re.findall(r"\.amdhsa_kernel ", text)) >= 4, src
        assert not re.findall(r"amdhsa_user_sgpr_dispatch_ptr 1", text), src
        assert set(re.findall(r"\.vgpr_spill_count: +(\d+)", text)) == {"0"} and set(re.findall(r"\.private_segment_fixed_size: +(\d+)", text)) == {"0"}, src
