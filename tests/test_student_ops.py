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


SOURCES = ("layernorm.hip", "distill_loss.hip")


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
