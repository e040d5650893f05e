"""What the post-training operators refuse, asked of the C ABI with pointers that are never followed (no GPU needed): every refusal comes before the first
launch and leaves a message."""
import ctypes as C
import math

import pytest

from paperkiln_amd import _lib

SHAPE, ARGUMENT, WORKSPACE = 1, 2, 3
SOME = C.c_void_p(1 << 20)          # stands for a device pointer
FAR = C.c_void_p(1 << 40)
CLOSE = C.c_void_p((1 << 20) + 64)


def T4(p=1 << 20):
    return C.byref(_lib.Tensor4(p, 64, 64, 64))


def qk(**kw):
    d = dict(B=1, T=2, Hq=2, Hkv=1, dk=64, rotary=0, halves=0, dtype=_lib.PK_BF16, eps=1e-5, theta=1e4, pos_stride_b=0)
    d.update(kw)
    return _lib.QkShape(*[d[n] for n, _ in _lib.QkShape._fields_])


QK_REFUSED = [(dict(dk=63), SHAPE), (dict(dk=258), SHAPE), (dict(dk=0), SHAPE), (dict(Hq=0), SHAPE), (dict(Hkv=-1), SHAPE), (dict(B=-1), SHAPE), (dict(T=-1), SHAPE),
              (dict(rotary=3), SHAPE), (dict(rotary=66), SHAPE), (dict(rotary=-2), SHAPE), (dict(dtype=2), ARGUMENT), (dict(theta=0.0), ARGUMENT),
              (dict(theta=math.nan), ARGUMENT), (dict(theta=math.inf), ARGUMENT), (dict(eps=-1.0), ARGUMENT), (dict(eps=math.nan), ARGUMENT)]


@pytest.mark.parametrize("change,code", QK_REFUSED, ids=str)
def test_qk_norm_rope_refuses(change, code):
    L, s = _lib.lib(), qk(**change)
    assert L.pk_qk_norm_rope_fwd(C.byref(s), T4(), T4(), SOME, SOME, SOME, T4(), T4(), None) == code and L.pk_last_error()
    assert L.pk_qk_norm_rope_bwd(C.byref(s), T4(), T4(), T4(), T4(), SOME, SOME, SOME, T4(), T4(), SOME, SOME, SOME, 1 << 30, None) == code
    assert L.pk_qk_norm_rope_bwd_workspace_bytes(C.byref(s)) == 0


def test_qk_norm_rope_refuses_null_and_small_workspaces():
    L, s = _lib.lib(), qk()
    fwd = [C.byref(s), T4(), T4(), SOME, SOME, SOME, T4(), T4(), None]
    for i in range(8):
        a = list(fwd)
        a[i] = T4(0) if i in (1, 2, 6, 7) else None
        assert L.pk_qk_norm_rope_fwd(*a) == ARGUMENT, i
    need = L.pk_qk_norm_rope_bwd_workspace_bytes(C.byref(s))
    bwd = [C.byref(s), T4(), T4(), T4(), T4(), SOME, SOME, SOME, T4(), T4(), SOME, SOME, SOME, need, None]
    for i in range(12):
        a = list(bwd)
        a[i] = T4(0) if i in (1, 2, 3, 4, 8, 9) else None
        assert L.pk_qk_norm_rope_bwd(*a) == ARGUMENT, i
    for ws, size in ((None, need), (SOME, need - 1), (C.c_void_p((1 << 20) + 2), need)):
        a = list(bwd)
        a[12], a[13] = ws, size
        assert L.pk_qk_norm_rope_bwd(*a) == WORKSPACE
    assert L.pk_qk_norm_rope_fwd(C.byref(qk(T=0)), T4(0), T4(0), None, None, None, T4(0), T4(0), None) == 0   # nothing to do


def test_qk_norm_rope_refuses_crossed_results():
    """A result that begins where the other one does, or where what the other one is made of does."""
    L, s = _lib.lib(), qk()
    at = lambda i: T4((1 + i) << 20)  # noqa: E731
    for yq, yk in ((5, 5), (2, 6), (5, 1), (2, 1)):   # q at 1, k at 2
        assert L.pk_qk_norm_rope_fwd(C.byref(s), at(1), at(2), SOME, SOME, SOME, at(yq), at(yk), None) == ARGUMENT and b"other" in L.pk_last_error()
    need = L.pk_qk_norm_rope_bwd_workspace_bytes(C.byref(s))
    for dq, dk in ((5, 5), (2, 6), (4, 6), (5, 1), (5, 3)):   # dyq, dyk at 3, 4
        assert L.pk_qk_norm_rope_bwd(C.byref(s), at(3), at(4), at(1), at(2), SOME, SOME, SOME, at(dq), at(dk), SOME, SOME, SOME, need, None) == ARGUMENT and b"other" in L.pk_last_error()


# In a buffer of 2 sequences of 3 tokens, each 8 heads of 64 bf16: queries are heads 0 to 3, keys 4 and 5. Places are (elements from the buffer's first, strides of sequences, tokens, heads).
FUSED, AWAY = (1536, 512, 64), 1 << 20
Q, K = (0, *FUSED), (256, *FUSED)
QK_OVERLAPS = [(512, *FUSED), (-512, *FUSED), (64, *FUSED), (1, *FUSED), (-1, *FUSED), (1536, *FUSED),   # a token, a head, an element, a sequence on
               (384, *FUSED), (192, *FUSED),                                                          # into the next token's queries, into the keys
               (0, 1536, 64, 512), (0, 768, 256, 64), (0, 1536, 512, 128),                              # the place, other strides
               (1024, 1536, -512, 64), (0, 0, 512, 64), (0, 1536, 512, 0)]                              # backwards; all sequences, all heads in one place
QK_SHARING = [(AWAY, 1536, 512, 32), (AWAY, 1536, 128, 64), (AWAY, 512, 512, 64), (AWAY, 0, 512, 64), (AWAY, 256, 512, 0)]


def place(at):
    return C.byref(_lib.Tensor4((1 << 30) + 2 * at[0], *at[1:]))


@pytest.mark.parametrize("out", QK_OVERLAPS + QK_SHARING, ids=str)
def test_qk_norm_rope_refuses_overlaps(out):
    """Queries' results over the queries, the gradient that arrives or themselves; over the keys' tensors and the other way round."""
    L, s, words = _lib.lib(), qk(B=2, T=3, Hq=4, Hkv=2), (SOME, SOME, SOME)
    far = [place((AWAY << i, *FUSED)) for i in range(1, 6)]
    end = (SOME, SOME, SOME, L.pk_qk_norm_rope_bwd_workspace_bytes(C.byref(s)), None)
    why = lambda: [w for w in ("share memory", "clear of it", "over the other one") if w in L.pk_last_error().decode()]  # noqa: E731
    at, q, k = place(out), place(Q), place(K)
    assert L.pk_qk_norm_rope_fwd(C.byref(s), q, far[0], *words, at, far[1], None) == ARGUMENT and why() != ["over the other one"]
    for dy, x in ((q, far[0]), (far[0], q)):
        assert L.pk_qk_norm_rope_bwd(C.byref(s), dy, far[1], x, far[2], *words, at, far[3], *end) == ARGUMENT and why() != ["over the other one"]
    if out == (192, *FUSED):
        assert L.pk_qk_norm_rope_fwd(C.byref(s), far[0], k, *words, at, far[1], None) == ARGUMENT and why() == ["over the other one"]
        assert L.pk_qk_norm_rope_fwd(C.byref(s), far[0], far[1], *words, at, k, None) == ARGUMENT and why() == ["over the other one"]
        for dy, x in ((k, far[0]), (far[0], k)):
            assert L.pk_qk_norm_rope_bwd(C.byref(s), far[1], dy, far[2], x, *words, at, far[3], *end) == ARGUMENT and why() == ["over the other one"]
        assert L.pk_qk_norm_rope_bwd(C.byref(s), at, far[0], far[1], far[2], *words, far[3], k, *end) == ARGUMENT and why() == ["over the other one"]


@pytest.mark.parametrize("which", range(3))
@pytest.mark.parametrize("at", [0, 2 * 510, 2 * (1536 + 700)])
def test_qk_norm_rope_refuses_results_over_weights_and_positions(which, at):
    L, s, far = _lib.lib(), qk(B=2, T=3, Hq=4, Hkv=4, dk=128), (AWAY << 1, *FUSED)   # heads fill their tokens
    words = [SOME, SOME, SOME]
    words[which] = C.c_void_p((1 << 30) + at)
    out, off = place((0, 1536, 512, 128)), place((AWAY << 2, 1536, 512, 128))
    for y in ((out, off), (off, out)):
        assert L.pk_qk_norm_rope_fwd(C.byref(s), place(far), place(far), *words, *y, None) == ARGUMENT and b"weights" in L.pk_last_error()
        assert L.pk_qk_norm_rope_bwd(C.byref(s), *[place(far)] * 4, *words, *y, SOME, SOME, SOME, 1 << 30, None) == ARGUMENT and b"weights" in L.pk_last_error()


# what is the same for the three entries that read logits and write their gradient
LOGITS_REFUSED = [(dict(rows=-1), SHAPE), (dict(rows=1 << 31), SHAPE), (dict(vocab=0), SHAPE), (dict(vocab=(1 << 30) + 1), SHAPE), (dict(ld=-1), SHAPE),
                  (dict(dld=99), SHAPE), (dict(dtype=7), ARGUMENT), (dict(scale=0.0), ARGUMENT), (dict(scale=-1.0), ARGUMENT), (dict(scale=math.inf), ARGUMENT),
                  (dict(scale=math.nan), ARGUMENT), (dict(scale=1e-25), ARGUMENT), (dict(scale=1e25), ARGUMENT), (dict(logits=None), ARGUMENT), (dict(targets=None), ARGUMENT), (dict(dlogits=None), ARGUMENT),
                  (dict(dlogits=CLOSE), ARGUMENT), (dict(dlogits=SOME, dld=200), ARGUMENT)]


def call(entry, **kw):
    d = dict(logits=SOME, ld=100, targets=SOME, rows=4, vocab=100, scale=1.0, dlogits=FAR, dld=100, dtype=_lib.PK_F32, v=SOME, ref=SOME, loss=SOME, low=0.2, high=0.2, kl=0.1,
             upstream=1.0, beta=0.1, smoothing=0.0, pairs=1, starts=SOME, ws=SOME, ws_bytes=1 << 20)
    d.update(kw)
    L = _lib.lib()
    x = d["logits"], d["ld"], d["targets"]
    if entry == "bwd":
        return L.pk_token_logprobs_bwd(*x, d["v"], d["v"], d["rows"], d["vocab"], d["scale"], d["dlogits"], d["dld"], d["dtype"], None)
    if entry == "policy":
        c = _lib.PolicyConfig(d["low"], d["high"], d["kl"], d["scale"], d["upstream"])
        return L.pk_policy_loss(C.byref(c), *x, d["v"], d["ref"], d["v"], d["v"], d["rows"], d["vocab"], d["dlogits"], d["dld"], d["v"], d["v"], d["loss"], d["ws"], d["ws_bytes"], d["dtype"], None)
    c = _lib.PreferenceConfig(d["beta"], d["smoothing"], d["scale"], d["upstream"])
    return L.pk_preference_loss(C.byref(c), *x, d["starts"], d["pairs"], d["ref"], d["rows"], d["vocab"], d["dlogits"], d["dld"], d["v"], d["v"], d["loss"], d["ws"],
                                d["ws_bytes"], d["dtype"], None)


@pytest.mark.parametrize("entry", ["bwd", "policy", "preference"])
@pytest.mark.parametrize("change,code", LOGITS_REFUSED, ids=str)
def test_losses_refuse_logits(entry, change, code):
    assert call(entry, **change) == code and _lib.lib().pk_last_error()


@pytest.mark.parametrize("entry,change,code", [
    ("bwd", dict(v=None), ARGUMENT), ("policy", dict(v=None), ARGUMENT), ("policy", dict(ref=None), ARGUMENT), ("policy", dict(loss=None), ARGUMENT),
    ("policy", dict(low=-0.1), ARGUMENT), ("policy", dict(high=math.nan), ARGUMENT), ("policy", dict(kl=math.inf), ARGUMENT), ("policy", dict(upstream=math.nan), ARGUMENT),
    ("preference", dict(v=None), ARGUMENT), ("preference", dict(ref=None), ARGUMENT), ("preference", dict(starts=None), ARGUMENT), ("preference", dict(loss=None), ARGUMENT),
    ("preference", dict(pairs=0), SHAPE), ("preference", dict(pairs=1 << 22), SHAPE), ("preference", dict(pairs=-3), SHAPE), ("preference", dict(beta=math.inf), ARGUMENT), ("preference", dict(smoothing=1.5), ARGUMENT),
    ("preference", dict(smoothing=math.nan), ARGUMENT), ("preference", dict(ws=None), WORKSPACE), ("preference", dict(ws_bytes=100), WORKSPACE)], ids=str)
def test_losses_refuse(entry, change, code):
    assert call(entry, **change) == code and _lib.lib().pk_last_error()


def test_token_logprobs_refuses():
    L = _lib.lib()
    for change, code in (((None, 100, SOME, 4, 100, 1.0, SOME), ARGUMENT), ((SOME, 100, None, 4, 100, 1.0, SOME), ARGUMENT), ((SOME, 100, SOME, 4, 100, 1.0, None), ARGUMENT),
                         ((SOME, 100, SOME, 4, 0, 1.0, SOME), SHAPE), ((SOME, 100, SOME, 4, 100, math.nan, SOME), ARGUMENT)):
        assert L.pk_token_logprobs_fwd(*change, None, None, 0, _lib.PK_F32, None) == code
    assert L.pk_token_logprobs_fwd(None, 100, None, 0, 100, 1.0, None, None, None, 0, _lib.PK_F32, None) == 0   # nothing to do
    need = L.pk_token_logprobs_workspace_bytes(3, 200000, _lib.PK_F32)   # a few rows that no workgroup holds: 32 parts of 8 bytes each
    assert need == 3 * 32 * 8 and L.pk_token_logprobs_workspace_bytes(3, 32000, _lib.PK_F32) == 0 and L.pk_token_logprobs_workspace_bytes(128, 200000, _lib.PK_F32) == 0
    for ws, size in ((SOME, need - 1), (C.c_void_p((1 << 20) + 4), need)):
        assert L.pk_token_logprobs_fwd(SOME, 200000, SOME, 3, 200000, 1.0, SOME, None, ws, size, _lib.PK_F32, None) == WORKSPACE
    need = L.pk_policy_loss_workspace_bytes(3, 200000, _lib.PK_F32)   # the same, and two words a row
    assert need == 3 * (32 * 8 + 8) and L.pk_policy_loss_workspace_bytes(3, 16000, _lib.PK_F32) == 0 and L.pk_policy_loss_workspace_bytes(65, 200000, _lib.PK_F32) == 0
    for ws, size in ((SOME, need - 1), (C.c_void_p((1 << 20) + 4), need)):
        assert call("policy", rows=3, vocab=200000, ld=200000, dld=200000, ws=ws, ws_bytes=size) == WORKSPACE
    assert L.pk_preference_loss_workspace_bytes(1000, 3) == 4096 + 4096 + 8192 + 256
    assert L.pk_preference_loss_workspace_bytes(100, 3) == 512 + 512 + 1024 + 256 + 100 * 32 * 8


def adamw(tensors, ws=SOME, ws_bytes=1 << 20, norm=SOME, **kw):
    d = dict(lr=1e-3, b1=0.9, b2=0.99, eps=1e-8, wd=0.0, max_norm=0.0, t=1, state_bits=32, grad_dtype=_lib.PK_F32, seed=0)
    d.update(kw)
    table = (_lib.AdamWTensor * max(1, len(tensors)))(*tensors)
    cfg = _lib.AdamWConfig(*[d[n] for n, _ in _lib.AdamWConfig._fields_])
    return _lib.lib().pk_adamw_many(table, len(tensors), C.byref(cfg), ws, ws_bytes, norm, None)


def tensor(at, n=100, g=1 << 30, scales=1 << 31, copy=None, m=None, v=None):
    return _lib.AdamWTensor(at, g, m if m is not None else at + 4 * n, v if v is not None else at + 8 * n, scales, scales, copy, n)


@pytest.mark.parametrize("change,code", [(dict(t=0), ARGUMENT), (dict(state_bits=16), ARGUMENT), (dict(grad_dtype=2), ARGUMENT), (dict(b1=1.0), ARGUMENT), (dict(b2=-0.1), ARGUMENT),
                                         (dict(b2=math.nan), ARGUMENT), (dict(max_norm=math.nan), ARGUMENT), (dict(max_norm=1.0, norm=None), ARGUMENT), (dict(max_norm=1.0, ws=None), WORKSPACE),
                                         (dict(max_norm=1.0, ws_bytes=263), WORKSPACE)], ids=str)
def test_adamw_many_refuses(change, code):
    assert adamw([tensor(1 << 20)], **change) == code and _lib.lib().pk_last_error()


def test_adamw_many_refuses_tables():
    one = tensor(1 << 20)
    for bad in (tensor(0, m=1, v=1), tensor(1 << 20, g=0), tensor(1 << 20, m=0), tensor(1 << 20, v=0)):
        assert adamw([bad]) == ARGUMENT
    assert adamw([tensor(1 << 20, scales=0)], state_bits=8) == ARGUMENT
    assert adamw([tensor(1 << 20, n=-1)]) == SHAPE and adamw([tensor(1 << 20, n=(1 << 40) + 1)]) == SHAPE and adamw([tensor(1 << 20, n=(1 << 35) + 1)]) == SHAPE
    for twice in (one, tensor((1 << 20) + 4 * 99), tensor(1 << 24, m=(1 << 20) + 4 * 150), tensor(1 << 24, v=1 << 20)):
        assert adamw([one, twice]) == ARGUMENT and b"twice" in _lib.lib().pk_last_error()
    assert adamw([tensor(1 << 48)]) == ARGUMENT and b"48 bits" in _lib.lib().pk_last_error()
    # scales of two tensors that meet, copies that do
    assert adamw([one, tensor(1 << 24, scales=(1 << 31) + 4)], state_bits=8) == ARGUMENT
    assert adamw([tensor(1 << 20, copy=1 << 33), tensor(1 << 24, copy=(1 << 33) + 198)]) == ARGUMENT
    assert adamw([]) == 0 and adamw([_lib.AdamWTensor(0, 0, 0, 0, 0, 0, 0, 0)]) == 0   # nothing to do
    assert _lib.lib().pk_adamw_many(None, 2, None, None, 0, None, None) == ARGUMENT


def tensor8(at, n=1000, g=1 << 30):
    """One with moments in 8 bits, everything in places of its own: four scales of 4 bytes in each of two."""
    blocks = (n + 255) // 256
    m, v = at + 4 * n, at + 5 * n
    ms = at + 6 * n
    return _lib.AdamWTensor(at, g, m, v, ms, ms + 4 * blocks, None, n)


@pytest.mark.parametrize("field", ["p", "m", "v", "m_scale", "v_scale"])
@pytest.mark.parametrize("off", [-1, 1], ids=["ends", "begins"])
def test_adamw_many_refuses_tensors_of_8_bits_that_meet(field, off):
    """Two tensors apart but for one word of one of them; with the clip's workspace missing the same table is refused for that, behind the check for what meets."""
    last = dict(p=4 * 1000, m=1000, v=1000, m_scale=16, v_scale=16)[field]
    refused = lambda a, b: (adamw([a, b], state_bits=8, max_norm=1.0, ws=None), b"twice" in _lib.lib().pk_last_error())  # noqa: E731
    assert refused(tensor8(1 << 20), tensor8(1 << 24)) == (WORKSPACE, False)
    for other in ("p", "m", "v", "m_scale", "v_scale"):
        for near in (0, 1):   # a byte of it beyond, and just clear
            a, b = tensor8(1 << 20), tensor8(1 << 24)
            size = dict(p=4 * 1000, m=1000, v=1000, m_scale=16, v_scale=16)[other]
            setattr(b, field, getattr(a, other) + size - near if off > 0 else getattr(a, other) - last + near)
            # beside the last word of a lies nothing of it, but before most of its words and behind others there is
            alone = not near and (other == "v_scale" if off > 0 else other == "p")
            assert refused(a, b) == ((WORKSPACE, False) if alone else (ARGUMENT, True)), (other, near)


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("grads", [_lib.PK_F32, _lib.PK_BF16], ids=["g32", "g16"])
def test_adamw_many_refuses_gradients_over_what_is_written(bits, grads):
    """One tensor's gradient in the place of another's parameter, state, scale or copy, in its own's but for an element, in the whole range and at both ends of it. With the
    clip's workspace missing a table without fault is refused for that."""
    size, n = 4 if grads == _lib.PK_F32 else 2, 1000

    def table(where=None, of=0, off=0, order=1):
        one = [tensor8(1 << 20, g=1 << 30), tensor8(1 << 24, g=1 << 31)]
        for x in one:
            if bits == 32:
                x.m, x.v = x.p + 4 * n, x.p + 8 * n
            x.copy = x.p + 16 * n
        if where:
            one[0].g = getattr(one[of], where) + off
        got = adamw(one[::order], state_bits=bits, grad_dtype=grads, max_norm=1.0, ws=None)
        return got, b"gradient" in _lib.lib().pk_last_error()

    width = dict(p=4, m=bits // 8, v=bits // 8, copy=2, **(dict(m_scale=0, v_scale=0) if bits == 8 else {}))
    assert table() == (WORKSPACE, False)
    for where, w in width.items():
        last = w * n - size if w else 12
        for order in (1, -1):
            for of in (0, 1):
                own = of == 0 and w == size
                assert table(where, of, 0, order) == ((WORKSPACE, False) if own else (ARGUMENT, True)), (where, of)
                for off in (size, -size, last, -size * n + size):
                    assert table(where, of, off, order) == (ARGUMENT, True), (where, of, off)
        assert table("p", 0, -size * n) == (WORKSPACE, False) and table("copy", 1, 2 * n) == (WORKSPACE, False)   # just clear


def test_torch_front_end_refuses_tensors_of_the_cpu():
    """Types, shapes and places are checked before any pointer is handed on."""
    import torch

    from paperkiln_amd import blockops, ops
    z = torch.zeros
    i32 = lambda *s: z(*s, dtype=torch.int32)  # noqa: E731
    for fn in (lambda: ops.qk_norm_rope_fwd(z(1, 2, 2, 4), z(1, 2, 2, 4), z(4), z(4), i32(2), 1e4), lambda: ops.token_logprobs(z(3, 5), i32(3)),
               lambda: blockops.policy_loss(z(3, 5), i32(3), z(3), z(3), z(3)), lambda: blockops.preference_loss(z(3, 5), i32(3), i32(3), z(3)),
               lambda: blockops.adamw_many_([z(3)], [z(3)], blockops.adamw_state([z(3)], 8), 1e-3)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            fn()
    with pytest.raises(RuntimeError, match="8 or in 32"):
        blockops.adamw_state([z(3)], 16)
    with pytest.raises(TypeError):
        ops.token_logprobs([1.0], i32(1))


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_state_of_what_can_be_gone_through_once(bits):
    """A model's parameters() is a generator: all of the state's lists are as long as it was."""
    import torch

    from paperkiln_amd import blockops
    sizes = [(3, 5), (700,), ()]
    state = blockops.adamw_state((torch.zeros(s) for s in sizes), bits)
    assert [m.shape for m in state.m] == [v.shape for v in state.v] == [torch.Size(s) for s in sizes]
    assert state.m_scale is None if bits == 32 else [x.numel() for x in state.m_scale] == [x.numel() for x in state.v_scale] == [1, 3, 1]


@pytest.fixture(scope="module")
def post_assembly(tmp_path_factory):
    import os
    import shutil
    import subprocess

    from test_asm_hazards import CSRC, FLAGS
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not found")
    out = tmp_path_factory.mktemp("post")
    jobs = {src: str(out / (src + ".s")) for src in ("qk_norm_rope.hip", "token_loss.hip", "adamw_many.hip")}
    running = [subprocess.Popen([hipcc, *FLAGS, os.path.join(CSRC, src), "-o", to], stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL) for src, to in jobs.items()]
    assert [p.wait() for p in running] == [0] * len(running)
    return jobs


def test_kernels_stay_in_registers(post_assembly):
    """Nothing spilled to memory, and no array kept in LDS by an offset from the launch's packet (which lies in the host's memory: a forward of 10 us took 22)."""
    import re
    for src, path in post_assembly.items():
        text = open(path).read()
        assert len(re.findall(r"\.amdhsa_kernel ", text)) >= 5, src
        assert not re.findall(r"amdhsa_user_sgpr_dispatch_ptr 1", text), src
        assert set(re.findall(r"\.vgpr_spill_count: +(\d+)", text)) == {"0"} and set(re.findall(r"\.private_segment_fixed_size: +(\d+)", text)) == {"0"}, src


def test_stores_in_asm_statements_keep_their_data_and_addresses(post_assembly):
    from test_asm_hazards import scalars_read_early, stores_overwritten
    path = post_assembly["qk_norm_rope.hip"]
    assert "global_store_dwordx4" in open(path).read()
    assert not stores_overwritten(path) and not scalars_read_early(path)
