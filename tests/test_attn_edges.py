"""What attention's operators refuse before a device is asked: status codes of the library, and the checks of the Python mirror on stand-ins
for device tensors.  No call below reaches a device."""
import copy
import ctypes

import numpy as np
import pytest
import torch

import attn_ref
import mx_ref
from hipster_amd import _lib, qmm
from hipster_amd._lib import KVMX, Attn, QmmError, Rope, Seqs
from test_mx_edges import OnDevice, launched  # noqa: F401

FORMAT, SHAPE, NULL, WORKSPACE, ARG = -1, -2, -3, -5, -6
D = 64                                        # an aligned address that nothing dereferences
BIG = 1 << 40


def kvmx(kq=D, ke=D, vq=D, ve=D, pages=4, page=16, heads=2, dim=64):
    return KVMX(kq, ke, vq, ve, pages, page, heads, dim)


def seqs(cu=D, lens=D, table=D, n=2, ld=4):
    return Seqs(cu, lens, table, n, ld)


CACHES = [(dict(kq=None), NULL), (dict(ke=None), NULL), (dict(vq=None), NULL), (dict(ve=None), NULL), (dict(kq=8), ARG), (dict(vq=24), ARG),
          (dict(ke=4), ARG), (dict(ve=1), ARG), (dict(pages=0), SHAPE), (dict(page=8), SHAPE), (dict(page=48), SHAPE), (dict(page=8192), SHAPE),
          (dict(page=0), SHAPE), (dict(page=-16), SHAPE), (dict(heads=0), SHAPE), (dict(dim=32), SHAPE), (dict(dim=96), SHAPE), (dict(dim=512), SHAPE)]
SEQS = [(dict(cu=None), NULL), (dict(lens=None), NULL), (dict(table=None), NULL), (dict(cu=2), ARG), (dict(n=0), SHAPE), (dict(n=-1), SHAPE),
        (dict(ld=0), SHAPE), (dict(ld=1 << 28), SHAPE)]


def test_cache_refusals():
    L = _lib.lib()

    def write(k=D, ldk=128, v=D, ldv=128, dtype=1, kv=None, s=None, rows=3):
        return L.qmm_kv_write_mxfp4(k, ldk, v, ldv, dtype, kvmx(**(kv or {})), seqs(**(s or {})), rows, None)

    def read(k=D, ldk=128, v=D, ldv=128, dtype=1, kv=None, s=None, rows=3):
        return L.qmm_kv_read_mxfp4(kvmx(**(kv or {})), seqs(**(s or {})), k, ldk, v, ldv, dtype, rows, None)

    for f in (write, read):
        for kw, want in CACHES:
            assert f(kv=kw) == want, kw
        for kw, want in SEQS:
            assert f(s=kw) == want, kw
        assert f(k=None) == NULL and f(v=None) == NULL and f(dtype=2) == FORMAT and f(dtype=-1) == FORMAT and f(rows=-1) == SHAPE
        assert f(ldk=127) == SHAPE and f(ldv=127) == SHAPE and f(k=65) == ARG and f(v=66, dtype=0) == ARG
        assert f(rows=0, k=None, v=None, kv=dict(kq=None), s=dict(cu=None)) == 0
        assert f(rows=0x7fffffff, kv=dict(heads=4096, dim=256), ldk=1 << 20, ldv=1 << 20) == SHAPE           # more waves than a launch has
    assert L.qmm_kv_write_mxfp4(D, 128, D, 128, 1, None, seqs(), 1, None) == NULL
    assert L.qmm_kv_read_mxfp4(kvmx(), None, D, 128, D, 128, 1, 1, None) == NULL


def test_attend_refusals():
    L = _lib.lib()

    def f(q=D, qt=1, ldq=256, kv=None, s=None, at=(None, 1.0, 0), out=D, ot=1, ldo=256, rows=3, heads=4, mr=2, ml=64, ws=D, wb=BIG):
        return L.qmm_attn_kv_mxfp4(q, qt, ldq, kvmx(**(kv or {})), seqs(**(s or {})), None if at is None else Attn(*at), out, ot, ldo, rows, heads, mr, ml,
                                   ws, wb, None)

    for kw, want in CACHES:
        assert f(kv=kw) == want, kw
    for kw, want in SEQS:
        assert f(s=kw) == want, kw
    assert f(q=None) == NULL and f(out=None) == NULL and f(at=None) == NULL and f(qt=2) == FORMAT and f(ot=7) == FORMAT
    assert f(rows=-1) == SHAPE and f(heads=0) == SHAPE and f(heads=3) == SHAPE and f(heads=34, ldq=BIG, ldo=BIG) == SHAPE       # 17 heads share one
    assert f(mr=0) == SHAPE and f(mr=17) == SHAPE and f(ml=0) == SHAPE and f(ml=(1 << 30) + 1) == SHAPE and f(at=(None, 1.0, -1)) == SHAPE
    assert f(ldq=255) == SHAPE and f(ldo=255) == SHAPE
    assert f(q=72) == ARG and f(ldq=260) == ARG and f(qt=0, ldq=258) == ARG and f(out=65) == ARG and f(ot=0, out=66) == ARG and f(at=(2, 1.0, 0)) == ARG
    need = L.qmm_attn_kv_ws_bytes(3, 4, 64, 4096)
    assert need == 3 * 4 * 8 * 66 * 4
    assert f(ml=4096, ws=None) == WORKSPACE and f(ml=4096, wb=need - 1) == WORKSPACE and f(ml=4096, ws=72) == ARG
    assert f(rows=0, q=None, out=None, kv=dict(kq=None), ws=None) == 0
    assert f(s=dict(n=1 << 20), kv=dict(heads=4096), heads=4096, ldq=BIG, ldo=BIG, ml=1 << 30) == SHAPE


@pytest.mark.parametrize("max_len,chunks", [(1, 1), (1024, 1), (1025, 5), (2048, 8), (2049, 5), (8192, 16), (65536, 128), (65537, 65), (1 << 30, 128)])
def test_attend_workspace(max_len, chunks):
    """A workspace for the chunks of max_len, none for one; sizes out of range: 0."""
    want = 0 if chunks == 1 else 5 * 8 * chunks * 130 * 4
    assert qmm.attn_kv_ws_bytes(5, 8, 128, max_len) == want
    for bad in ((0, 8, 128, max_len), (5, 0, 128, max_len), (5, 8, 96, max_len), (5, 8, 128, 0), (5, 8, 128, (1 << 30) + 1), (-1, 8, 128, max_len)):
        assert qmm.attn_kv_ws_bytes(*bad) == 0


@pytest.mark.parametrize("max_len,chunks", [(1, 1), (512, 1), (513, 3), (1024, 4), (4096, 16), (4097, 9), (1 << 30, 128)])
def test_attend_workspace_of_256_dims(max_len, chunks):
    assert qmm.attn_kv_ws_bytes(3, 4, 256, max_len) == (0 if chunks == 1 else 3 * 4 * chunks * 258 * 4)


def test_prompt_refusals():
    L = _lib.lib()

    def f(q=D, ldq=256, k=D, ldk=128, v=D, ldv=128, out=D, ldo=256, cuq=D, cuk=D, n=2, at=(None, 1.0, 0), rows=3, krows=3, heads=4, kvh=2, dim=64, ws=None, wb=0):
        return L.qmm_attn_prompt_bf16(q, ldq, k, ldk, v, ldv, out, ldo, cuq, cuk, n, None if at is None else Attn(*at), rows, krows, heads, kvh, dim, ws, wb, None)

    assert f(q=None) == NULL and f(k=None) == NULL and f(v=None) == NULL and f(out=None) == NULL and f(cuq=None) == NULL and f(at=None) == NULL
    assert f(dim=32) == SHAPE and f(dim=192) == SHAPE and f(rows=-1) == SHAPE and f(krows=-1) == SHAPE and f(n=-1) == SHAPE
    assert f(heads=0) == SHAPE and f(kvh=0) == SHAPE and f(heads=5) == SHAPE and f(at=(None, 1.0, -5)) == SHAPE
    assert f(ldq=248) == SHAPE and f(ldk=120) == SHAPE and f(ldv=120) == SHAPE and f(ldo=248) == SHAPE and f(ldk=(1 << 24) + 8) == SHAPE
    for kw in (dict(ldq=260), dict(ldk=132), dict(ldv=129), dict(ldo=257), dict(q=72), dict(k=68), dict(v=80 + 8), dict(out=66), dict(cuq=66), dict(cuk=67),
               dict(at=(5, 1.0, 0))):
        assert f(**kw) == ARG, kw
    assert f(rows=0, q=None, out=None, cuq=None) == 0 and f(n=0, q=None, cuq=None) == 0
    assert f(rows=0x7fffff00, heads=65536, kvh=65536, ldq=BIG, ldk=1 << 22, ldv=1 << 22, ldo=BIG) == SHAPE
    need = L.qmm_attn_prompt_ws_bytes(40, 9000, 1, 4, 64)
    assert need > 0 and f(rows=40, krows=9000, n=1, ws=D, wb=need - 1) == WORKSPACE and f(rows=40, krows=9000, n=1, ws=72, wb=need) == ARG
    for none in ((4000, 4000, 1, 32, 128), (40, 300, 1, 4, 64), (0, 9000, 1, 4, 64), (40, 9000, 0, 4, 64), (40, 9000, 1, 4, 80)):
        assert L.qmm_attn_prompt_ws_bytes(*none) == 0


@pytest.mark.parametrize("scale,want", [(float("nan"), ARG), (float("inf"), ARG), (-float("inf"), ARG), (2.0 ** 101, ARG), (-2.0 ** 101, ARG)])
def test_scales_that_are_refused(scale, want):
    L = _lib.lib()
    assert L.qmm_attn_kv_mxfp4(D, 1, 256, kvmx(), seqs(), Attn(None, scale, 0), D, 1, 256, 3, 4, 2, 64, D, BIG, None) == want
    assert L.qmm_attn_prompt_bf16(D, 256, D, 128, D, 128, D, 256, D, D, 2, Attn(None, scale, 0), 3, 3, 4, 2, 64, None, 0, None) == want


def test_rope_refusals():
    L = _lib.lib()

    def f(x=D, t=1, ldx=256, out=D, ot=1, ldo=256, rope=None, rows=3, heads=4, dim=64):
        r = dict(freq=D, axis=None, pos=D, ldp=3, axes=3, pairs=16, style=0, scale=1.0) | (rope or {})
        return L.qmm_rope_axes(x, t, ldx, out, ot, ldo, Rope(*r.values()), rows, heads, dim, None)

    assert f(x=None) == NULL and f(out=None) == NULL and f(rope=dict(freq=None)) == NULL and f(rope=dict(pos=None)) == NULL
    assert L.qmm_rope_axes(D, 1, 256, D, 1, 256, None, 3, 4, 64, None) == NULL
    assert f(t=2) == FORMAT and f(ot=-1) == FORMAT
    assert f(rows=-1) == SHAPE and f(heads=0) == SHAPE and f(dim=0) == SHAPE and f(dim=1025, ldx=BIG, ldo=BIG) == SHAPE and f(ldx=255) == SHAPE and f(ldo=255) == SHAPE
    assert f(rope=dict(pairs=33)) == SHAPE and f(rope=dict(pairs=-1)) == SHAPE and f(rope=dict(axes=0)) == SHAPE and f(rope=dict(axes=256)) == SHAPE
    assert f(rope=dict(ldp=2)) == SHAPE and f(rows=0x7fffffff, rope=dict(ldp=BIG), heads=65536, ldx=BIG, ldo=BIG) == SHAPE
    assert f(rope=dict(style=2)) == ARG and f(x=65) == ARG and f(t=0, x=66) == ARG and f(out=128, ot=0, x=129) == ARG and f(rope=dict(freq=66)) == ARG
    assert f(ot=0) == ARG and f(ldo=264) == ARG                           # in place: one type, one stride
    assert f(rows=0, x=None, out=None, rope=dict(freq=None, pos=None)) == 0


# ---- the mirror's checks ----
class Rows(OnDevice):
    """Rows of contiguous values, `ld` apart."""

    def __init__(self, rows, n, dtype=torch.bfloat16, ld=None, dev=0):
        super().__init__(rows * n, dtype)
        self.shape, self.ld, self.dev = (rows, n), ld or n, dev

    def dim(self):
        return 2

    def stride(self, d=None):
        return (self.ld, 1) if d is None else self.ld if d == 0 else 1

    def get_device(self):
        return self.dev

    def is_contiguous(self):
        return self.ld == self.shape[1]


def cache(**kw):
    kv = qmm.KVMXBuf(4, 16, 2, 64, device="cpu")
    for x, n in (("kq", 4 * 2 * 16 * 32), ("ke", 4 * 2 * 16 * 2), ("vq", 4 * 2 * 16 * 32), ("ve", 4 * 2 * 16 * 2)):
        setattr(kv, x, OnDevice(n, torch.uint8))
    for x, v in kw.items():
        setattr(kv, x, v)
    return kv


def other(t):
    t.get_device = lambda: 1
    return t


def test_python_checks_of_the_cache_calls(launched):  # noqa: F811
    i32 = torch.int32
    good = dict(k=Rows(3, 128), v=Rows(3, 128), kv=cache(), cu=OnDevice(3, i32), lens=OnDevice(2, i32), table=Rows(2, 4, i32), rows=3)

    def write(**kw):
        a = good | kw
        qmm.kv_write_mxfp4(a["k"], a["v"], a["kv"], a["cu"], a["lens"], a["table"], a["rows"])

    def read(**kw):
        a = good | kw
        qmm.kv_read_mxfp4(a["kv"], a["cu"], a["lens"], a["table"], a["k"], a["v"], a["rows"])

    def attend(**kw):
        a = good | kw
        qmm.attn_kv_mxfp4(a.get("q", Rows(3, 256)), a["kv"], a["cu"], a["lens"], a["table"], a.get("out", Rows(3, 256)), a["rows"], 4, 2, 64, None,
                          sinks=a.get("sinks"))

    for f in (write, read, attend):
        f()
    n = len(launched)
    assert n == 3
    short = [dict(cu=OnDevice(2, i32)), dict(table=Rows(1, 4, i32)), dict(table=OnDevice(8, i32)), dict(cu=OnDevice(3, torch.int64)), dict(lens=other(OnDevice(2, i32))),
             dict(table=other(Rows(2, 4, i32))), dict(kv=cache(pages=5)), dict(kv=cache(page=32)), dict(kv=cache(heads=4)), dict(kv=cache(kq=OnDevice(4095, torch.uint8))),
             dict(kv=cache(ve=OnDevice(255, torch.uint8))), dict(kv=cache(ke=OnDevice(256, torch.int8))), dict(kv=cache(vq=other(OnDevice(4096, torch.uint8)))),
             dict(table=Rows(2, 4, i32, ld=5))]
    for kw in short:
        for f in (write, read, attend):
            with pytest.raises(QmmError):
                f(**kw)
    for kw in (dict(k=Rows(2, 128)), dict(v=Rows(3, 64)), dict(k=Rows(3, 128, torch.float32)), dict(k=Rows(3, 128, torch.float16), v=Rows(3, 128, torch.float16)),
               dict(k=Rows(3, 128, ld=100)), dict(v=Rows(3, 128, dev=1))):
        for f in (write, read):
            with pytest.raises(QmmError):
                f(**kw)
    for kw in (dict(q=Rows(2, 256)), dict(out=Rows(3, 128)), dict(q=Rows(3, 256, torch.float16)), dict(sinks=OnDevice(3, torch.float32)), dict(out=Rows(3, 256, dev=1)),
               dict(sinks=OnDevice(4, torch.bfloat16))):
        with pytest.raises(QmmError):
            attend(**kw)
    assert len(launched) == n


def test_a_cache_is_checked_again_when_it_changed(launched):  # noqa: F811
    """A cache's tensors are checked once, and again when one was replaced, moved or the current device is another."""
    a = dict(k=Rows(3, 128), v=Rows(3, 128), cu=OnDevice(3, torch.int32), lens=OnDevice(2, torch.int32), table=Rows(2, 4, torch.int32))
    kv = cache()
    f = lambda: qmm.kv_write_mxfp4(a["k"], a["v"], kv, a["cu"], a["lens"], a["table"], 3)      # noqa: E731
    f()
    f()
    kv.pages = 3
    f()
    assert launched[-1][1][5].pages == 3
    kv.kq = OnDevice(10, torch.uint8)
    with pytest.raises(QmmError, match="kv.kq"):
        f()
    kv.kq = OnDevice(4096, torch.uint8)
    f()
    kv.kq.data_ptr = lambda: 8192                                        # set in place
    f()
    assert launched[-1][1][5].kq == 8192
    kv.kq.n = 1                                                          # and cut where it lies
    with pytest.raises(QmmError, match="kv.kq"):
        f()


def test_a_cache_can_be_copied_after_a_call():
    kv = qmm.KVMXBuf(2, 16, 1, 64, device="cpu")
    kv.held = (kv.c(), ())
    kv2 = copy.deepcopy(kv)
    assert kv2.held is None and kv2.pages == 2 and torch.equal(kv2.kq, kv.kq) and kv2.kq.data_ptr() != kv.kq.data_ptr()


def test_python_checks_of_prompt_and_rope(launched):  # noqa: F811
    i32, f32 = torch.int32, torch.float32
    good = dict(q=Rows(3, 256), k=Rows(3, 128), v=Rows(3, 128), cu=OnDevice(3, i32), cuk=None, out=Rows(3, 256), sinks=None, ws=False)

    def prompt(**kw):
        a = good | kw
        qmm.attn_prompt_bf16(a["q"], a["k"], a["v"], a["cu"], a["cuk"], a["out"], 4, 2, 64, sinks=a["sinks"], ws=a["ws"])

    prompt()
    prompt(ws=OnDevice(100, torch.uint8))
    assert launched[0][1][17:19] == (None, 0) and launched[1][1][17:19] == (4096, 100)
    for kw in (dict(q=Rows(3, 256, f32)), dict(k=Rows(3, 128, torch.float16)), dict(v=Rows(2, 128)), dict(out=Rows(2, 256)), dict(cuk=OnDevice(2, i32)),
               dict(cu=OnDevice(3, torch.int64)), dict(sinks=OnDevice(3, f32)), dict(ws=OnDevice(100, f32)), dict(q=Rows(3, 128)), dict(out=Rows(3, 256, dev=1))):
        with pytest.raises(QmmError):
            prompt(**kw)

    def rope(x=Rows(3, 256), y=Rows(3, 256), pos=Rows(3, 3, i32), freq=OnDevice(16, f32), axis=OnDevice(16, torch.uint8), style="halves"):
        qmm.rope_axes(x, y, pos, freq, axis, 3, 4, 64, style=style)

    n = len(launched)
    rope()
    rope(axis=None)
    for kw in (dict(x=Rows(2, 256)), dict(y=Rows(3, 128)), dict(pos=Rows(3, 2, i32)), dict(pos=Rows(3, 3, torch.int64)), dict(freq=OnDevice(16, torch.float64)),
               dict(axis=OnDevice(15, torch.uint8)), dict(axis=OnDevice(16, i32)), dict(style="quarters"), dict(x=Rows(3, 256, torch.float16)), dict(x=Rows(3, 256, dev=1))):
        with pytest.raises(QmmError):
            rope(**kw)
    assert len(launched) == n + 2


def test_host_tensors_are_refused():
    x, i = torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int32)
    kv = qmm.KVMXBuf(1, 16, 1, 64, device="cpu")
    for f in (lambda: qmm.kv_write_mxfp4(x, x, kv, i, i[:2], i.view(1, 3), 2), lambda: qmm.kv_read_mxfp4(kv, i, i[:2], i.view(1, 3), x, x, 2),
              lambda: qmm.attn_kv_mxfp4(x, kv, i, i[:2], i.view(1, 3), x, 2, 1, 1, 16, None), lambda: qmm.attn_prompt_bf16(x, x, x, i, None, x, 1, 1, 64),
              lambda: qmm.rope_axes(x, x, i, torch.ones(4), None, 2, 1, 64)):
        with pytest.raises((QmmError, RuntimeError, AssertionError)):
            f()


# ---- the tests' own definitions ----
def test_oracle_rope_is_a_rotation():
    rng = np.random.default_rng(0)
    x, pos, freq, axis = rng.normal(size=(5, 2, 16)), rng.integers(-99, 99, (3, 5)), rng.uniform(0, 1, 6).astype(np.float32), rng.integers(0, 3, 6)
    for style in ("halves", "neighbours"):
        y, _ = attn_ref.rope(x, pos, freq, axis, style, 1.0)
        back, _ = attn_ref.rope(y, -pos, freq, axis, style, 1.0)
        assert np.allclose(back, x) and np.allclose((y ** 2).sum(-1), (x ** 2).sum(-1)) and np.array_equal(y[:, :, 12:], x[:, :, 12:])


def test_oracle_attention_by_torch():
    """Against torch's softmax, a sink as one more key of value 0."""
    rng = np.random.default_rng(1)
    q, k, v, pos = rng.normal(size=(4, 8)), rng.normal(size=(9, 8)), rng.normal(size=(9, 8)), np.array([-1, 0, 5, 8])
    for window in (0, 3):
        for sink in (None, 0.7):
            o, bound = attn_ref.attention(q, k, v, pos, 0.4, window, sink, 2, 2.0 ** -8, 4)
            j = np.arange(9)
            for i, p in enumerate(pos):
                see = (j <= p) & (j > p - (window or 99))
                if not see.any():
                    assert not o[i].any()
                    continue
                t = torch.tensor(np.concatenate([k[see] @ q[i] * 0.4, [sink] if sink is not None else []]))
                assert np.allclose(o[i], torch.softmax(t, 0).numpy()[:see.sum()] @ v[see])
    assert (bound[1:] > 0).all() and (bound < 0.2).all()


def test_oracle_quantise_is_the_formats():
    x = np.random.default_rng(2).normal(size=(3, 2, 64)).astype(np.float32)
    q, e = attn_ref.quantise(x)
    code, byte = mx_ref.quantise(x.reshape(6, 64))
    assert np.array_equal(attn_ref.values(q, e).reshape(6, 64), mx_ref.values(code, byte)[:, :64])
