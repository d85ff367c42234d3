"""What the MXFP4 block operators refuse before a device is asked: status codes of the library, and the checks of the Python
mirror on stand-ins for device tensors.  No call below reaches a device."""
import ctypes

import numpy as np
import pytest
import torch

import mx_ref
from gguf_writer import STR, write_gguf
from hipster_amd import _lib, gguf, qmm
from hipster_amd._lib import QmmError, XMX

FORMAT, SHAPE, NULL, ARG = -1, -2, -3, -6
D = ctypes.c_void_p(64)                       # a non-null, aligned pointer that nothing dereferences
X = XMX(64, 64)


class OnDevice:
    """A tensor as the checks see one: on device 0, contiguous, its address nothing that is read."""
    is_cuda = True

    def __init__(self, n, dtype):
        self.n, self.dtype, self.device = n, dtype, "cuda:0"

        self.shape = (n,)

    def is_contiguous(self):
        return True

    def stride(self, dim):
        return 1

    def get_device(self):
        return 0

    def numel(self):
        return self.n

    def data_ptr(self):
        return 4096


class Rows:
    """An XMXBuf of such tensors."""

    def __init__(self, rows, K):
        self.rows, self.K = rows, K
        self.q, self.e = (OnDevice(rows * per * qmm.mxfp4_steps(K), torch.uint8) for per in (64, 4))


@pytest.fixture
def launched(monkeypatch):
    """The arguments of the library calls that get through, which do nothing."""
    calls = []

    class Lib:
        def __getattr__(self, name):
            return lambda *a: calls.append((name, a)) or 0

    monkeypatch.setattr(qmm, "_device", lambda: 0)
    monkeypatch.setattr(qmm, "_raw_stream", lambda d: 0)
    monkeypatch.setattr(_lib, "lib", lambda: Lib())
    return calls


def test_sorted_experts_sizes(launched):
    """D, the table, x and the experts' weights hold what the tiles may name, or the call is refused."""
    E, TS, N, K, cap = 4, 24, 40, 300, 9
    one = 3 * (3 * 1024 + 256)
    i32, u8, f32 = torch.int32, torch.uint8, torch.float32

    def call(w=E * one, tab=TS, d=TS * N, xr=6, eb=one, **kw):
        qmm.moe_gemm_mxfp4(OnDevice(w, u8), None, eb, OnDevice(3 * cap, i32), OnDevice(2, i32), cap, None if tab is None else OnDevice(tab, i32),
                           Rows(xr, K), OnDevice(d, f32), N, K, **kw)

    call()
    call(tab=None, xr=TS)
    call(tab=None, xr=TS + 8, rows=TS)
    call(tab=TS + 8, rows=TS)
    call(nexperts=E)
    assert len(launched) == 5
    for kw, what in ((dict(d=TS * N - 1), "D holds"), (dict(d=6 * N), "D holds"), (dict(tab=None, xr=TS, d=TS * N - N), "D holds"),
                     (dict(tab=TS - 1, rows=TS), "rowtab holds"), (dict(nexperts=E + 1), "W holds"), (dict(w=one - 16), "W holds")):
        with pytest.raises(QmmError, match=what):
            call(**kw)
    assert len(launched) == 5
    # the bounds that the device gets
    name, a = launched[0]
    assert name == "qmm_moe_gemm_mxfp4_n" and (a[3], a[8], a[10]) == (E, TS, 6)


def test_sorted_experts_refusals():
    L, one = _lib.lib(), qmm.mxfp4_weight_bytes(32, 64)

    def f(W=D, eb=one, E=2, tiles=D, counts=D, n=4, tab=D, rows=8, xrows=8, N=32, K=64, dtype=0):
        return L.qmm_moe_gemm_mxfp4_n(W, None, eb, E, tiles, counts, n, tab, rows, X, xrows, D, dtype, N, K, None)

    assert f(W=None) == NULL and f(tiles=None) == NULL and f(counts=None) == NULL and f(dtype=2) == FORMAT
    assert f(E=0) == SHAPE and f(rows=-1) == SHAPE and f(xrows=0) == SHAPE and f(tab=None, xrows=7) == SHAPE and f(n=-1) == SHAPE
    assert f(eb=one - 16) == ARG and f(eb=0) == ARG and f(eb=one + 8) == ARG and f(tab=ctypes.c_void_p(66)) == ARG
    assert f(rows=0) == 0 and f(rows=0, xrows=0) == 0 and f(n=0) == 0


@pytest.mark.parametrize("ds", [False, True])
def test_norm_to_q8_elsewhere(launched, ds):
    """The q8 rows of a norm are on the device that it runs on, as its other tensors are."""
    n, v = 64, OnDevice(64, torch.float32)
    good = qmm.XQ8Buf(1, n, device="cpu", with_ds=ds)
    good.q, good.d, good.s = OnDevice(n, torch.int8), OnDevice(2, torch.float32), OnDevice(2, torch.float32)
    good.ds = OnDevice(4, torch.float32) if ds else None
    qmm.postnorm_add_rmsnorm_quant(v, v, v, v, v, good, 1, n, 1e-6)
    assert len(launched) == 1
    for part in ("q", "d", "s") + (("ds",) if ds else ()):
        for wrong in (getattr(qmm.XQ8Buf(1, n, device="cpu", with_ds=ds), part), "other"):
            bad = qmm.XQ8Buf(1, n, device="cpu", with_ds=ds)
            bad.q, bad.d, bad.s, bad.ds = good.q, good.d, good.s, good.ds
            if wrong == "other":                                         # of another device
                wrong = OnDevice(getattr(good, part).n, getattr(good, part).dtype)
                wrong.get_device = lambda: 1
            setattr(bad, part, wrong)
            with pytest.raises(QmmError, match="xq"):
                qmm.postnorm_add_rmsnorm_quant(v, v, v, v, v, bad, 1, n, 1e-6)
    assert len(launched) == 1


def test_calls_for_no_rows():
    """Nothing to do, and no buffers to do it in (an empty tensor has no address); the other arguments are checked as ever."""
    L, no, eb = _lib.lib(), XMX(None, None), qmm.mxfp4_weight_bytes(32, 64)
    r = _lib.RouteRule(None, 1.0, 0, 1, 1, 1, 1, 0)
    q8 = _lib.XQ8(None, None, None, None)
    calls = [lambda t, n=64: L.qmm_quantize_mxfp4(None, 0, 64, no, t, n, None), lambda t, n=64: L.qmm_dequant_mxfp4(no, None, 0, t, n, None),
             lambda t, n=64: L.qmm_gemv_mxfp4(D, no, None, 0, t, 32, n, None), lambda t, n=64: L.qmm_gemm_mxfp4(D, no, None, 0, t, 32, n, None),
             lambda t, n=64: L.qmm_gemv_moe_mxfp4(D, None, eb, None, no, None, 0, t, 4, 8, 32, n, 0, None),
             lambda t, n=64: L.qmm_moe_gemm_mxfp4_n(D, None, eb, 8, D, D, 4, None, t, no, t, None, 0, 32, n, None),
             lambda t, n=64: L.qmm_moe_route_groups(None, n, ctypes.byref(r), None, None, t, n, 4, None),
             lambda t, n=64: L.qmm_postnorm_add_rmsnorm_bf16(None, None, 0, n, None, None, 1.0, None, D, None, t, n, 1e-6, None),
             lambda t, n=64: L.qmm_postnorm_add_rmsnorm_quant(None, None, 0, n, None, None, 1.0, None, D, None, q8, t, n, 1e-6, None),
             lambda t, n=64: L.qmm_postnorm_add_rmsnorm_mxfp4(None, None, 0, n, None, None, 1.0, None, D, no, t, n, 1e-6, None)]
    for i, call in enumerate(calls):
        assert call(0) == 0 and call(1) == NULL and call(0, 0) == SHAPE, i


def test_launches_beyond_the_grid():
    """More threads than a launch may have: refused before anything is launched."""
    L, eb = _lib.lib(), 1 << 40
    assert L.qmm_pack_mxfp4(X, D, (1 << 30) + 16, 32, None) == SHAPE                                  # 2^26 strips and one, a wave each
    assert L.qmm_gemv_mxfp4(D, X, D, 0, 1, (1 << 28) + 32, 1 << 15, None) == SHAPE                    # 2^23 pairs of strips, eight waves each
    assert L.qmm_gemv_moe_mxfp4(D, None, eb, D, X, D, 0, 1, 1, 1, (1 << 28) + 32, 1 << 15, 0, None) == SHAPE
    assert L.qmm_gemm_mxfp4(D, X, D, 0, 1 << 30, 1 << 20, 32, None) == SHAPE
    assert L.qmm_moe_gemm_mxfp4_n(D, None, eb, 1, D, D, 1 << 24, None, 1, X, 1, D, 0, 129, 32, None) == SHAPE
    big = ((1 << 24) + 1, (1 << 23) + 1, (1 << 22) + 1)
    for T, n in zip(big, (128, 5632, 8320)):
        assert L.qmm_postnorm_add_rmsnorm_bf16(D, D, 0, n, None, None, 1.0, D, D, D, T, n, 1e-6, None) == SHAPE
    r = _lib.RouteRule(None, 1.0, 0, 1, 1, 1, 1, 0)
    assert L.qmm_moe_route_groups(D, 8, ctypes.byref(r), D, D, (1 << 26) + 4, 8, 2, None) == SHAPE


def test_weights_of_a_model_file(tmp_path):
    """A file with MXFP4 tensors opens (ggml type 39, 17 bytes a block), and its rows go to the rows that are packed."""
    E, N, K = 2, 3, 160
    blocks = np.random.default_rng(1).integers(0, 255, (E * N, K // 32, 17), dtype=np.uint8)
    path = str(tmp_path / "m.gguf")
    write_gguf(path, [("a", 0, (8,), np.arange(8, dtype=np.float32)), ("w", gguf.GType.MXFP4, (K, N, E), blocks), ("b", 0, (4,), np.ones(4, np.float32))],
               {"general.architecture": (STR, "x")})
    assert gguf.gtype_block(gguf.GType.MXFP4) == (32, 17) and gguf.gtype_row_bytes(gguf.GType.MXFP4, K) == K // 32 * 17
    with gguf.GGUF(path) as g:
        assert g.get("b").array().view(np.float32).tolist() == [1.0] * 4
        t = g.get("w")
        assert t.type == 39 and t.ne == (K, N, E, 1) and t.nbytes == blocks.size
        for raw in (t.array(), g.read_tensor(t)):
            for row, want in zip(raw.reshape(E * N, -1), blocks):
                q, e = qmm.repack_row_mxfp4(row, K)
                code = np.stack([q & 15, q >> 4], 1).reshape(1, -1)
                byte = np.zeros((1, 8), np.uint8)
                byte[0, :K // 32] = want[:, 0]
                assert np.array_equal(e, byte[0])
                # ggml: weight i of a block is the low half of byte i, weight i + 16 the high half, times 2^(byte - 127)
                level = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6])
                vals = level[np.concatenate([want[:, 1:] & 15, want[:, 1:] >> 4], 1)] * np.exp2(want[:, :1].astype(np.float64) - 127)
                assert np.array_equal(mx_ref.values(code, byte)[0, :K], vals.reshape(-1))
        with pytest.raises(QmmError, match="QMM_ERR_FORMAT"):           # no layout of the q8 products
            gguf.upload_lin(g, "w", device="cpu")
    for other in (31, 38, 40):
        write_gguf(path, [("t", other, (32,), np.zeros(32, np.uint8))])
        with pytest.raises(QmmError, match="QMM_ERR_FORMAT"):
            gguf.GGUF(path)
