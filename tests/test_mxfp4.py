"""MXFP4 entry points without a GPU: the host repack of GGUF rows, packed sizes, and refusals (status codes
before any device work; the calls below never reach a device)."""
import ctypes

import numpy as np
import pytest
import torch

import mx_ref
from hipster_amd import _lib, qmm
from hipster_amd._lib import Gate, QmmError, RouteRule, XMX, XQ8

FORMAT, SHAPE, NULL, ARG = -1, -2, -3, -6
D = ctypes.c_void_p(64)                       # a non-null, aligned pointer that nothing dereferences
X = XMX(64, 64)


@pytest.mark.parametrize("K", [32, 96, 128, 640, 2880])
def test_repack_gguf_row(K):
    g = np.random.default_rng(K)
    blocks = g.integers(0, 256, (K // 32, 17), dtype=np.uint8)
    q, e = qmm.repack_row_mxfp4(blocks.reshape(-1), K)
    code = np.concatenate([blocks[:, 1:] & 15, blocks[:, 1:] >> 4], 1).reshape(1, -1)     # weight i, then i + 16
    pad = np.zeros((1, 128 * mx_ref.steps(K)), np.uint8)
    pad[:, :K] = code
    assert np.array_equal(q, mx_ref.pack(pad)[0])
    assert np.array_equal(e[:K // 32], blocks[:, 0]) and not e[K // 32:].any()


def test_repack_refusals():
    L = _lib.lib()
    b = np.zeros(64, np.uint8)
    assert L.qmm_repack_row_mxfp4(None, b.ctypes.data, b.ctypes.data, 32) == NULL
    assert L.qmm_repack_row_mxfp4(b.ctypes.data, b.ctypes.data, b.ctypes.data, 40) == SHAPE
    with pytest.raises(QmmError):
        qmm.repack_row_mxfp4(b[:16], 32)


def test_weight_bytes():
    assert qmm.mxfp4_weight_bytes(16, 512) == 4 * 1024 + 256
    assert qmm.mxfp4_weight_bytes(17, 129) == 2 * (2 * 1024 + 256)
    assert qmm.mxfp4_weight_bytes(1, 1) == 1024 + 256
    assert qmm.mxfp4_weight_bytes(0, 128) == 0 and qmm.mxfp4_weight_bytes(16, 0) == 0 and qmm.mxfp4_weight_bytes(16, (1 << 24) + 1) == 0


def test_quantise_refusals():
    L = _lib.lib()
    assert L.qmm_quantize_mxfp4(None, 0, 64, X, 1, 64, None) == NULL
    assert L.qmm_quantize_mxfp4(D, 0, 64, XMX(None, 64), 1, 64, None) == NULL
    assert L.qmm_quantize_mxfp4(D, 2, 64, X, 1, 64, None) == FORMAT
    assert L.qmm_quantize_mxfp4(D, 0, 63, X, 1, 64, None) == SHAPE              # row stride below K
    assert L.qmm_quantize_mxfp4(D, 0, 64, X, 1, 0, None) == SHAPE
    assert L.qmm_quantize_mxfp4(D, 0, 64, X, -1, 64, None) == SHAPE
    assert L.qmm_quantize_mxfp4(D, 0, 64, XMX(72, 64), 1, 64, None) == ARG      # q not 16-byte aligned
    assert L.qmm_quantize_mxfp4(ctypes.c_void_p(66), 0, 64, X, 1, 64, None) == ARG
    assert L.qmm_quantize_mxfp4(D, 0, 1 << 24, X, 1 << 20, 1 << 24, None) == SHAPE    # more pieces than a grid has threads
    assert L.qmm_quantize_mxfp4(D, 0, 64, X, 0, 64, None) == 0
    assert L.qmm_dequant_mxfp4(X, None, 0, 1, 64, None) == NULL
    assert L.qmm_dequant_mxfp4(X, D, 3, 1, 64, None) == FORMAT
    assert L.qmm_dequant_mxfp4(X, D, 0, 1, 0, None) == SHAPE
    assert L.qmm_dequant_mxfp4(X, D, 0, 0, 64, None) == 0
    assert L.qmm_pack_mxfp4(X, None, 16, 64, None) == NULL
    assert L.qmm_pack_mxfp4(X, D, 0, 64, None) == SHAPE
    assert L.qmm_pack_mxfp4(X, ctypes.c_void_p(72), 16, 64, None) == ARG


def test_product_refusals():
    L = _lib.lib()
    for f in (lambda W, x, y, t, m, N, K: L.qmm_gemv_mxfp4(W, x, y, t, m, N, K, None),
              lambda W, x, y, t, m, N, K: L.qmm_gemm_mxfp4(W, x, y, t, m, N, K, None)):
        assert f(None, X, D, 0, 1, 16, 64) == NULL
        assert f(D, XMX(64, None), D, 0, 1, 16, 64) == NULL
        assert f(D, X, None, 0, 1, 16, 64) == NULL
        assert f(D, X, D, 5, 1, 16, 64) == FORMAT
        assert f(D, X, D, 0, 1, 0, 64) == SHAPE
        assert f(D, X, D, 0, 1, 16, 0) == SHAPE
        assert f(D, X, D, 0, 1, 16, (1 << 24) + 1) == SHAPE
        assert f(D, X, D, 0, -1, 16, 64) == SHAPE
        assert f(ctypes.c_void_p(72), X, D, 0, 1, 16, 64) == ARG
        assert f(D, X, ctypes.c_void_p(66), 0, 1, 16, 64) == ARG
        assert f(D, X, D, 0, 0, 16, 64) == 0
    assert L.qmm_gemv_mxfp4(D, X, D, 0, 65, 16, 64, None) == SHAPE


def test_expert_product_refusals():
    L = _lib.lib()
    one = qmm.mxfp4_weight_bytes(32, 64)
    f = lambda T=1, slots=4, E=8, eb=one, ids=D, Wsh=None: L.qmm_gemv_moe_mxfp4(D, Wsh, eb, ids, X, D, 0, T, slots, E, 32, 64, 0, None)   # noqa: E731
    assert f(ids=None) == NULL
    assert f(T=17) == SHAPE and f(T=-1) == SHAPE and f(slots=17) == SHAPE and f(slots=0) == SHAPE and f(E=0) == SHAPE
    assert f(eb=one + 8) == ARG and f(eb=one - 16) == ARG and f(Wsh=ctypes.c_void_p(72)) == ARG
    assert f(T=0) == 0
    g = lambda tiles=D, counts=D, n=4, eb=one, tab=D: L.qmm_moe_gemm_mxfp4(D, None, eb, tiles, counts, n, tab, X, D, 0, 32, 64, None)   # noqa: E731
    assert g(tiles=None) == NULL and g(counts=None) == NULL and g(n=-1) == SHAPE
    assert g(eb=one + 8) == ARG and g(tab=ctypes.c_void_p(66)) == ARG
    assert g(n=0) == 0


def test_route_refusals():
    L = _lib.lib()

    def f(logits=D, T=1, E=64, k=4, stride=64, **kw):
        r = RouteRule(None, 1.0, 0, 1, 1, 1, 1, 0)
        for n, v in kw.items():
            setattr(r, n, v)
        return L.qmm_moe_route_groups(logits, stride, ctypes.byref(r), D, D, T, E, k, None)

    assert f(logits=None) == NULL and L.qmm_moe_route_groups(D, 64, None, D, D, 1, 64, 4, None) == NULL
    assert f(score=2) == ARG and f(shared=3) == ARG and f(best=3) == ARG and f(best=0) == ARG
    assert f(E=1025, stride=2000) == SHAPE and f(E=0) == SHAPE and f(k=17) == SHAPE and f(k=0) == SHAPE and f(T=-1) == SHAPE
    assert f(stride=63) == SHAPE and f(shared=1) == SHAPE                        # no room for the shared gate's logit
    assert f(groups=3) == SHAPE and f(groups=0) == SHAPE and f(groups=65) == SHAPE
    assert f(groups=8, keep=9) == SHAPE and f(groups=8, keep=0) == SHAPE
    assert f(groups=64, keep=2, k=3) == SHAPE                                    # two experts stay, three are asked for
    assert f(E=4, stride=4, k=5) == SHAPE
    assert f(T=0) == 0


def test_postnorm_refusals():
    L = _lib.lib()
    q8 = XQ8(64, 64, 64, 0)

    def f(x=D, y=D, yt=0, ldy=64, wy=None, gate=None, xo=D, w=D, out=D, T=1, n=64):
        return L.qmm_postnorm_add_rmsnorm_bf16(x, y, yt, ldy, wy, None if gate is None else ctypes.byref(gate), 1.0, xo, w, out, T, n, 1e-6, None)

    assert f(x=None) == NULL and f(y=None) == NULL and f(xo=None) == NULL and f(w=None) == NULL and f(out=None) == NULL
    assert f(yt=4) == FORMAT and f(n=0) == SHAPE and f(n=16385, ldy=20000) == SHAPE and f(T=-1) == SHAPE and f(ldy=63) == SHAPE
    assert f(gate=Gate(64, 0, 7, 0, 1)) == FORMAT and f(gate=Gate(64, 0, 0, 3, 1)) == ARG and f(gate=Gate(64, 63, 0, 0, 1)) == SHAPE
    assert f(gate=Gate(66, 64, 0, 0, 1)) == ARG and f(y=ctypes.c_void_p(66)) == ARG and f(out=ctypes.c_void_p(65)) == ARG
    assert f(T=0) == 0
    assert L.qmm_postnorm_add_rmsnorm_quant(D, D, 0, 100, None, None, 1.0, D, D, D, q8, 1, 100, 1e-6, None) == SHAPE      # n % 32
    assert L.qmm_postnorm_add_rmsnorm_quant(D, D, 0, 64, None, None, 1.0, D, D, D, XQ8(64, 64, 0, 0), 1, 64, 1e-6, None) == NULL
    assert L.qmm_postnorm_add_rmsnorm_mxfp4(D, D, 0, 64, None, None, 1.0, D, D, XMX(64, None), 1, 64, 1e-6, None) == NULL


def test_python_refusals_on_host_tensors():
    """The Python mirror refuses what it can see (host tensors) before the library is called."""
    t = torch.zeros(4, 64)
    with pytest.raises(QmmError):
        qmm.quantize_mxfp4(t, qmm.XMXBuf(4, 64, device="cpu"), 4, 64)
    with pytest.raises(QmmError):
        qmm.moe_route_groups(t, t.int(), t, 4, 64, 4)
    with pytest.raises(QmmError):
        qmm.postnorm_add_rmsnorm_bf16(t, t, None, t[0], t.bfloat16(), 4, 64, 1e-6)


def test_sizes_near_the_int_limit():
    """A tile past the last row would leave the ints that count rows: refused."""
    L, big = _lib.lib(), (1 << 31) - 1
    assert qmm.mxfp4_weight_bytes(big, 32) == 0 and qmm.mxfp4_weight_bytes(big - 255, 32) > 0
    assert L.qmm_pack_mxfp4(X, D, big, 32, None) == SHAPE
    assert L.qmm_gemv_mxfp4(D, X, D, 0, 1, big, 32, None) == SHAPE
    assert L.qmm_gemm_mxfp4(D, X, D, 0, 1, big, 32, None) == SHAPE
    assert L.qmm_gemm_mxfp4(D, X, D, 0, big, 32, 32, None) == SHAPE
    assert L.qmm_gemm_mxfp4_tile(big, 32, 32) == SHAPE and L.qmm_gemm_mxfp4_tile(32, big, 32) == SHAPE
    assert L.qmm_moe_gemm_mxfp4(D, None, 1 << 20, D, D, 1, None, X, D, 0, big, 32, None) == SHAPE
    assert L.qmm_gemv_moe_mxfp4(D, None, 1 << 20, D, X, D, 0, 1, 1, 1, big, 32, 0, None) == SHAPE


def test_experts_a_negative_distance_apart():
    W = torch.zeros(4096, dtype=torch.uint8)
    for call in (lambda: qmm.gemv_moe_mxfp4(W, None, -16, None, None, None, 1, 1, 2, 16, 32), lambda: qmm.moe_gemm_mxfp4(W, None, -16, None, None, 1, None, None, None, 16, 32)):
        with pytest.raises(QmmError, match="apart"):
            call()
