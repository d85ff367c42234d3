"""The norms around a block (qmm_postnorm_add_rmsnorm_*) against tests/mx_ref.py, with its derived bounds."""
import numpy as np
import pytest
import torch

import mx_ref
from hipster_amd import qmm
from hipster_amd._lib import QmmError
from tests.gpu_util import dev, host

pytestmark = pytest.mark.gpu

EPS = 1e-6
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def inputs(seed, T, n, ydt, gate, gdt="f32"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, n, generator=g) * 3
    y = (torch.randn(T, n, generator=g) * torch.exp2(torch.randint(-6, 6, (T, 1), generator=g).float())).to(DT[ydt])
    wy, w = 1 + 0.2 * torch.randn(n, generator=g), 1 + 0.2 * torch.randn(n, generator=g)
    shape = {"none": None, "token": (T, 1), "channel": (n,), "value": (T, n)}[gate]
    gt = (torch.randn(shape, generator=g) * 3).to(DT[gdt]) if shape else None
    return [None if t is None else t.cuda() for t in (x, y, wy, w, gt)]


def ref(x, y, wy, w, g, act, alpha):
    f = lambda t: None if t is None else host(t.float())                 # noqa: E731
    return mx_ref.postnorm(f(x), f(y), f(wy), f(w), f(g), act, alpha, EPS)


def check(got, want, bound, what):
    err = np.abs(host(got.float()).astype(np.float64) - want)
    assert (err <= bound).all(), (what, float((err / np.maximum(bound, 1e-300)).max()))


@pytest.mark.parametrize("T,n", [(1, 1), (1, 5120), (3, 7), (2, 130), (5, 1024), (4, 1028), (7, 2880), (3, 4096), (2, 4100), (3, 4101), (2, 5128), (3, 8192),
                                 (2, 8200), (1, 16384), (2, 16383), (70, 256)])
@pytest.mark.parametrize("ydt,post,gate,act,gdt", [("f32", True, "none", "none", "f32"), ("bf16", True, "value", "silu", "bf16"), ("f32", False, "token", "sigmoid", "f32"),
                                                   ("bf16", False, "channel", "none", "f32"), ("f32", True, "value", "sigmoid", "f32")])
def test_bf16_out(gpu, T, n, ydt, post, gate, act, gdt):
    x, y, wy, w, g = inputs(T * 131 + n, T, n, ydt, gate, gdt)
    wy = wy if post else None
    alpha = float(np.float32(0.22))
    xo, xn, bo, bn = ref(x, y, wy, w, g, act, alpha)
    out, xb = torch.full((T + 1, n), -7.0, device="cuda"), torch.full((T + 1, n), -7.0, dtype=torch.bfloat16, device="cuda")
    x0 = host(x).copy()
    qmm.postnorm_add_rmsnorm_bf16(x, y, wy, w, xb, T, n, EPS, gate=g, act=act, alpha=alpha, xo=out)
    check(out[:T], xo, bo, "xo")
    check(xb[:T], xn, bn + 2.0 ** -8 * (np.abs(xn) + bn), "xn")
    assert (host(out[T]) == -7).all() and (host(xb[T].float()) == -7).all() and np.array_equal(host(x), x0)
    inplace, xb2 = x.clone(), torch.empty_like(xb)
    qmm.postnorm_add_rmsnorm_bf16(inplace, y, wy, w, xb2, T, n, EPS, gate=g, act=act, alpha=alpha)       # x is written back
    assert torch.equal(inplace, out[:T]) and torch.equal(xb2[:T], xb[:T])


@pytest.mark.parametrize("T,n", [(1, 32), (3, 2048), (2, 5120), (5, 6144), (1, 16384)])
def test_quant_out(gpu, T, n):
    """xn in f32, and the q8 that quantize_x_q8 makes of it, bit for bit."""
    x, y, wy, w, g = inputs(n, T, n, "bf16", "token", "bf16")
    xo, xn, bo, bn = ref(x, y, wy, w, g, "sigmoid", 1.0)
    got, xq = torch.empty(T, n, device="cuda"), qmm.XQ8Buf(T, n, with_ds=True)
    qmm.postnorm_add_rmsnorm_quant(x, y, wy, w, got, xq, T, n, EPS, gate=g, act="sigmoid")
    check(x, xo, bo, "xo")
    check(got, xn, bn, "xn")
    want = qmm.XQ8Buf(T, n)
    qmm.quantize_x_q8(got, want, T, n)
    for a, b in ((xq.q, want.q), (xq.d, want.d), (xq.s, want.s), (xq.ds[..., 0], want.d), (xq.ds[..., 1], want.s)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("T,n", [(1, 3), (3, 100), (2, 1000), (4, 2880), (2, 5120), (3, 4099), (2, 8190), (1, 16383)])
def test_mxfp4_out(gpu, T, n):
    """The codes that quantize_mxfp4 makes of the f32 xn, bit for bit, padding included."""
    x, y, wy, w, g = inputs(n, T, n, "f32", "value")
    b = qmm.XMXBuf(T, n)
    b.q.fill_(0x77); b.e.fill_(0x77)
    out = torch.empty_like(x)
    qmm.postnorm_add_rmsnorm_mxfp4(x, y, wy, w, b, T, n, EPS, gate=g, act="silu", xo=out)
    if n % 32 == 0:
        xn, xq = torch.empty(T, n, device="cuda"), qmm.XQ8Buf(T, n)
        qmm.postnorm_add_rmsnorm_quant(x, y, wy, w, xn, xq, T, n, EPS, gate=g, act="silu", xo=torch.empty_like(x))
        code, byte = mx_ref.quantise(host(xn))
        assert np.array_equal(host(b.e), byte) and np.array_equal(host(b.q), mx_ref.pack(code))
    # any n: each value within half a step of its block plus the bound of xn (a step is at most a third of 4 .. 6:
    # values up to 8 units saturate at 6, two units; below, half a step is at most one unit)
    xo, xn, bo, bn = ref(x, y, wy, w, g, "silu", 1.0)
    check(out, xo, bo, "xo")
    v = torch.empty(T, n, device="cuda")
    qmm.dequant_mxfp4(b, v, T, n)
    unit = np.exp2(np.repeat(host(b.e).astype(np.float64), 32, 1)[:, :n] - 127)
    assert (np.abs(host(v) - xn) <= 2 * unit + bn).all()
    codes = host(b.q)
    full = np.stack([codes & 15, codes >> 4], -1).reshape(T, -1)
    assert not full[:, n:].any() and not host(b.e)[:, -(-n // 32):].any()


def test_strided_block_output_and_gate(gpu):
    """y and a gate that are columns of one wider product, aligned and not."""
    T, n = 6, 640
    for off in (0, 4, 3):
        wide = torch.randn(T, 2 * n + 40).cuda()
        y, g = wide[:, off:off + n], wide[:, n + 20 + off:2 * n + 20 + off]
        x, _, wy, w, _ = inputs(off, T, n, "f32", "none")
        xo, xn, bo, bn = ref(x, y, wy, w, g, "silu", 1.0)
        xb = torch.empty(T, n, dtype=torch.bfloat16, device="cuda")
        qmm.postnorm_add_rmsnorm_bf16(x, y, wy, w, xb, T, n, EPS, gate=g, act="silu")
        check(x, xo, bo, "xo")
        check(xb, xn, bn + 2.0 ** -8 * (np.abs(xn) + bn), "xn")


def test_zero_rows_and_not_finite(gpu):
    x, y = torch.zeros(4, 256, device="cuda"), torch.zeros(4, 256, device="cuda")
    x[2], y[2] = 1.0, float("nan")
    y[3, 5] = float("inf")
    w = torch.ones(256, device="cuda")
    xb = torch.empty(4, 256, dtype=torch.bfloat16, device="cuda")
    qmm.postnorm_add_rmsnorm_bf16(x, y, w, w, xb, 4, 256, EPS)
    out = host(xb.float())
    assert (out[:2] == 0).all() and np.isnan(out[2]).all() and np.isnan(out[3]).any()
    b = qmm.XMXBuf(4, 256)
    qmm.postnorm_add_rmsnorm_mxfp4(torch.ones(4, 256, device="cuda"), y, w, w, b, 4, 256, EPS)
    e = host(b.e)
    assert (e[:2] == 124).all() and (e[2] == 255).all()                  # 1 / sqrt(1 + eps) < 1: scale 2^-3


def test_plain_residual_norm_is_the_old_one(gpu):
    """Without a post norm, a gate or a scale it is add_rmsnorm_bf16 (its sums in another order)."""
    x, y, _, w, _ = inputs(9, 5, 2048, "f32", "none")
    x2, xb, xb2 = x.clone(), torch.empty(5, 2048, dtype=torch.bfloat16, device="cuda"), torch.empty(5, 2048, dtype=torch.bfloat16, device="cuda")
    qmm.add_rmsnorm_bf16(x2, y, w, xb2, 5, 2048, EPS)
    qmm.postnorm_add_rmsnorm_bf16(x, y, None, w, xb, 5, 2048, EPS)
    assert torch.equal(x, x2)
    assert (np.abs(host(xb.float()) - host(xb2.float())) <= 2.0 ** -7 * np.abs(host(xb2.float()))).all()


def test_refusals(gpu):
    x, y, wy, w, g = inputs(1, 4, 64, "f32", "value")
    xb = torch.empty(4, 64, dtype=torch.bfloat16, device="cuda")
    f = lambda **k: qmm.postnorm_add_rmsnorm_bf16(k.get("x", x), k.get("y", y), wy, k.get("w", w), k.get("xb", xb), k.get("T", 4), 64, EPS,     # noqa: E731
                                                  gate=k.get("gate"), act=k.get("act", "none"))
    for bad in (dict(y=y.half()), dict(x=x.double()), dict(xb=xb.float()), dict(T=5), dict(w=w[:63]), dict(y=y.t()), dict(gate=g[:, :63]), dict(gate=g[:2]),
                dict(gate=g.half()), dict(act="gelu"), dict(gate=g.cpu()), dict(gate=g[:3, :1])):
        with pytest.raises(QmmError):
            f(**bad)
    with pytest.raises(QmmError):
        qmm.postnorm_add_rmsnorm_quant(x, y, wy, w, torch.empty_like(x), qmm.XQ8Buf(3, 64), 4, 64, EPS)


def test_graph(gpu):
    x, y, wy, w, g = inputs(3, 33, 1024, "bf16", "value", "bf16")
    out, xb = torch.empty_like(x), torch.empty(33, 1024, dtype=torch.bfloat16, device="cuda")
    work = lambda: qmm.postnorm_add_rmsnorm_bf16(x, y, wy, w, xb, 33, 1024, EPS, gate=g, act="silu", xo=out)      # noqa: E731
    work()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        work()
    for i in range(3):
        x.copy_(torch.randn(33, 1024)); y.copy_(torch.randn(33, 1024))
        out.fill_(0)
        graph.replay()
        xo, xn, bo, bn = ref(x, y, wy, w, g, "silu", 1.0)
        check(out, xo, bo, "xo")
        check(xb, xn, bn + 2.0 ** -8 * (np.abs(xn) + bn), "xn")
        work()
        torch.cuda.synchronize()
