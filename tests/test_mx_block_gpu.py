"""The MXFP4 operators run one after another as a decoder block uses them: norm around the block, routing, sorting,
experts' products, combination.  Each stage is held against its definition in float64 on what the stage before it
left on the device, so that a bound is one operator's own; and the whole run is captured and replayed."""
import numpy as np
import pytest
import torch

import mx_ref
from hipster_amd import qmm
from tests.gpu_util import dev, host

pytestmark = pytest.mark.gpu

EPS = 1e-6
E, K_TOP, SLOTS, H, F = 24, 3, 4, 416, 224                               # experts, chosen, + the shared one, width, an expert's width
RULE = dict(score="sigmoid", groups=6, keep=3, best=2, renorm=True, scale=2.5, shared="gate")


def packed(rng, n, N, K):
    """n weights packed one after another, and their values."""
    eb, vals = qmm.mxfp4_weight_bytes(N, K), []
    W = torch.empty(n, eb, dtype=torch.uint8, device="cuda")
    for i in range(n):
        c, b = mx_ref.random_rows(rng, N, K, spread=1)
        b[:, :-(-K // 32)] -= 6                                          # about 1 / sqrt(K) in size
        qmm.pack_mxfp4(dev(mx_ref.pack(c)), dev(b), W[i], N, K)
        vals.append(mx_ref.values(c, b))
    return W, vals


class Block:
    """Weights and every buffer of a block, once."""

    def __init__(self, T, seed):
        rng = np.random.default_rng(seed)
        f32 = lambda *s: torch.zeros(s, device="cuda")                   # noqa: E731
        i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
        self.T, TS = T, T * SLOTS
        self.Wg, self.vg = packed(rng, E + 1, F, H)
        self.Wu, self.vu = packed(rng, E + 1, F, H)
        self.Wd, self.vd = packed(rng, E + 1, H, F)
        self.router = dev((rng.standard_normal((E + 1, H)) / 8).astype(np.float32))
        self.bias = dev((rng.standard_normal(E) / 10).astype(np.float32))
        self.wy, self.w = (dev((1 + 0.2 * rng.standard_normal(H)).astype(np.float32)) for _ in range(2))
        self.x, self.y0 = f32(T, H), torch.zeros(T, H, dtype=torch.bfloat16, device="cuda")
        self.xo, self.xn, self.xq8, self.xq = f32(T, H), f32(T, H), qmm.XQ8Buf(T, H), qmm.XMXBuf(T, H)
        self.logits, self.ids, self.p = f32(T, E + 1), i32(T, SLOTS), f32(T, SLOTS)
        self.cap = qmm.moe_tiles_capacity(T, SLOTS, E)
        self.kpos, self.rowtok, self.tiles, self.counts = i32(TS), i32(TS), i32(self.cap, 3), i32(2)
        self.straight = torch.arange(TS, dtype=torch.int32, device="cuda")
        self.g, self.u, self.h = f32(TS, F), f32(TS, F), torch.zeros(TS, F, dtype=torch.bfloat16, device="cuda")
        self.hq, self.d, self.y = qmm.XMXBuf(TS, F), f32(TS, H), f32(T, H)
        self.xo2, self.xb2 = f32(T, H), torch.zeros(T, H, dtype=torch.bfloat16, device="cuda")

    def feed(self, seed):
        g = torch.Generator().manual_seed(seed)
        self.x.copy_(torch.randn(self.T, H, generator=g))
        self.y0.copy_(torch.randn(self.T, H, generator=g) * 3)

    def run(self):
        T, TS, few = self.T, self.T * SLOTS, self.T <= 16
        qmm.postnorm_add_rmsnorm_quant(self.x, self.y0, self.wy, self.w, self.xn, self.xq8, T, H, EPS, alpha=0.5, xo=self.xo)
        qmm.quantize_mxfp4(self.xn, self.xq, T, H)
        (qmm.f32_gemv(self.router, self.xn, self.logits, E + 1, H, T) if few else qmm.gemm_f32(self.xn, self.router, self.logits, T, E + 1, H))
        qmm.moe_route_groups(self.logits, self.ids, self.p, T, E, K_TOP, bias=self.bias, **RULE)
        if few:
            def product(W, x, out, n, k, each):
                qmm.gemv_moe_mxfp4(W[:E], W[E], W.shape[1], self.ids, x, out, T, SLOTS, E, n, k, xrow_te=each)
        else:
            qmm.moe_sort(self.ids, T, SLOTS, E, 128, self.kpos, self.rowtok, self.tiles, self.counts)

            def product(W, x, out, n, k, each):
                qmm.moe_gemm_mxfp4(W[:E], W[E], W.shape[1], self.tiles, self.counts, self.cap, None if each else self.rowtok, x, out, n, k)
        product(self.Wg, self.xq, self.g, F, H, False)
        product(self.Wu, self.xq, self.u, F, H, False)
        qmm.silu_mul_bf16(self.g, self.u, self.h, TS * F)
        qmm.quantize_mxfp4(self.h, self.hq, TS, F)
        product(self.Wd, self.hq, self.d, H, F, True)
        qmm.moe_combine_sorted(self.d, self.p, self.straight if few else self.kpos, self.y, T, SLOTS, H)
        qmm.postnorm_add_rmsnorm_bf16(self.xo, self.y, None, self.w, self.xb2, T, H, EPS, gate=self.p[:, SLOTS - 1:], act="sigmoid", xo=self.xo2)

    def check(self):
        T, TS = self.T, self.T * SLOTS
        f = lambda t: host(t.float()).astype(np.float64)                 # noqa: E731
        xo, xn, bo, bn = mx_ref.postnorm(f(self.x), f(self.y0), f(self.wy), f(self.w), None, "none", 0.5, EPS)
        assert (np.abs(f(self.xo) - xo) <= bo).all() and (np.abs(f(self.xn) - xn) <= bn).all()
        code, byte = mx_ref.quantise(host(self.xn))
        assert np.array_equal(host(self.xq.q), mx_ref.pack(code)) and np.array_equal(host(self.xq.e), byte)
        # a logit: at most H roundings of the sum's magnitude, whatever its order
        a, r = f(self.xn), f(self.router)
        assert (np.abs(f(self.logits) - a @ r.T) <= H * 2.0 ** -24 * (np.abs(a) @ np.abs(r).T)).all()
        ids, p = mx_ref.route(host(self.logits), E, K_TOP, bias=host(self.bias), **RULE)
        assert np.array_equal(host(self.ids), ids) and (np.abs(f(self.p) - p) <= (2.0 ** -24 + 1e-13) * np.abs(p)).all()
        at = np.arange(TS) if T <= 16 else host(self.kpos)               # where slot te's row is
        a, flat = mx_ref.values(code, byte), ids.reshape(-1)
        G, U, Dn = f(self.g)[at], f(self.u)[at], f(self.d)[at]
        hc, hb = mx_ref.quantise(host(self.h.float()))
        assert np.array_equal(host(self.hq.q), mx_ref.pack(hc)) and np.array_equal(host(self.hq.e), hb)
        hv = mx_ref.values(hc, hb)[at]
        for e in range(-1, E):                                           # vals[-1]: the shared expert, the last
            s = np.nonzero(flat == e)[0]
            if len(s) == 0:
                continue
            for got, rows, v, k in ((G, a[s // SLOTS], self.vg[e], H), (U, a[s // SLOTS], self.vu[e], H), (Dn, hv[s], self.vd[e], F)):
                ref, bound = mx_ref.product_bound(rows, v, k)
                assert (np.abs(got[s] - ref) <= bound).all(), e
        # silu * up: the exponential is off by a rounding of its argument (|g| < 64 here) and a few of its own
        assert np.abs(G).max() < 64
        ref = G / (1 + np.exp(-G)) * U
        assert (np.abs(f(self.h)[at] - ref) <= (2.0 ** -8 + 80 * 2.0 ** -24) * np.abs(ref)).all()
        parts = f(self.p)[:, :, None] * Dn.reshape(T, SLOTS, H)
        assert (np.abs(f(self.y) - parts.sum(1)) <= (SLOTS + 1) * 2.0 ** -24 * np.abs(parts).sum(1)).all()
        xo, xn, bo, bn = mx_ref.postnorm(f(self.xo), f(self.y), None, f(self.w), f(self.p)[:, SLOTS - 1:], "sigmoid", 1.0, EPS)
        assert (np.abs(f(self.xo2) - xo) <= bo).all() and (np.abs(f(self.xb2) - xn) <= bn + 2.0 ** -8 * (np.abs(xn) + bn)).all()


@pytest.mark.parametrize("T", [1, 3, 16, 17, 210])
def test_expert_block(gpu, T):
    b = Block(T, T)
    b.feed(1)
    b.run()
    b.check()


@pytest.mark.parametrize("T", [2, 40])
def test_expert_block_replayed(gpu, T):
    """Captured on a stream of its own, replayed with new inputs between eager runs of another block."""
    b, other = Block(T, 7), Block(T, 8)
    b.feed(1)
    b.run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        b.run()
    torch.cuda.synchronize()
    for i in range(3):
        b.feed(10 + i)
        graph.replay()
        other.feed(20 + i)
        other.run()
        b.check()
        other.check()
        got = b.xb2.clone()
        b.run()
        assert torch.equal(got, b.xb2)


def test_two_blocks_at_once(gpu):
    """Two streams, the runs in flight together: nothing is shared between calls."""
    blocks = [(Block(T, 30 + T), torch.cuda.Stream()) for T in (60, 5)]
    for i, (b, s) in enumerate(blocks):
        b.feed(i)
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        for b, s in blocks:
            with torch.cuda.stream(s):
                b.run()
    torch.cuda.synchronize()
    for b, _ in blocks:
        b.check()


@pytest.mark.parametrize("T", [1, 40, 64, 65, 300])
def test_dense_block(gpu, T):
    """norm -> MXFP4 in one call, gate and up, silu, down, norm; the same codes from the two ways to them."""
    rng = np.random.default_rng(T)
    n, f = 384, 1090
    (Wg, vg), (Wu, vu), (Wd, vd) = packed(rng, 1, f, n), packed(rng, 1, f, n), packed(rng, 1, n, f)
    x, y = dev(rng.standard_normal((T, n)).astype(np.float32)), dev(rng.standard_normal((T, n)).astype(np.float32))
    w = dev((1 + 0.2 * rng.standard_normal(n)).astype(np.float32))
    product = qmm.gemv_mxfp4 if T <= 64 else qmm.gemm_mxfp4
    xq, hq, other = qmm.XMXBuf(T, n), qmm.XMXBuf(T, f), qmm.XMXBuf(T, n)
    xo, xn = torch.empty_like(x), torch.empty_like(x)
    qmm.postnorm_add_rmsnorm_mxfp4(x, y, w, w, xq, T, n, EPS, xo=xo)
    qmm.postnorm_add_rmsnorm_quant(x, y, w, w, xn, qmm.XQ8Buf(T, n), T, n, EPS, xo=torch.empty_like(x))
    qmm.quantize_mxfp4(xn, other, T, n)
    assert torch.equal(xq.q, other.q) and torch.equal(xq.e, other.e)
    g, u, d = torch.empty(T, f, device="cuda"), torch.empty(T, f, device="cuda"), torch.empty(T, n, device="cuda")
    h = torch.empty(T, f, dtype=torch.bfloat16, device="cuda")
    product(Wg, xq, g, T, f, n)
    product(Wu, xq, u, T, f, n)
    qmm.silu_mul_bf16(g, u, h, T * f)
    qmm.quantize_mxfp4(h, hq, T, f)
    product(Wd, hq, d, T, n, f)
    a = mx_ref.values(*mx_ref.quantise(host(xn)))
    hv = mx_ref.values(*mx_ref.quantise(host(h.float())))
    for got, rows, v, k in ((g, a, vg[0], n), (u, a, vu[0], n), (d, hv, vd[0], f)):
        ref, bound = mx_ref.product_bound(rows, v, k)
        assert (np.abs(host(got) - ref) <= bound).all()
    xb = torch.empty(T, n, dtype=torch.bfloat16, device="cuda")
    qmm.postnorm_add_rmsnorm_bf16(xo, d, w, w, xb, T, n, EPS)
    # in place: xo holds x + the two blocks' outputs, xb its norm
    first, _, b1, _ = mx_ref.postnorm(host(x), host(y), host(w), host(w), None, "none", 1.0, EPS)
    second, _, b2, _ = mx_ref.postnorm(first, host(d), host(w), host(w), None, "none", 1.0, EPS)
    assert (np.abs(host(xo) - second) <= b1 + b2).all()
    _, xn2, _, bn = mx_ref.postnorm(host(xo), np.zeros((T, n)), None, host(w), None, "none", 1.0, EPS)
    assert (np.abs(host(xb.float()) - xn2) <= bn + 2.0 ** -8 * (np.abs(xn2) + bn)).all()
