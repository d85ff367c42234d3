"""Calls of the MXFP4 block operators at the edges of what their header allows, against tests/mx_ref.py."""
import numpy as np
import pytest
import torch

import mx_ref
from hipster_amd import qmm
from hipster_amd._lib import QmmError
from tests.gpu_util import dev, host

pytestmark = pytest.mark.gpu

ROUTE_TOL = 2.0 ** -24 + 1e-13                                           # one rounding to f32, and float64 on both sides


def route(logits, E, k, bias=None, **kw):
    """moe_route_groups' ids and weights, held against the definition."""
    T, slots = logits.shape[0], k + (kw.get("shared") is not None)
    ids, w = torch.full((T, slots), -9, dtype=torch.int32, device="cuda"), torch.full((T, slots), -9.0, device="cuda")
    qmm.moe_route_groups(dev(logits), ids, w, T, E, k, bias=None if bias is None else dev(bias), **kw)
    ids, w = host(ids), host(w)
    rid, rw = mx_ref.route(logits, E, k, bias=bias, **kw)
    assert np.array_equal(ids, rid)
    assert np.array_equal(np.isnan(w), np.isnan(rw))
    ok = ~np.isnan(rw)
    assert (np.abs(w - rw)[ok] <= ROUTE_TOL * np.abs(rw[ok]) + 2.0 ** -150).all()
    return ids, w


@pytest.mark.parametrize("T", [1, 9])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_shared_gate_that_is_not_finite(gpu, score, T):
    """The shared expert's weight is the sigmoid of its logit, whatever that is; a row of NaN shows it."""
    big = np.finfo(np.float32).max
    for first in (np.nan, np.inf, -np.inf, big, -big, 0.0):
        l = np.random.default_rng(T).standard_normal((T, 65)).astype(np.float32)
        l[:, 64] = np.resize(np.array([first, np.nan, np.inf, -np.inf, big, -big, -0.0, 1e-40, -104.0], np.float32), T)
        with np.errstate(over="ignore"):
            route(l, 64, 6, score=score, shared="gate")
            route(l, 64, 6, score=score, shared="gate", groups=8, keep=3, best=2, scale=2.5)
            l[0] = np.nan
            ids, w = route(l, 64, 6, score=score, shared="gate")
        assert (ids[0] == -1).all() and (w[0, :6] == 0).all() and np.isnan(w[0, 6])


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_bias_that_masks(gpu, score):
    """A bias of -inf masks an expert as a logit of -inf does, also where too few experts are left."""
    rng = np.random.default_rng(1)
    l = rng.standard_normal((7, 64)).astype(np.float32)
    l[0, :60] = np.nan
    l[1, 4:] = -np.inf
    b = (rng.standard_normal(64) * 0.1).astype(np.float32)
    b[[0, 2, 61, 63]] = -np.inf, np.nan, -np.inf, np.inf
    ids, w = route(l, 64, 6, score=score, bias=b)
    assert not np.isin(ids, (0, 2, 61)).any() and (ids[0, 3:] == -1).all() and (ids[1, 2:] == -1).all() and (w[ids < 0] == 0).all()
    route(l, 64, 6, score=score, bias=b, groups=8, keep=2, best=2, shared="one")
    b[:] = -np.inf                                                       # every expert
    ids, w = route(l, 64, 6, score=score, bias=b, groups=8, keep=2, best=2)
    assert (ids == -1).all() and (w == 0).all()
    b[32:] = 0.0                                                         # groups without an expert lose
    ids, _ = route(l[2:], 64, 6, score=score, bias=b, groups=8, keep=4, best=2)
    assert (ids >= 32).all()


def packed(rng, n, N, K):
    """n weights packed one after another, and their values."""
    W, vals = torch.empty(n, qmm.mxfp4_weight_bytes(N, K), dtype=torch.uint8, device="cuda"), []
    for i in range(n):
        c, b = mx_ref.random_rows(rng, N, K)
        qmm.pack_mxfp4(dev(mx_ref.pack(c)), dev(b), W[i], N, K)
        vals.append(mx_ref.values(c, b))
    return W, vals


def rows_of(code, byte):
    b = qmm.XMXBuf(*code.shape)
    b.q.copy_(dev(mx_ref.pack(code)))
    b.e.copy_(dev(byte))
    return b


def test_sorted_experts_stay_inside_their_buffers(gpu):
    """Tiles and a table of another model: experts and rows beyond the last are the last, rows past the end of D stay."""
    rng = np.random.default_rng(2)
    E, N, K, TX, ROWS, ALL = 3, 72, 200, 5, 40, 64
    W, vals = packed(rng, E, N, K)
    ac, ab = mx_ref.random_rows(rng, TX, K)
    a = mx_ref.values(ac, ab)
    tab = rng.integers(-2, TX + 3, ALL).astype(np.int32)
    tab[[3, 9]] = 2 ** 31 - 1, -2 ** 31
    tiles = np.array([(0, 0, 10), (7, 10, 20), (1, 30, 10 ** 9), (2, ROWS, 8), (2 ** 31 - 1, 2 ** 31 - 1, 128), (0, -8, 4), (1, 2, -5)], np.int32)
    counts = dev(np.array([2 ** 30, 5], np.int32))                       # more tiles than there are
    D = torch.full((ALL, N), -7.0, device="cuda")
    qmm.moe_gemm_mxfp4(W, None, W.shape[1], dev(tiles), counts, len(tiles), dev(tab), rows_of(ac, ab), D, N, K, rows=ROWS)
    got = host(D)
    expert = np.repeat([0, E - 1, 1], [10, 20, ROWS - 30])
    ref, bound = np.empty((ROWS, N)), np.empty((ROWS, N))
    for r in range(ROWS):
        ref[r], bound[r] = (v[0] for v in mx_ref.product_bound(a[[min(max(tab[r], 0), TX - 1)]], vals[expert[r]], K))
    assert (np.abs(got[:ROWS] - ref) <= bound).all()
    assert (got[ROWS:] == -7).all()


def test_sorted_experts_refuse_short_buffers(gpu):
    W, _ = packed(np.random.default_rng(3), 2, 32, 128)
    tiles, counts, tab = (torch.zeros(s, dtype=torch.int32, device="cuda") for s in ((4, 3), 2, 12))
    x, D = qmm.XMXBuf(4, 128), torch.full((12, 32), -7.0, device="cuda")
    f = lambda D=D, tab=tab, **kw: qmm.moe_gemm_mxfp4(W, None, W.shape[1], tiles, counts, 4, tab, x, D, 32, 128, **kw)      # noqa: E731
    f()
    f(D=D[:11], rows=11)
    for bad in (lambda: f(D=D[:4]), lambda: f(D=D[:11]), lambda: f(tab=tab[:11], rows=12), lambda: f(nexperts=3), lambda: f(tab=None, rows=5)):
        with pytest.raises(QmmError):
            bad()
    assert (host(D) == -7).all()


def shifted(t, by):
    """t's values in rows that start `by` elements off an aligned address and lie an odd number of elements apart (2-d)."""
    if t.dim() == 1:
        out = torch.zeros(len(t) + 8, dtype=t.dtype, device="cuda")[by:by + len(t)]
    else:
        out = torch.zeros(t.shape[0], t.shape[1] + 9 - t.shape[1] % 2, dtype=t.dtype, device="cuda")[:, by:by + t.shape[1]]
    out.copy_(t)
    return out


@pytest.mark.parametrize("ydt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [4, 32, 640, 2880, 4100, 5120, 5632, 8192, 12288, 16384])
def test_norm_bits_do_not_depend_on_alignment(gpu, n, ydt):
    """A row has the same bits wherever its arrays lie, and whether it is one of many or alone."""
    g = torch.Generator().manual_seed(n)
    T, eps = 3, 1e-6
    x, y, gate = (torch.randn(T, n, generator=g).cuda() for _ in range(3))
    y, gate = y.to(ydt), gate.to(ydt)
    wy, w = ((1 + 0.2 * torch.randn(n, generator=g)).cuda() for _ in range(2))

    def run(x, y, wy, w, gate, off, rows=T):
        flat = lambda dt: torch.full((rows * n + 8,), 7.0, device="cuda").to(dt)     # noqa: E731
        xo, xb, xn = flat(torch.float32)[off:], flat(torch.bfloat16)[off:], flat(torch.float32)[off:]
        kw = dict(gate=gate, act="silu", xo=xo, alpha=0.5)
        qmm.postnorm_add_rmsnorm_bf16(x, y, wy, w, xb, rows, n, eps, **kw)
        out = [xo[:rows * n].clone(), xb[:rows * n]]
        m = qmm.XMXBuf(rows, n)
        if off:
            m.q = torch.zeros(m.q.numel() + 8, dtype=torch.uint8, device="cuda")[off:off + m.q.numel()].view(m.q.shape)
        qmm.postnorm_add_rmsnorm_mxfp4(x, y, wy, w, m, rows, n, eps, **kw)
        out += [xo[:rows * n].clone(), m.q, m.e]
        if n % 32 == 0:
            q8 = qmm.XQ8Buf(rows, n)
            if off:
                q8.q = torch.zeros(rows * n + 8, dtype=torch.int8, device="cuda")[off:off + rows * n].view(rows, n)
            qmm.postnorm_add_rmsnorm_quant(x, y, wy, w, xn, q8, rows, n, eps, **kw)
            out += [xo[:rows * n].clone(), xn[:rows * n], q8.q, q8.d, q8.s]
        assert (xo[rows * n:] == 7).all() and (xb[rows * n:] == 7).all() and (n % 32 or (xn[rows * n:] == 7).all())
        return [t.clone() for t in out]

    want = run(x, y, wy, w, gate, 0)
    xs = torch.zeros(T * n + 8, device="cuda")[1:1 + T * n].view(T, n).copy_(x)
    for got in (run(x, shifted(y, 0), wy, w, gate, 0), run(x, shifted(y, 3), wy, w, shifted(gate, 1), 0), run(xs, y, shifted(wy, 1), shifted(w, 2), gate, 0),
                run(x, y, wy, w, gate, 1), run(xs, shifted(y, 1), shifted(wy, 3), shifted(w, 3), shifted(gate, 5), 3)):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    one = run(x[2:], shifted(y, 3)[2:], wy, w, shifted(gate, 1)[2:], 0, rows=1)
    assert torch.equal(one[0], want[0][2 * n:]) and torch.equal(one[1], want[1][2 * n:]) and torch.equal(one[3][0], want[3][2])


@pytest.mark.parametrize("n", [1024, 1028, 2048, 2052, 3040, 3104, 4096, 4100, 5120, 5124, 6144, 6148, 8192, 8196, 12288, 12292, 16384])
def test_norm_widths_around_its_launches(gpu, n):
    """Both sides of every width at which the launch changes, all outputs."""
    g = torch.Generator().manual_seed(n)
    T, eps = 2, 1e-6
    x, y = torch.randn(T, n, generator=g).cuda() * 3, torch.randn(T, n, generator=g).cuda()
    wy, w = ((1 + 0.2 * torch.randn(n, generator=g)).cuda() for _ in range(2))
    xo, xn, bo, bn = mx_ref.postnorm(host(x), host(y), host(wy), host(w), None, "none", 1.0, eps)
    out, xb, m = torch.empty_like(x), torch.full((T + 1, n), 7.0, device="cuda").bfloat16(), qmm.XMXBuf(T, n)
    qmm.postnorm_add_rmsnorm_bf16(x, y, wy, w, xb, T, n, eps, xo=out)
    assert (np.abs(host(out) - xo) <= bo).all()
    assert (np.abs(host(xb[:T].float()) - xn) <= bn + 2.0 ** -8 * (np.abs(xn) + bn)).all() and (xb[T] == 7).all()
    out2 = torch.empty_like(x)
    qmm.postnorm_add_rmsnorm_mxfp4(x, y, wy, w, m, T, n, eps, xo=out2)
    assert torch.equal(out2, out)
    if n % 32 == 0:
        f, q8, mq = torch.empty_like(x), qmm.XQ8Buf(T, n), qmm.XMXBuf(T, n)
        qmm.postnorm_add_rmsnorm_quant(x, y, wy, w, f, q8, T, n, eps, xo=out2)
        assert torch.equal(out2, out) and (np.abs(host(f) - xn) <= bn).all() and torch.equal(f.bfloat16(), xb[:T])
        qmm.quantize_mxfp4(f, mq, T, n)
        assert torch.equal(mq.q, m.q) and torch.equal(mq.e, m.e)


def test_no_rows(gpu):
    """A batch without tokens: every call takes its empty tensors."""
    T, E, k, n = 0, 8, 2, 64
    e = lambda *s, dt=torch.float32: torch.empty(s, dtype=dt, device="cuda")         # noqa: E731
    (W, _), x, xq, w = packed(np.random.default_rng(5), E, 32, n), e(T, n), qmm.XMXBuf(T, n), torch.ones(n, device="cuda")
    ids, tiles, counts = e(T, k, dt=torch.int32), torch.zeros(E + 2, 3, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    qmm.quantize_mxfp4(x, xq, T, n)
    qmm.dequant_mxfp4(xq, x, T, n)
    qmm.gemv_mxfp4(W[0], xq, e(T, 32), T, 32, n)
    qmm.gemm_mxfp4(W[0], xq, e(T, 32), T, 32, n)
    qmm.moe_route_groups(e(T, E), ids, e(T, k), T, E, k)
    qmm.gemv_moe_mxfp4(W, None, W.shape[1], ids, xq, e(T * k, 32), T, k, E, 32, n)
    qmm.moe_gemm_mxfp4(W, None, W.shape[1], tiles, counts, E + 2, e(T * k, dt=torch.int32), xq, e(T * k, 32), 32, n)
    qmm.postnorm_add_rmsnorm_bf16(x, e(T, n), w, w, e(T, n, dt=torch.bfloat16), T, n, 1e-6)
    qmm.postnorm_add_rmsnorm_quant(x, e(T, n), w, w, e(T, n), qmm.XQ8Buf(T, n), T, n, 1e-6)
    qmm.postnorm_add_rmsnorm_mxfp4(x, e(T, n), w, w, xq, T, n, 1e-6, gate=e(T, n), act="silu")
    with pytest.raises(QmmError):
        qmm.quantize_mxfp4(x, xq, 1, n)
