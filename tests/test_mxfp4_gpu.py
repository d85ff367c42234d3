"""The MXFP4 quantiser, packing and products on the GPU against tests/mx_ref.py (float64, from the definitions)."""
import numpy as np
import pytest
import torch

import mx_ref
from hipster_amd import qmm
from hipster_amd._lib import QmmError
from tests.gpu_util import dev, host

pytestmark = pytest.mark.gpu

T = {"f32": torch.float32, "bf16": torch.bfloat16}


def xmx(code, byte):
    """XMXBuf of numpy codes and scale bytes."""
    b = qmm.XMXBuf(code.shape[0], code.shape[1])
    b.q.copy_(dev(mx_ref.pack(code)))
    b.e.copy_(dev(byte))
    return b


def packed(code, byte, N, K):
    b = xmx(code, byte)
    W = torch.full((qmm.mxfp4_weight_bytes(N, K),), 0xEE, dtype=torch.uint8, device="cuda")
    qmm.pack_mxfp4(b.q, b.e, W, N, K)
    return W


def check_quantised(x, K, buf):
    code, byte = mx_ref.quantise(host(x.float()))
    assert np.array_equal(host(buf.e), byte)
    assert np.array_equal(host(buf.q), mx_ref.pack(code))
    return code, byte


# ---------------------------------------------------------------- quantisation
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("R,K", [(1, 1), (1, 32), (3, 33), (2, 127), (5, 128), (7, 1000), (16, 2880), (33, 4100), (300, 264)])
def test_quantise(gpu, R, K, dtype):
    g = torch.Generator().manual_seed(R * 10007 + K)
    x = (torch.randn(R, K, generator=g) * torch.exp2(torch.randint(-20, 20, (R, 1), generator=g).float())).to(T[dtype]).cuda()
    b = qmm.XMXBuf(R + 1, K)
    b.q.fill_(0x5A); b.e.fill_(0x5A)
    qmm.quantize_mxfp4(x, b, R, K)
    assert (host(b.q)[R] == 0x5A).all() and (host(b.e)[R] == 0x5A).all()         # the row behind the last
    b.q, b.e = b.q[:R], b.e[:R]
    code, byte = check_quantised(x, K, b)
    for out in ("f32", "bf16"):
        v = torch.full((R * K + 5,), -7.0, dtype=T[out], device="cuda")
        b.rows = R
        qmm.dequant_mxfp4(b, v, R, K)
        assert np.array_equal(host(v[:R * K].float()).reshape(R, K), mx_ref.values(code, byte)[:, :K])
        assert (host(v[R * K:].float()) == -7).all()


def test_quantise_borders_and_extremes(gpu):
    """Every tie of the grid at every scale, subnormals, the largest numbers, zeros of both signs."""
    ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 7.99])
    near = np.concatenate([ties, np.nextafter(np.float32(ties), np.float32(0)), np.nextafter(np.float32(ties), np.float32(8))])
    row = np.concatenate([near, -near[:4], [4.0]]).astype(np.float32)[:32]
    row[0] = 4.5                                                         # every block's largest lies in [4, 8)
    rows = [row * np.float32(2.0 ** e) for e in (-120, -60, -1, 0, 1, 60, 120)]
    rows += [np.full(32, s * v, np.float32) for v in (1e-45, 1e-40, 2.0 ** -126, 2.0 ** -125, 3.4028235e38, 2.0 ** -124) for s in (1, -1)]
    rows += [np.zeros(32, np.float32), np.full(32, -0.0, np.float32)]
    mixed = np.zeros(32, np.float32); mixed[5] = 1e-44; mixed[7] = -3e-45
    rows.append(mixed)
    x = dev(np.stack(rows))
    b = qmm.XMXBuf(len(rows), 32)
    qmm.quantize_mxfp4(x, b, len(rows), 32)
    check_quantised(x, 32, b)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_quantise_not_finite(gpu, dtype, bad):
    """The block that holds it becomes NaN, its neighbours stay."""
    x = torch.randn(3, 200).to(T[dtype])
    x[1, 70] = bad
    b = qmm.XMXBuf(3, 200)
    qmm.quantize_mxfp4(x.cuda(), b, 3, 200)
    v = torch.empty(3, 200, device="cuda")
    qmm.dequant_mxfp4(b, v, 3, 200)
    nan = np.isnan(host(v))
    want = np.zeros((3, 200), bool); want[1, 64:96] = True
    assert np.array_equal(nan, want)
    check_quantised(x, 200, b)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_quantise_strided_and_unaligned_rows(gpu, dtype):
    full = torch.randn(9, 515).to(T[dtype]).cuda()
    for x, K in ((full[:, :256], 256), (full[:, 3:103], 100), (full[::2, 8:72], 64), (full.flatten()[1:1 + 4 * 384].view(4, 384), 384)):
        R = x.shape[0]
        b = qmm.XMXBuf(R, K)
        qmm.quantize_mxfp4(x, b, R, K)
        check_quantised(x, K, b)
    with pytest.raises(QmmError):
        qmm.quantize_mxfp4(full.t(), qmm.XMXBuf(515, 9), 515, 9)
    with pytest.raises(QmmError):
        qmm.quantize_mxfp4(full.half(), qmm.XMXBuf(9, 515), 9, 515)
    with pytest.raises(QmmError):
        qmm.quantize_mxfp4(full, qmm.XMXBuf(8, 515), 9, 515)


def test_quantise_rows_far_apart(gpu):
    """A row beyond 2^32 bytes of its matrix."""
    far = torch.empty((1 << 32) + 4096, dtype=torch.uint8, device="cuda").view(torch.bfloat16)
    ld = (1 << 31) + 64
    x = torch.as_strided(far, (2, 64), (ld, 1))
    x.copy_(torch.randn(2, 64))
    b = qmm.XMXBuf(2, 64)
    qmm.quantize_mxfp4(x, b, 2, 64)
    check_quantised(x, 64, b)


# ---------------------------------------------------------------- packing
@pytest.mark.parametrize("N,K", [(1, 32), (16, 128), (17, 130), (40, 512), (33, 1600)])
def test_pack(gpu, N, K):
    rng = np.random.default_rng(N + K)
    code, byte = mx_ref.random_rows(rng, N, K)
    W = host(packed(code, byte, N, K))
    k128, groups = mx_ref.steps(K), -(-mx_ref.steps(K) // 4)
    q, e = mx_ref.pack(code).reshape(N, k128, 4, 16), byte.reshape(N, k128, 4)
    W = W.reshape(-1, k128 * 1024 + groups * 256)
    for s in range(W.shape[0]):
        codes = W[s, :k128 * 1024].reshape(k128, 64, 16)
        scales = W[s, k128 * 1024:].reshape(groups, 64, 4)
        for lane in range(64):
            r, blk = 16 * s + lane % 16, lane // 16
            assert np.array_equal(codes[:, lane], q[r, :, blk] if r < N else np.zeros((k128, 16)))
            want = np.zeros(groups * 4, np.uint8)
            if r < N:
                want[:k128] = e[r, :, blk]
            assert np.array_equal(scales[:, lane].reshape(-1), want)


# ---------------------------------------------------------------- dense products
def run_dense(f, W, x, M, N, K, out, pad=3):
    y = torch.full((M + pad, N), -7.0, dtype=T[out], device="cuda")
    f(W, x, y, M, N, K)
    assert (host(y[M:].float()) == -7).all()                             # rows behind the last
    return y[:M]


def check_dense(y, a, w, K, out):
    ref, bound = mx_ref.product_bound(a, w, K)
    if out == "bf16":
        bound = bound + 2.0 ** -8 * (np.abs(ref) + bound)
    err = np.abs(host(y.float()).astype(np.float64) - ref)
    assert (err <= bound).all(), float((err / np.maximum(bound, 1e-300)).max())


GEMV = [(1, 1, 32), (1, 16, 128), (2, 17, 130), (3, 100, 640), (16, 64, 512), (17, 48, 1100), (32, 33, 4224), (33, 80, 1024), (64, 250, 2050),
        (1, 40, 17408), (5, 1000, 5120), (48, 7, 8200), (64, 16, 300)]


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("M,N,K", GEMV)
def test_gemv(gpu, M, N, K, out):
    rng = np.random.default_rng(M * 31 + N * 7 + K)
    (ac, ab), (wc, wb) = mx_ref.random_rows(rng, M, K), mx_ref.random_rows(rng, N, K)
    W, x = packed(wc, wb, N, K), xmx(ac, ab)
    y = run_dense(qmm.gemv_mxfp4, W, x, M, N, K, out)
    check_dense(y, mx_ref.values(ac, ab), mx_ref.values(wc, wb), K, out)


GEMM = [(1, 1, 32), (2, 17, 130), (16, 100, 640), (65, 64, 512), (128, 256, 128), (129, 257, 1100), (200, 1000, 384), (300, 515, 2050), (1000, 130, 260),
        (2100, 520, 136), (2049, 2050, 70), (700, 12300, 513), (4100, 8200, 200), (70, 16, 9000)]


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("M,N,K", GEMM)
def test_gemm(gpu, M, N, K, out):
    rng = np.random.default_rng(M * 31 + N * 7 + K)
    (ac, ab), (wc, wb) = mx_ref.random_rows(rng, M, K), mx_ref.random_rows(rng, N, K)
    W, x = packed(wc, wb, N, K), xmx(ac, ab)
    y = run_dense(qmm.gemm_mxfp4, W, x, M, N, K, out)
    check_dense(y, mx_ref.values(ac, ab), mx_ref.values(wc, wb), K, out)


def test_wide_scales(gpu):
    """Blocks 2^80 apart: every product is exact, so the f32 bound holds whatever the scales."""
    rng = np.random.default_rng(5)
    K = 640
    (ac, ab), (wc, wb) = mx_ref.random_rows(rng, 20, K, spread=40), mx_ref.random_rows(rng, 40, K, spread=40)
    W, x = packed(wc, wb, 40, K), xmx(ac, ab)
    for f in (qmm.gemv_mxfp4, qmm.gemm_mxfp4):
        check_dense(run_dense(f, W, x, 20, 40, K, "f32"), mx_ref.values(ac, ab), mx_ref.values(wc, wb), K, "f32")


def test_nan_block_reaches_its_row_only(gpu):
    rng = np.random.default_rng(6)
    (ac, ab), (wc, wb) = mx_ref.random_rows(rng, 70, 300), mx_ref.random_rows(rng, 40, 300)
    ab[3, 2] = 255
    wb[21, 9] = 255
    for f, M in ((qmm.gemv_mxfp4, 20), (qmm.gemm_mxfp4, 70)):
        y = host(run_dense(f, packed(wc, wb, 40, 300), xmx(ac, ab), M, 40, 300, "f32"))
        want = np.zeros((M, 40), bool); want[3] = True; want[:, 21] = True
        assert np.array_equal(np.isnan(y), want)


def test_bits_do_not_depend_on_the_call(gpu):
    """A row alone, among others, in every tile the GEMM takes, and against a joined weight: the same bits."""
    rng = np.random.default_rng(7)
    K, N = 1700, 2064
    (ac, ab), (wc, wb) = mx_ref.random_rows(rng, 1100, K), mx_ref.random_rows(rng, N, K)
    W, x = packed(wc, wb, N, K), xmx(ac, ab)
    W2 = torch.cat([W, packed(wc[:48], wb[:48], 48, K)])
    bits = lambda t: host(t).view(np.uint32)                             # noqa: E731
    v64 = bits(run_dense(qmm.gemv_mxfp4, W, x, 64, N, K, "f32"))
    for M in (1, 2, 15, 16, 17, 31, 33, 50):
        assert np.array_equal(bits(run_dense(qmm.gemv_mxfp4, W, x, M, N, K, "f32")), v64[:M])
    assert np.array_equal(bits(run_dense(qmm.gemv_mxfp4, W2, x, 9, N + 48, K, "f32"))[:, :N], v64[:9])
    m = bits(run_dense(qmm.gemm_mxfp4, W, x, 1100, N, K, "f32"))
    for M in (1, 16, 64, 65, 129, 300, 640, 1000):
        assert np.array_equal(bits(run_dense(qmm.gemm_mxfp4, W, x, M, N, K, "f32")), m[:M])
    assert np.array_equal(bits(run_dense(qmm.gemm_mxfp4, W2, x, 700, N + 48, K, "f32"))[:, :N], m[:700])


# shapes whose choice is each tile, with steps of 128 that end everywhere in a group of four and a pair
TILES = [(0, 6000, 20000, 130), (0, 4000, 12300, 260), (0, 2000, 16400, 400), (0, 2000, 8200, 513), (0, 577, 20000, 900), (0, 577, 20000, 1025),
         (0, 577, 20000, 1160), (0, 577, 16400, 2050), (1, 3000, 20000, 400), (1, 3000, 20000, 640), (1, 500, 16400, 900), (1, 385, 20000, 1025),
         (1, 385, 20000, 1160), (1, 769, 10000, 2050), (2, 6000, 12300, 400), (2, 6000, 12300, 513), (2, 6000, 6200, 900), (2, 577, 10000, 1160),
         (2, 700, 8200, 2050), (3, 769, 10000, 260), (3, 769, 5000, 400), (3, 200, 16400, 640), (3, 200, 8200, 1025), (4, 200, 1000, 32),
         (4, 200, 8200, 513), (4, 200, 12300, 1160), (5, 385, 4100, 300), (5, 200, 5000, 900), (5, 200, 5000, 2050), (6, 200, 1000, 513),
         (6, 200, 1000, 1025), (6, 200, 1000, 2180), (7, 769, 5000, 2050), (7, 961, 4900, 2180), (7, 1000, 4100, 2400), (7, 1153, 4100, 2433)]


@pytest.mark.parametrize("tile,M,N,K", TILES)
def test_gemm_every_tile(gpu, tile, M, N, K):
    """Each tile against float64 (on the GPU: the sizes that choose the large ones), odd ends of M, N and K; and its bits
    against those of calls of few rows, which run small tiles."""
    assert qmm.gemm_mxfp4_tile(M, N, K) == tile
    rng = np.random.default_rng(tile + K)
    (ac, ab), (wc, wb) = mx_ref.random_rows(rng, M, K), mx_ref.random_rows(rng, N, K)
    W, x = packed(wc, wb, N, K), xmx(ac, ab)
    y = run_dense(qmm.gemm_mxfp4, W, x, M, N, K, "f32")
    a, w = dev(mx_ref.values(ac, ab)), dev(mx_ref.values(wc, wb))
    err = (y.double() - a @ w.t()).abs_()
    bound = (a.abs() @ w.abs().t()) * ((mx_ref.steps(K) + 8) * 2.0 ** -23)
    assert bool((err <= bound).all()), float((err / bound).max())
    del err, bound
    for r in (0, M // 2, M - 40):
        part = run_dense(qmm.gemm_mxfp4, W, xmx(ac[r:r + 40], ab[r:r + 40]), 40, N, K, "f32")
        assert torch.equal(part, y[r:r + 40])
    low = run_dense(qmm.gemm_mxfp4, W, x, M, N, K, "bf16")
    assert torch.equal(low, y.bfloat16())


def test_output_beyond_32_bits(gpu):
    """M x N beyond 2^32 elements: the last rows are right."""
    rng = np.random.default_rng(8)
    M, N, K = 65600, 65552, 96
    (ac, ab), (wc, wb) = mx_ref.random_rows(rng, 64, K), mx_ref.random_rows(rng, 64, K)
    x = xmx(np.tile(ac, (M // 64, 1)), np.tile(ab, (M // 64, 1)))
    rep = -(-N // 64)
    W = packed(np.tile(wc, (rep, 1))[:N], np.tile(wb, (rep, 1))[:N], N, K)
    y = torch.empty((M, N), dtype=torch.bfloat16, device="cuda")
    qmm.gemm_mxfp4(W, x, y, M, N, K)
    ref, bound = mx_ref.product_bound(mx_ref.values(ac, ab), mx_ref.values(wc, wb), K)
    for r0, c0 in ((0, 0), (M // 128 * 64, N // 128 * 64), (M - 64, N - 16 - 64)):
        got = host(y[r0:r0 + 64, c0:c0 + 64].float()).astype(np.float64)
        cols = (c0 + np.arange(64)) % 64
        assert (np.abs(got - ref[:, cols]) <= bound[:, cols] + 2.0 ** -8 * (np.abs(ref[:, cols]) + bound[:, cols])).all(), (r0, c0)


def test_streams_and_graph(gpu):
    """Quantise and multiply on a side stream; captured once, replayed on changing inputs with eager work between."""
    rng = np.random.default_rng(9)
    K, N, M = 520, 96, 90
    wc, wb = mx_ref.random_rows(rng, N, K)
    W, w64 = packed(wc, wb, N, K), mx_ref.values(wc, wb)
    x, b = torch.zeros(M, K, device="cuda"), qmm.XMXBuf(M, K)
    y, v = torch.zeros(M, N, device="cuda"), torch.zeros(32, N, device="cuda")

    def work():
        qmm.quantize_mxfp4(x, b, M, K)
        qmm.gemm_mxfp4(W, b, y, M, N, K)
        qmm.gemv_mxfp4(W, b, v, 32, N, K)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        work()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        work()
    for i in range(4):
        xi = rng.standard_normal((M, K)).astype(np.float32) * (i + 1)
        x.copy_(torch.from_numpy(xi))
        y.fill_(-1); v.fill_(-1)
        graph.replay()
        torch.cuda.synchronize()
        a = mx_ref.values(*mx_ref.quantise(xi))
        check_dense(y, a, w64, K, "f32")
        check_dense(v, a[:32], w64, K, "f32")
        work()                                                           # eager work between replays
        check_dense(y, a, w64, K, "f32")


# ---------------------------------------------------------------- experts
def experts(rng, E, N, K, shared=True):
    """Packed weights of E experts and a shared one, and their float64 values."""
    Ws, vals = [], []
    for _ in range(E + shared):
        c, b = mx_ref.random_rows(rng, N, K)
        Ws.append(packed(c, b, N, K))
        vals.append(mx_ref.values(c, b))
    return torch.stack(Ws[:E]), Ws[E] if shared else None, vals


def dense_rows(W, Wsh, ids, te, E):
    e = min(max(int(ids), -1 if Wsh is not None else 0), E - 1)
    return Wsh if e < 0 else W[e]


@pytest.mark.parametrize("xrow_te", [False, True])
@pytest.mark.parametrize("T,slots,E,N,K", [(1, 1, 1, 16, 128), (1, 11, 64, 40, 640), (4, 9, 16, 72, 2048), (16, 16, 8, 33, 260), (16, 3, 40, 64, 5000)])
def test_gemv_moe(gpu, T, slots, E, N, K, xrow_te):
    rng = np.random.default_rng(T + slots + E + K)
    W, Wsh, _ = experts(rng, E, N, K)
    ids = np.full((T, slots), -1, np.int32)
    for t in range(T):
        ids[t, :min(slots, E)] = rng.permutation(E)[:slots]
    ids[:, -1] = -1 if slots > 1 else ids[:, -1]
    ac, ab = mx_ref.random_rows(rng, T * slots if xrow_te else T, K)
    x, eb = xmx(ac, ab), W.shape[1]
    y = torch.full((T * slots + 2, N), -7.0, device="cuda")
    qmm.gemv_moe_mxfp4(W, Wsh, eb, dev(ids), x, y, T, slots, E, N, K, xrow_te=xrow_te)
    assert (host(y[T * slots:]) == -7).all()
    for te in range(T * slots):                                          # the bits of the dense GEMV of its expert
        row = te if xrow_te else te // slots
        one = torch.empty(1, N, device="cuda")
        qmm.gemv_mxfp4(dense_rows(W, Wsh, ids.flat[te], te, E), xmx(ac[row:row + 1], ab[row:row + 1]), one, 1, N, K)
        assert np.array_equal(host(y[te]).view(np.uint32), host(one[0]).view(np.uint32)), te


def test_gemv_moe_odd_ids(gpu):
    """The same expert in every slot of 16 tokens (256 columns), ids beyond the range, and no shared expert."""
    rng = np.random.default_rng(3)
    T, slots, E, N, K = 16, 16, 5, 40, 300
    W, Wsh, _ = experts(rng, E, N, K)
    ac, ab = mx_ref.random_rows(rng, T, K)
    x = xmx(ac, ab)
    for ids, sh in ((np.full((T, slots), 2), Wsh), (rng.integers(-3, E + 4, (T, slots)), Wsh), (rng.integers(-3, E + 4, (T, slots)), None)):
        y = torch.full((T * slots, N), -7.0, dtype=torch.bfloat16, device="cuda")
        qmm.gemv_moe_mxfp4(W, sh, W.shape[1], dev(ids.astype(np.int32)), x, y, T, slots, E, N, K)
        want = torch.empty(T, N, dtype=torch.bfloat16, device="cuda")
        for e in range(-1, E):
            at = np.nonzero(np.clip(ids, -1 if sh is not None else 0, E - 1) == e)
            if e < 0 and sh is None or len(at[0]) == 0:
                continue
            qmm.gemv_mxfp4(sh if e < 0 else W[e], x, want, T, N, K)
            got = host(y.view(T, slots, N).float())[at]
            assert np.array_equal(got, host(want.float())[at[0]]), e


def sorted_rows(ids, E, cap_rows=128):
    T, slots = ids.shape
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")    # noqa: E731
    cap = qmm.moe_tiles_capacity(T, slots, E, cap_rows)
    kpos, rowtok, tiles, counts = i32(T * slots), i32(T * slots), i32(cap, 3), i32(2)
    qmm.moe_sort(dev(ids), T, slots, E, cap_rows, kpos, rowtok, tiles, counts)
    return kpos, rowtok, tiles, counts, cap


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("T,slots,E,N,K,cap_rows", [(1, 2, 4, 16, 128, 128), (40, 5, 7, 130, 300, 128), (150, 3, 2, 257, 640, 128), (64, 4, 100, 64, 1100, 128),
                                                    (90, 4, 3, 48, 520, 17), (500, 2, 3, 140, 256, 128), (75, 2, 1, 200, 1300, 128),
                                                    (97, 2, 1, 64, 384, 128)])
def test_moe_gemm(gpu, T, slots, E, N, K, cap_rows, out):
    rng = np.random.default_rng(T + E + K)
    W, Wsh, vals = experts(rng, E, N, K)
    ids = rng.integers(0, E, (T, slots)).astype(np.int32)
    ids[:, -1] = -1
    kpos, rowtok, tiles, counts, cap = sorted_rows(ids, E, cap_rows)
    ac, ab = mx_ref.random_rows(rng, T, K)
    x = xmx(ac, ab)
    D = torch.full((T * slots + 2, N), -7.0, dtype=T_(out), device="cuda")
    qmm.moe_gemm_mxfp4(W, Wsh, W.shape[1], tiles, counts, cap, rowtok, x, D, N, K)
    assert (host(D[T * slots:].float()) == -7).all()
    k, tok = host(kpos), np.arange(T * slots) // slots
    a = mx_ref.values(ac, ab)
    got = host(D.float()).astype(np.float64)
    dense = torch.empty(T, N, dtype=T_(out), device="cuda")
    for e in range(-1, E):
        at = np.nonzero(ids.reshape(-1) == e)[0]
        if len(at) == 0:
            continue
        ref, bound = mx_ref.product_bound(a[tok[at]], vals[e], K)
        if out == "bf16":
            bound = bound + 2.0 ** -8 * (np.abs(ref) + bound)
        assert (np.abs(got[k[at]] - ref) <= bound).all(), e
        qmm.gemm_mxfp4(Wsh if e < 0 else W[e], x, dense, T, N, K)        # the bits of the dense product
        assert np.array_equal(got[k[at]], host(dense.float())[tok[at]].astype(np.float64)), e
    # sorted rows as they are (no table): the second product of an MoE block
    c2, b2 = mx_ref.random_rows(rng, T * slots, K)
    qmm.moe_gemm_mxfp4(W, Wsh, W.shape[1], tiles, counts, cap, None, xmx(c2, b2), D, N, K)
    ref, bound = mx_ref.product_bound(mx_ref.values(c2, b2)[k[:slots]][:1], vals[ids[0, 0]], K)
    bound = bound + (2.0 ** -8 * (np.abs(ref) + bound) if out == "bf16" else 0)
    assert (np.abs(host(D.float())[k[0]] - ref[0]) <= bound[0]).all()


def T_(name):
    return T[name]


def test_moe_no_rows_and_far_experts(gpu):
    """Counts of zero leave the output; an expert beyond 2^32 bytes of the first is read where it is."""
    rng = np.random.default_rng(4)
    N, K, E = 48, 256, 2
    one = qmm.mxfp4_weight_bytes(N, K)
    eb = (1 << 32) + 4096
    W = torch.empty(eb + one, dtype=torch.uint8, device="cuda")
    vals = []
    for e in range(E):
        c, b = mx_ref.random_rows(rng, N, K)
        W[e * eb:e * eb + one] = packed(c, b, N, K)
        vals.append(mx_ref.values(c, b))
    ac, ab = mx_ref.random_rows(rng, 6, K)
    x, a = xmx(ac, ab), mx_ref.values(ac, ab)
    ids = np.array([[0], [1], [1], [0], [1], [1]], np.int32)
    y = torch.full((6, N), -7.0, device="cuda")
    qmm.gemv_moe_mxfp4(W, None, eb, dev(ids), x, y, 6, 1, E, N, K)
    kpos, rowtok, tiles, counts, cap = sorted_rows(ids, E)
    D = torch.full((6, N), -7.0, device="cuda")
    qmm.moe_gemm_mxfp4(W, None, eb, tiles, torch.zeros_like(counts), cap, rowtok, x, D, N, K)
    assert (host(D) == -7).all()
    qmm.moe_gemm_mxfp4(W, None, eb, tiles, counts, cap, rowtok, x, D, N, K)
    for t in range(6):
        ref, bound = mx_ref.product_bound(a[t:t + 1], vals[ids[t, 0]], K)
        assert (np.abs(host(y)[t] - ref[0]) <= bound[0]).all() and (np.abs(host(D)[host(kpos)[t]] - ref[0]) <= bound[0]).all()


def test_refusals_seen_from_python(gpu):
    x, W = qmm.XMXBuf(4, 256), torch.zeros(qmm.mxfp4_weight_bytes(32, 256), dtype=torch.uint8, device="cuda")
    y = torch.zeros(4, 32, device="cuda")
    for bad in (lambda: qmm.gemv_mxfp4(W[:-16], x, y, 4, 32, 256), lambda: qmm.gemv_mxfp4(W, x, y, 5, 32, 256), lambda: qmm.gemv_mxfp4(W, x, y.half(), 4, 32, 256),
                lambda: qmm.gemm_mxfp4(W, x, y[:3], 4, 32, 256), lambda: qmm.gemm_mxfp4(W, x, y, 4, 32, 512), lambda: qmm.gemm_mxfp4(W, x, y.t(), 4, 32, 256),
                lambda: qmm.pack_mxfp4(x.q, x.e, W, 5, 256), lambda: qmm.dequant_mxfp4(x, y, 4, 256)):
        with pytest.raises(QmmError):
            bad()
