"""Rotary positions, the MXFP4 cache, attention over it and attention of prompts on the GPU, against the definitions in float64."""
import numpy as np
import pytest
import torch

import attn_ref
from hipster_amd import qmm
from hipster_amd._lib import QmmError

pytestmark = pytest.mark.gpu
T = {"f32": torch.float32, "bf16": torch.bfloat16}


def host(t):
    return t.detach().float().cpu().numpy()


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def offsets(n):
    return [0] + list(np.cumsum(n))


def rows(g, n, heads, D, dtype):
    x = torch.randn((n, heads, D), generator=g)
    x[:, :, torch.randint(0, D, (max(1, D // 32),), generator=g)] *= 3.0
    return x.to(T[dtype]).cuda()


# ---------------------------------------------------------------- rotary positions
def run_rope(Tn, H, D, P, style, axes, dtype, out, far, scale=1.0, pad=0, inplace=False, one=False):
    g = torch.Generator().manual_seed(Tn * 1000 + H + D + P)
    full = torch.randn((Tn, H * D + pad), generator=g).to(T[dtype]).cuda()
    x = full[:, :H * D]
    freq = (torch.rand(P, generator=g) * 2 - 1).float()
    if P:
        freq[0] = 1.0
    axis = None if one else torch.randint(0, axes, (P,), generator=g).to(torch.uint8)
    pos = torch.randint(-far, far + 1, (axes, Tn), generator=g).int()
    want, bound = attn_ref.rope(host(x).reshape(Tn, H, D), pos.numpy(), freq.numpy(), None if one else axis.long().numpy(), style, scale)
    y = x if inplace else torch.full((Tn, H * D), 7.0, dtype=T[out], device="cuda")
    rest = full[:, H * D:].clone()
    qmm.rope_axes(x, y, pos.cuda() if axes > 1 else pos[0].cuda(), freq.cuda(), None if one else axis.cuda(), Tn, H, D, style=style, scale=scale)
    got = host(y).reshape(Tn, H, D)
    bound = bound + attn_ref.HALF[out] * np.abs(want)
    bound[:, :, 2 * P:] = attn_ref.HALF[out] * np.abs(want[:, :, 2 * P:]) if T[dtype] != T[out] else 0
    assert (np.abs(got - want) <= bound).all(), np.abs(got - want).max()
    assert torch.equal(full[:, H * D:], rest)


@pytest.mark.parametrize("style", ["halves", "neighbours"])
@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("Tn,H,D,P", [(1, 40, 128, 64), (5, 3, 64, 32), (300, 7, 128, 16), (33, 2, 256, 32), (7, 1, 80, 37), (4, 2, 33, 16), (9, 3, 8, 0)])
def test_rope(gpu, style, dtype, out, Tn, H, D, P):
    run_rope(Tn, H, D, P, style, 3, dtype, out, 50000)


def test_rope_far_positions(gpu):
    """The angle of a far position is as good as a near one's."""
    run_rope(50, 2, 128, 64, "halves", 3, "f32", "f32", (1 << 31) - 2)


def test_rope_many_tokens(gpu):
    run_rope(2100, 33, 128, 64, "halves", 2, "bf16", "bf16", 5000)


@pytest.mark.parametrize("style", ["halves", "neighbours"])
def test_rope_in_place_strided_one_axis(gpu, style):
    run_rope(70, 5, 128, 64, style, 1, "bf16", "bf16", 900, scale=1.25, pad=72, inplace=True, one=True)
    run_rope(70, 5, 64, 20, style, 3, "f32", "f32", 900, scale=0.5, pad=3, inplace=True)


def test_rope_axis_number_out_of_range(gpu):
    """Numbers of axes lie on the device: one past the last is the last."""
    x, y = torch.randn(3, 64, device="cuda"), torch.empty(2, 3, 64, device="cuda")
    pos, freq = ints([[1, 2, 3], [4, 5, 6]]), torch.rand(32, device="cuda")
    for i, a in enumerate((1, 250)):
        qmm.rope_axes(x, y[i], pos, freq, torch.full((32,), a, dtype=torch.uint8, device="cuda"), 3, 1, 64)
    assert torch.equal(y[0], y[1])


# ---------------------------------------------------------------- the cache
def cache(g, lens, Hk, D, page, spare=3, ld=None):
    """An empty cache with pages in any order: (kv, table)."""
    need = [-(-n // page) for n in lens]
    kv = qmm.KVMXBuf(sum(need) + spare, page, Hk, D)
    for t in (kv.kq, kv.ke, kv.vq, kv.ve):
        t.copy_(torch.randint(0, 255, t.shape, generator=g))                   # what is not written holds anything, NaN scales too
    kv.ke[:, :, ::3] = 255
    kv.ve[:, :, ::3] = 255
    order = torch.randperm(kv.pages, generator=g).int()
    table = torch.full((len(lens), max(max(need), 1) if ld is None else ld), -7, dtype=torch.int32)
    at = offsets(need)
    for b, n in enumerate(need):
        table[b, :n] = order[at[b]:at[b] + n]
    return kv, table.cuda()


def places(table, lens, ms, page):
    """(row, page, place) of every row of the sequences."""
    out, r = [], 0
    for b, (n, m) in enumerate(zip(lens, ms)):
        for i in range(m):
            p = n - m + i
            out.append((r + i, int(table[b, p // page]), p % page) if p >= 0 else (r + i, -1, 0))
        r += m
    return out


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lens,ms,Hk,D,page", [([1], [1], 1, 64, 16), ([40, 1, 300], [40, 1, 300], 2, 128, 16), ([700, 33, 5, 64], [1, 1, 1, 1], 8, 128, 64),
                                               ([90, 16, 260], [3, 0, 8], 3, 256, 32), ([20] * 130, [1] * 130, 1, 64, 64)])
def test_cache_write_and_read(gpu, lens, ms, Hk, D, page, dtype):
    g = torch.Generator().manual_seed(len(lens) + D)
    kv, table = cache(g, lens, Hk, D, page)
    R = sum(ms)
    cu, ln = ints(offsets(ms)), ints(lens)
    k, v = rows(g, R + 2, Hk, D, dtype), rows(g, R + 2, Hk, D, dtype)           # two rows more, of no sequence
    want = {x: getattr(kv, x).cpu().numpy().copy() for x in ("kq", "ke", "vq", "ve")}
    for x, t in (("k", k), ("v", v)):
        q, e = attn_ref.quantise(host(t))
        for r, pg, at in places(table, lens, ms, page):
            want[x + "q"][pg, :, at], want[x + "e"][pg, :, at] = q[r], e[r]
    qmm.kv_write_mxfp4(k, v, kv, cu, ln, table, R + 2)
    for x in want:
        assert np.array_equal(getattr(kv, x).cpu().numpy(), want[x]), x
    for out in ("f32", "bf16"):
        ko, vo = (torch.full((R + 2, Hk * D), 5.0, dtype=T[out], device="cuda") for _ in range(2))
        qmm.kv_read_mxfp4(kv, cu, ln, table, ko, vo, R + 2)
        for x, t in (("k", ko), ("v", vo)):
            q, e = attn_ref.quantise(host(k if x == "k" else v))
            ref = attn_ref.values(q, e).reshape(R + 2, -1)
            ref[R:] = 5.0
            assert np.array_equal(host(t), ref.astype(np.float32)), (x, out)


def test_cache_places_that_are_none(gpu):
    """Rows at negative positions, beyond the table, on pages outside the cache: nothing is written; reads give NaN or leave rows."""
    g = torch.Generator().manual_seed(1)
    Hk, D, page = 2, 64, 16
    kv, table = cache(g, [32, 32, 32], Hk, D, page, ld=2)
    table[2, 1] = kv.pages                                                      # outside
    table[1, 1] = -1
    lens, ms = [2, 36, 32], [4, 8, 20]
    before = {x: getattr(kv, x).clone() for x in ("kq", "ke", "vq", "ve")}
    cu, ln = ints(offsets(ms)), ints(lens)
    k, v = rows(g, sum(ms), Hk, D, "bf16"), rows(g, sum(ms), Hk, D, "bf16")
    qmm.kv_write_mxfp4(k, v, kv, cu, ln, table, sum(ms))
    pos = [n - m + i for n, m in zip(lens, ms) for i in range(m)]
    seq = [b for b, m in enumerate(ms) for _ in range(m)]
    tab = table.cpu().numpy()
    for x in before:
        want = before[x].cpu().numpy()
        q = attn_ref.quantise(host(k if x[0] == "k" else v))[x[1] == "e"]
        for r, (p, b) in enumerate(zip(pos, seq)):
            if 0 <= p < 32 and 0 <= tab[b, p // page] < kv.pages:
                want[tab[b, p // page], :, p % page] = q[r]
        assert np.array_equal(getattr(kv, x).cpu().numpy(), want), x
    ko, vo = (torch.full((sum(ms), Hk * D), 5.0, device="cuda") for _ in range(2))
    qmm.kv_read_mxfp4(kv, cu, ln, table, ko, vo, sum(ms))
    for r, (p, b) in enumerate(zip(pos, seq)):
        if not 0 <= p < 32:
            assert (ko[r] == 5).all() and (vo[r] == 5).all()
        elif not 0 <= tab[b, p // page] < kv.pages:
            assert ko[r].isnan().all() and vo[r].isnan().all()
        else:
            assert np.array_equal(host(ko[r]), attn_ref.values(*attn_ref.quantise(host(k[r]))).astype(np.float32).ravel())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_cache_strided_and_unaligned_rows(gpu, dtype):
    g = torch.Generator().manual_seed(2)
    Hk, D, page, lens = 3, 64, 32, [50, 7]
    n, R = Hk * D, 57
    full = torch.randn((R, 3 * n + 5), generator=g).to(T[dtype]).cuda()
    cu, ln = ints([0, 50, 57]), ints(lens)
    got = []
    for k, v in ((full[:, 1:1 + n], full[:, n + 2:2 * n + 2]), (full[:, 1:1 + n].contiguous(), full[:, n + 2:2 * n + 2].contiguous())):
        kv, table = cache(torch.Generator().manual_seed(3), lens, Hk, D, page)
        qmm.kv_write_mxfp4(k, v, kv, cu, ln, table, R)
        out = torch.full((R, 2 * n + 3), 9.0, dtype=T[dtype], device="cuda")
        qmm.kv_read_mxfp4(kv, cu, ln, table, out[:, 1:n + 1], out[:, n + 2:2 * n + 2], R)
        assert (out[:, [0, n + 1, 2 * n + 2]] == 9).all()
        got.append((kv, out[:, 1:n + 1].clone(), out[:, n + 2:2 * n + 2].clone()))
    for x in ("kq", "ke", "vq", "ve"):
        assert torch.equal(getattr(got[0][0], x), getattr(got[1][0], x))
    assert torch.equal(got[0][1], got[1][1]) and torch.equal(got[0][2], got[1][2])


def test_cache_not_finite(gpu):
    """A block that holds a NaN or an infinity becomes NaN, the others stay."""
    k, v = torch.randn(2, 128, device="cuda"), torch.randn(2, 128, device="cuda")
    k[0, 40], v[1, 127] = float("inf"), float("nan")
    kv = qmm.KVMXBuf(1, 16, 1, 128)
    cu, ln, table = ints([0, 2]), ints([2]), ints([[0]])
    qmm.kv_write_mxfp4(k, v, kv, cu, ln, table, 2)
    ko, vo = torch.empty(2, 128, device="cuda"), torch.empty(2, 128, device="cuda")
    qmm.kv_read_mxfp4(kv, cu, ln, table, ko, vo, 2)
    want = torch.zeros(2, 2, 128, dtype=torch.bool)
    want[0, 0, 32:64] = want[1, 1, 96:] = True
    assert torch.equal(torch.stack([ko, vo]).isnan().cpu(), want)


# ---------------------------------------------------------------- attention over the cache
def attend(g, lens, ms, Hq, Hk, D, page, qt="bf16", ot="bf16", window=0, sinks=False, scale=None, max_len=None, max_rows=None, kv=None, table=None, q=None,
           extra=1):
    """A filled cache, random queries, one call: (out, kv, table, q, sinks)."""
    R = sum(ms)
    if kv is None:
        kv, table = cache(g, lens, Hk, D, page)
        al = offsets(lens)
        k, v = rows(g, al[-1], Hk, D, "bf16"), rows(g, al[-1], Hk, D, "bf16")
        if al[-1]:
            qmm.kv_write_mxfp4(k, v, kv, ints(al), ints(lens), table, al[-1])
    if q is None:
        q = rows(g, R + extra, Hq, D, qt)
    s = torch.randn(Hq, generator=g).cuda() if sinks is True else sinks if sinks is not False else None
    out = torch.full((R + extra, Hq * D), 3.0, dtype=T[ot], device="cuda")
    max_len = max_len or max(max(lens), 1)
    max_rows = max_rows or max(max(ms), 1)
    ws = torch.full((qmm.attn_kv_ws_bytes(R + extra, Hq, D, max_len),), 255, dtype=torch.uint8, device="cuda")
    qmm.attn_kv_mxfp4(q, kv, ints(offsets(ms)), ints(lens), table, out, R + extra, Hq, max_rows, max_len, ws, scale=scale, window=window, sinks=s)
    return out, kv, table, q, s


def fetched(kv, table):
    """The cache and the table on the host."""
    return {x: getattr(kv, x).cpu().numpy() for x in ("kq", "ke", "vq", "ve")} | {"table": table.cpu().numpy(), "page": kv.page}


def gather(c, b, n, h):
    """float64 keys and values of head h of sequence b, of a fetched cache."""
    p = np.arange(n)
    pg, at = c["table"][b][p // c["page"]], p % c["page"]
    return [attn_ref.values(c[x + "q"][pg, h, at], c[x + "e"][pg, h, at]) for x in "kv"]


def check_attend(out, kv, table, q, s, lens, ms, Hq, Hk, D, qt, ot, window, scale=None, max_rows=16):
    got, qh = host(out).reshape(-1, Hq, D), host(q).astype(np.float64).reshape(-1, Hq, D)
    wide, c = "f32" in (qt, ot), fetched(kv, table)
    r = 0
    for b, (n, m) in enumerate(zip(lens, ms)):
        mm = min(m, max_rows)
        for h in range(Hq if mm else 0):
            if h % (Hq // Hk) == 0:
                k, v = gather(c, b, n, h // (Hq // Hk))
            want, bound = attn_ref.attention(qh[r:r + mm, h], k, v, n - m + np.arange(mm), D ** -0.5 if scale is None else scale, window,
                                             None if s is None else float(s[h]), D // 32 * (3 if wide else 1) + 1, 2.0 ** -16 if wide else 2.0 ** -8, 24)
            err = np.abs(got[r:r + mm, h] - want)
            lim = bound + attn_ref.HALF[ot] * np.abs(want)
            assert (err <= lim).all(), (b, n, m, h, np.unravel_index(np.argmax(err - lim), err.shape), err.max(), lim.max())
        assert (got[r + min(m, max_rows):r + m] == 3).all()
        r += m
    assert (got[r:] == 3).all()


SHAPES = [([1], [1], 1, 1, 64, 16), ([700], [1], 32, 8, 128, 64), ([15, 16, 17, 31, 32, 33, 63, 64, 65], [1] * 9, 4, 2, 128, 16),
          ([255, 256, 257, 511, 513, 1100], [1, 2, 3, 1, 1, 4], 6, 2, 64, 32), ([40, 0, 300, 1], [5, 0, 8, 1], 8, 1, 256, 256),
          ([129, 600], [16, 7], 12, 4, 128, 128), ([1000, 3], [2, 2], 10, 2, 256, 32), ([77], [13], 16, 1, 64, 64), ([260, 50], [4, 1], 7, 1, 128, 4096)]


@pytest.mark.parametrize("qt,ot", [("bf16", "bf16"), ("f32", "f32"), ("bf16", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("lens,ms,Hq,Hk,D,page", SHAPES)
def test_attend(gpu, lens, ms, Hq, Hk, D, page, qt, ot):
    g = torch.Generator().manual_seed(sum(lens) + D)
    out, kv, table, q, s = attend(g, lens, ms, Hq, Hk, D, page, qt, ot)
    check_attend(out, kv, table, q, s, lens, ms, Hq, Hk, D, qt, ot, 0)


@pytest.mark.parametrize("window", [0, 1, 7, 32, 300])
@pytest.mark.parametrize("qt", ["bf16", "f32"])
@pytest.mark.parametrize("D,scale", [(64, None), (128, -0.2), (256, 0.0)])
def test_attend_window_and_sinks(gpu, window, qt, D, scale):
    g = torch.Generator().manual_seed(window + D)
    lens, ms = [400, 33, 1, 270], [3, 5, 1, 16]
    out, kv, table, q, s = attend(g, lens, ms, 8, 2, D, 32, qt, qt, window, True, scale)
    check_attend(out, kv, table, q, s, lens, ms, 8, 2, D, qt, qt, window, scale)


def test_attend_many_chunks(gpu):
    """More keys than 128 chunks of 256: longer chunks; and a max_len far beyond the sequences."""
    g = torch.Generator().manual_seed(5)
    lens, ms = [40000, 900], [2, 1]
    out, kv, table, q, s = attend(g, lens, ms, 2, 1, 64, 256)
    check_attend(out, kv, table, q, s, lens, ms, 2, 1, 64, "bf16", "bf16", 0)
    for max_len in (1 << 20, 1 << 30):
        far = attend(g, lens, ms, 2, 1, 64, 256, kv=kv, table=table, q=q, max_len=max_len)[0]
        check_attend(far, kv, table, q, s, lens, ms, 2, 1, 64, "bf16", "bf16", 0)


@pytest.mark.parametrize("D,B,m,Hq,Hk,window", [(64, 70, 1, 8, 8, 0), (128, 45, 1, 16, 8, 0), (256, 40, 2, 8, 8, 0), (128, 100, 3, 24, 4, 700), (64, 90, 2, 40, 4, 0)])
def test_attend_more_units_than_workgroups(gpu, D, B, m, Hq, Hk, window):
    """Workgroups that go from one sequence and head to the next, more sequences than a wave has lanes among them."""
    g = torch.Generator().manual_seed(B)
    lens = [1030 + (i * 211) % 1018 for i in range(B)]
    ms = [m if i % 7 else 0 for i in range(B)]
    out, kv, table, q, s = attend(g, lens, ms, Hq, Hk, D, 64, window=window, max_len=2048)
    check_attend(out, kv, table, q, s, lens, ms, Hq, Hk, D, "bf16", "bf16", window)


@pytest.mark.parametrize("D,Hk,share,m", [(64, 2, 8, 3), (64, 2, 8, 5), (64, 2, 7, 9), (64, 2, 10, 8), (64, 2, 8, 16), (128, 2, 8, 3), (128, 2, 5, 13), (256, 2, 8, 4)])
@pytest.mark.parametrize("qt", ["bf16", "f32"])
@pytest.mark.parametrize("chunks", [1, 118])
def test_attend_groups_of_many_rows(gpu, D, Hk, share, m, qt, chunks):
    """More units than are resident at once: groups of more than 16 rows, with the bits that a sequence by itself gives in groups of 16."""
    g = torch.Generator().manual_seed(m + D)
    if chunks == 1:
        lens, max_len = [1 + (i * 37) % 61 for i in range(140)], 1000 if D < 256 else 500
    else:
        lens, max_len = [530, 40, 1270], 512 * chunks
    ms = [m if i % 3 == 0 else 1 + i % m for i in range(len(lens))]
    Hq = Hk * share
    out, kv, table, q, s = attend(g, lens, ms, Hq, Hk, D, 32, qt, qt, 0, True, max_len=max_len)
    at = offsets(ms)
    for b in range(0, len(lens), 1 if chunks > 1 else 9):
        lone, *_ = attend(g, [lens[b]], [ms[b]], Hq, Hk, D, 32, qt, qt, 0, s, max_len=max_len, max_rows=m, kv=kv, table=table[b:b + 1],
                          q=q[at[b]:at[b + 1]], extra=0)
        assert torch.equal(lone, out[at[b]:at[b + 1]]), b
        check_attend(lone, kv, table[b:b + 1], q[at[b]:at[b + 1]], s, [lens[b]], [ms[b]], Hq, Hk, D, qt, qt, 0)


def test_attend_rows_that_see_nothing(gpu):
    """Positions below 0: zeros, with and without a sink; keys beyond max_len are not seen."""
    g = torch.Generator().manual_seed(6)
    for sinks in (False, True):
        lens, ms = [3, 20], [6, 2]
        out, kv, table, q, s = attend(g, lens, ms, 4, 2, 64, 16, sinks=sinks)
        assert (out[:3] == 0).all() and (out[3:6] != 0).any()
        check_attend(out, kv, table, q, s, lens, ms, 4, 2, 64, "bf16", "bf16", 0)
    for window in (0, 4):                                                       # max_len 8: 8 keys of 20, or none of the window's
        cut, *_ = attend(g, [20], [1], 4, 2, 64, 16, kv=kv, table=table[1:], q=q, max_len=8, window=window, extra=0)
        k, v = gather(fetched(kv, table), 1, 8, 0)
        want, bound = attn_ref.attention(host(q).astype(np.float64)[:1, 0], k, v, [19], 0.125, window, None, 3, 2.0 ** -8, 24)
        assert (np.abs(host(cut)[0, :64] - want) <= bound + 2.0 ** -8 * np.abs(want)).all()


@pytest.mark.parametrize("D,Hq,Hk", [(64, 8, 2), (128, 4, 1), (256, 8, 1), (128, 12, 1)])
@pytest.mark.parametrize("qt,ml", [("bf16", 512), ("f32", 512), ("bf16", 600), ("f32", 600), ("bf16", 3000), ("f32", 3000)])
def test_attend_rows_do_not_depend_on_each_other(gpu, D, Hq, Hk, qt, ml):
    """Drafted rows checked together are the bits that one after the other gives, and other sequences change nothing."""
    g = torch.Generator().manual_seed(7)
    lens, ms = [min(530, ml), 40, 270], [6, 1, 3]
    if ml > 600:                                         # several chunks, some rows' last key the first of one
        lens = [1540, 40, 513]
    out, kv, table, q, _ = attend(g, lens, ms, Hq, Hk, D, 32, qt, qt, max_len=ml)
    at = offsets(ms)
    for b, (n, m) in enumerate(zip(lens, ms)):
        for i in range(m):
            one, *_ = attend(g, [n - m + 1 + i], [1], Hq, Hk, D, 32, qt, qt, max_len=ml, kv=kv, table=table[b:b + 1], q=q[at[b] + i:at[b] + i + 1], extra=0)
            assert torch.equal(one[0], out[at[b] + i]), (b, i)


def test_attend_repeats_bit_for_bit(gpu):
    g = torch.Generator().manual_seed(8)
    a = attend(g, [3000, 900, 50], [1, 4, 2], 16, 4, 128, 64)
    for _ in range(3):
        assert torch.equal(attend(g, [3000, 900, 50], [1, 4, 2], 16, 4, 128, 64, kv=a[1], table=a[2], q=a[3])[0], a[0])


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("qt", ["bf16", "f32"])
def test_attend_nan_reaches_those_that_see_it(gpu, D, qt):
    """A NaN block of a value: that block of the rows that see the key.  A NaN key: those rows whole.  Other rows keep their bits."""
    g = torch.Generator().manual_seed(9)
    lens, ms, Hq, Hk = [300], [6], 4, 2
    out, kv, table, q, _ = attend(g, lens, ms, Hq, Hk, D, 16, qt, qt, extra=0)
    for name, key, blk in (("ve", 297, D // 32 - 1), ("ke", 296, 0), ("ve", 10, 0)):
        pg = int(table[0, key // 16])
        t = getattr(kv, name)
        kept = t.clone()
        t[pg, 1, key % 16, blk] = 255
        got = attend(g, lens, ms, Hq, Hk, D, 16, qt, qt, kv=kv, table=table, q=q, extra=0)[0].view(6, Hq, D)
        want = out.view(6, Hq, D).clone()
        seen = [i for i in range(6) if 294 + i >= key]
        for i in seen:
            if name == "ke":
                want[i, 2:] = float("nan")
            else:
                want[i, 2:, 32 * blk:32 * blk + 32] = float("nan")
        assert torch.equal(got.isnan(), want.isnan()), name
        assert torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0)), name
        t.copy_(kept)
    bad = q.clone()
    bad[2, 1, 5] = float("nan")
    got = attend(g, lens, ms, Hq, Hk, D, 16, qt, qt, kv=kv, table=table, q=bad, extra=0)[0].view(6, Hq, D)
    want = out.view(6, Hq, D).clone()
    want[2, 1] = float("nan")
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))


@pytest.mark.parametrize("byte", [253, 254, 255])
@pytest.mark.parametrize("qt", ["bf16", "f32"])
def test_scale_bytes_past_bf16(gpu, byte, qt):
    """They are NaN whatever the codes: in reads, and for the rows that see them; other rows keep their bits."""
    g = torch.Generator().manual_seed(14)
    lens, ms, D = [50], [4], 128
    out, kv, table, q, _ = attend(g, lens, ms, 2, 2, D, 16, qt, qt, extra=0)
    pg, at, want = int(table[0, 3]), 0, out.view(4, 2, D).clone()               # the key at 48: rows 2 and 3 see it
    kv.ve[pg, 1, at, 2] = byte
    want[2:, 1, 64:96] = float("nan")
    got = attend(g, lens, ms, 2, 2, D, 16, qt, qt, kv=kv, table=table, q=q, extra=0)[0].view(4, 2, D)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))
    kv.ke[pg, 1, at, 0] = byte
    want[2:, 1] = float("nan")
    got = attend(g, lens, ms, 2, 2, D, 16, qt, qt, kv=kv, table=table, q=q, extra=0)[0].view(4, 2, D)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))
    ko, vo = torch.zeros(2, 4, 2, D, dtype=T[qt], device="cuda")
    qmm.kv_read_mxfp4(kv, ints([0, 4]), ints(lens), table, ko, vo, 4)
    nan = torch.zeros(2, 4, 2, D, dtype=torch.bool)
    nan[0, 2, 1, :32] = nan[1, 2, 1, 64:96] = True
    assert torch.equal(torch.stack([ko, vo]).isnan().cpu(), nan)


def test_attend_page_outside_the_cache(gpu):
    """Its rows become NaN if they see the page, other sequences keep their bits."""
    g = torch.Generator().manual_seed(10)
    lens, ms = [100, 90], [1, 1]
    out, kv, table, q, _ = attend(g, lens, ms, 4, 2, 64, 16)
    for bad in (-1, kv.pages, 0x7fffffff, -0x80000000):
        t = table.clone()
        t[0, 3] = bad
        got = attend(g, lens, ms, 4, 2, 64, 16, kv=kv, table=t, q=q)[0]
        assert got[0].isnan().all() and torch.equal(got[1:], out[1:])
        t[0, 3], t[0, 6] = table[0, 3], bad                                     # the last page, beyond the window's first keys
        got = attend(g, [96, 90], ms, 4, 2, 64, 16, kv=kv, table=t, q=q)[0]
        assert not got[0].isnan().any()


def test_attend_strided_rows(gpu):
    """q and out as columns of wider rows."""
    g = torch.Generator().manual_seed(11)
    lens, ms, Hq, Hk, D = [90, 20], [2, 1], 4, 2, 64
    out, kv, table, q, _ = attend(g, lens, ms, Hq, Hk, D, 16, extra=0)
    full = torch.zeros(3, Hq * D + 16, dtype=torch.bfloat16, device="cuda")
    full[:, 8:8 + Hq * D] = q.view(3, -1)
    wide = torch.full((3, Hq * D + 3), 3.0, dtype=torch.bfloat16, device="cuda")
    qmm.attn_kv_mxfp4(full[:, 8:8 + Hq * D], kv, ints(offsets(ms)), ints(lens), table, wide[:, 1:1 + Hq * D], 3, Hq, 2, 90, None)
    assert torch.equal(wide[:, 1:1 + Hq * D], out) and (wide[:, [0, -2, -1]] == 3).all()


def test_attend_rows_beyond_max_rows(gpu):
    g = torch.Generator().manual_seed(12)
    lens, ms = [60, 300], [5, 2]
    out, kv, table, q, s = attend(g, lens, ms, 4, 2, 128, 16, max_rows=2)
    check_attend(out, kv, table, q, s, lens, ms, 4, 2, 128, "bf16", "bf16", 0, max_rows=2)


def test_attend_cache_beyond_32_bits(gpu):
    """Pages whose bytes lie past 2^32."""
    g = torch.Generator().manual_seed(13)
    Hk, D, page, lens = 8, 256, 256, [300]
    pages = (1 << 32) // (Hk * page * D // 2) + 40
    kv = qmm.KVMXBuf(1, page, Hk, D)
    kv.pages = pages
    for x, per in (("kq", 2), ("vq", 2), ("ke", 32), ("ve", 32)):
        setattr(kv, x, torch.empty((pages, Hk, page, D // per), dtype=torch.uint8, device="cuda"))
    table = ints([[pages - 1, pages - 30]])
    k, v = rows(g, 300, Hk, D, "bf16"), rows(g, 300, Hk, D, "bf16")
    qmm.kv_write_mxfp4(k, v, kv, ints([0, 300]), ints(lens), table, 300)
    ko, vo = (torch.empty(300, Hk * D, device="cuda") for _ in range(2))
    qmm.kv_read_mxfp4(kv, ints([0, 300]), ints(lens), table, ko, vo, 300)
    ref = [attn_ref.values(*attn_ref.quantise(host(t))) for t in (k, v)]
    assert np.array_equal(host(ko), ref[0].astype(np.float32).reshape(300, -1)) and np.array_equal(host(vo), ref[1].astype(np.float32).reshape(300, -1))
    out, _, _, q, _ = attend(g, lens, [2], 16, Hk, D, page, kv=kv, table=table)
    qh, got = host(q).astype(np.float64), host(out).reshape(-1, 16, D)
    for h in (0, 15):
        want, bound = attn_ref.attention(qh[:2, h], ref[0][:, h // 2], ref[1][:, h // 2], [298, 299], D ** -0.5, 0, None, 9, 2.0 ** -8, 24)
        assert (np.abs(got[:2, h] - want) <= bound + 2.0 ** -8 * np.abs(want)).all()


# ---------------------------------------------------------------- attention of prompts
def run_prompt(lens, ms, Hq, Hk, D, window=0, sinks=False, scale=None, seed=0, check=True, kv_rows=None):
    g = torch.Generator().manual_seed(sum(lens) + D + seed)
    aq, ak = offsets(ms), offsets(lens)
    q, k, v = rows(g, aq[-1] + 1, Hq, D, "bf16"), rows(g, ak[-1] + 1, Hk, D, "bf16"), rows(g, ak[-1] + 1, Hk, D, "bf16")
    k[-1], v[-1] = float("nan"), float("nan")                                   # rows of no sequence
    s = torch.randn(Hq, generator=g).cuda() if sinks else None
    out = torch.full((aq[-1] + 1, Hq, D), 3.0, dtype=torch.bfloat16, device="cuda")
    qmm.attn_prompt_bf16(q, k, v, ints(aq), None if lens is ms else ints(ak), out, Hq, Hk, D, scale=scale, window=window, sinks=s)
    if check:
        check_prompt(out, q, k, v, s, lens, ms, Hq, Hk, D, window, scale)
    return out, q, k, v, s


def check_prompt(out, q, k, v, s, lens, ms, Hq, Hk, D, window=0, scale=None):
    aq, ak = offsets(ms), offsets(lens)
    got, qh, kh, vh = (host(t).astype(np.float64) for t in (out, q, k, v))
    for b, (n, m) in enumerate(zip(lens, ms)):
        for h in range(Hq):
            hk = h // (Hq // Hk)
            want, bound = attn_ref.attention(qh[aq[b]:aq[b + 1], h], kh[ak[b]:ak[b + 1], hk], vh[ak[b]:ak[b + 1], hk], n - m + np.arange(m),
                                             D ** -0.5 if scale is None else scale, window, None if s is None else float(s[h]), D // 16 + 1, 2.0 ** -8,
                                             n / 16 + 4)
            err, lim = np.abs(got[aq[b]:aq[b + 1], h] - want), bound + 2.0 ** -8 * np.abs(want)
            assert (err <= lim).all(), (b, n, m, h, np.unravel_index(np.argmax(err - lim), err.shape), err.max(), lim.max())
    assert (got[aq[-1]:] == 3).all()


PROMPTS = [([1], 1, 1), ([300], 4, 2), ([31, 1, 33, 64, 65, 0, 127, 129], 2, 1), ([500, 20], 6, 2), ([257, 256], 3, 3)]


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("lens,Hq,Hk", PROMPTS)
def test_prompt(gpu, lens, Hq, Hk, D):
    run_prompt(lens, lens, Hq, Hk, D)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("lens,ms", [([400, 70], [30, 70]), ([200, 1, 640], [1, 1, 129]), ([5, 100, 0], [9, 130, 3])])
def test_prompt_behind_cached_keys(gpu, lens, ms, D):
    """Fewer rows than keys; more of them: the first rows see nothing."""
    run_prompt(lens, ms, 4, 2, D)
    run_prompt(lens, ms, 4, 2, D, sinks=True, window=50)


@pytest.mark.parametrize("window", [1, 5, 64, 100])
@pytest.mark.parametrize("D,scale", [(64, None), (128, -0.2), (256, 0.0)])
def test_prompt_window_and_sinks(gpu, window, D, scale):
    run_prompt([330, 70], [330, 70], 4, 1, D, window, True, scale)


def test_prompt_many_sequences(gpu):
    """More sequences than a wave has lanes, some empty."""
    lens = [(i * 7) % 23 for i in range(150)]
    run_prompt(lens, lens, 2, 1, 64)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_prompt_not_finite_values_where_masked(gpu, D):
    """Infinities and NaN reach the rows that see them: rows before them keep their bits, and the next sequence's too."""
    lens = [100, 90]
    out, q, k, v, _ = run_prompt(lens, lens, 2, 1, D)
    v2, k2 = v.clone(), k.clone()
    v2[40, 0, 3], v2[70, 0, D - 1], k2[80, 0, 7] = float("inf"), float("nan"), float("nan")
    got = torch.full_like(out, 3.0)
    qmm.attn_prompt_bf16(q, k2, v2, ints([0, 100, 190]), None, got, 2, 1, D)
    want = out.float()
    want[40:100, :, 3] = float("inf")
    want[70:100, :, D - 1] = float("nan")
    want[80:100] = float("nan")
    w, o = want[:190], got.float()[:190]
    assert torch.equal(o.isnan(), w.isnan()) and torch.equal(o.isinf(), w.isinf())
    fin = w.isfinite()
    assert torch.equal(o[fin], w[fin])


def test_prompt_strided_rows_of_one_product(gpu):
    """q, k and v as columns of the rows that one product made, out as columns of wider rows."""
    Hq, Hk, D, lens = 4, 2, 64, [130, 40]
    out, q, k, v, _ = run_prompt(lens, lens, Hq, Hk, D)
    R = 170
    full = torch.cat([t[:R].reshape(R, -1) for t in (q, k, v)] + [torch.zeros(R, 8, device="cuda", dtype=torch.bfloat16)], 1)
    a, b = Hq * D, Hk * D
    wide = torch.full((R, a + 16), 3.0, dtype=torch.bfloat16, device="cuda")
    qmm.attn_prompt_bf16(full[:, :a], full[:, a:a + b], full[:, a + b:a + 2 * b], ints([0, 130, 170]), None, wide[:, 8:8 + a], Hq, Hk, D)
    assert torch.equal(wide[:, 8:8 + a], out[:R].view(R, -1)) and (wide[:, :8] == 3).all() and (wide[:, 8 + a:] == 3).all()


def test_prompt_offsets_that_lead_out(gpu):
    """Offsets lie on the device: beyond the rows they are cut."""
    out, q, k, v, _ = run_prompt([50], [50], 2, 1, 64)
    for cu in ([0, 1000], [-5, 51], [60, 70], [30, 10], [0x7fffffff, -0x80000000]):
        got = torch.full_like(out, 3.0)
        qmm.attn_prompt_bf16(q[:50], k[:50], v[:50], ints(cu), None, got[:50], 2, 1, 64)
        assert torch.equal(got[:50], out[:50]) if cu in ([0, 1000], [-5, 51]) else (got == 3).all()


def test_prompt_rows_far_apart(gpu):
    """Keys and values whose rows lie beyond 2^32 bytes of the first one."""
    n, ld, D = 61000, 40000, 64
    far = torch.empty((n, ld), dtype=torch.bfloat16, device="cuda")
    k, v = far[:, :D], far[:, ld - D:]
    g = torch.Generator().manual_seed(30)
    k.copy_(torch.randn(n, D, generator=g))
    v.copy_(torch.randn(n, D, generator=g))
    q = torch.randn(3, D, generator=g).bfloat16().cuda()
    for ws in (None, False):
        out = torch.empty_like(q)
        qmm.attn_prompt_bf16(q, k, v, ints([0, 3]), ints([0, n]), out, 1, 1, D, ws=ws)
        qh, kh, vh = (host(t).astype(np.float64) for t in (q, k, v))
        want, bound = attn_ref.attention(qh, kh, vh, [n - 3, n - 2, n - 1], D ** -0.5, 0, None, D // 16 + 1, 2.0 ** -8, n / 16 + 4)
        assert (np.abs(host(out) - want) <= bound + 2.0 ** -8 * np.abs(want)).all()


def test_prompt_long(gpu):
    """2100 keys: sampled rows."""
    D, Hq, Hk, n = 128, 4, 2, 2100
    out, q, k, v, _ = run_prompt([n], [n], Hq, Hk, D, check=False)
    got, qh, kh, vh = (host(t).astype(np.float64) for t in (out, q, k, v))
    pick = np.array([0, 1, 63, 64, 1000, 1023, 1024, 2047, 2048, 2098, 2099])
    for h in range(Hq):
        want, bound = attn_ref.attention(qh[pick, h], kh[:n, h // 2], vh[:n, h // 2], pick, D ** -0.5, 0, None, D // 16 + 1, 2.0 ** -8, n / 16 + 4)
        assert (np.abs(got[pick, h] - want) <= bound + 2.0 ** -8 * np.abs(want)).all()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("window,sinks", [(0, False), (1500, True)])
def test_prompt_keys_in_parts(gpu, D, window, sinks):
    """Few rows behind many keys: the keys are cut into parts.  A workspace of the caller's gives the bits of the one that is made; without one
    the formula holds too; one too small is refused."""
    lens, ms, Hq, Hk = [4600, 2500], [70, 20], 4, 2
    out, q, k, v, s = run_prompt(lens, ms, Hq, Hk, D, window, sinks)
    size = qmm.attn_prompt_ws_bytes(91, 7101, 2, Hq, D)
    assert size > 0
    ws = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
    args = (q, k, v, ints(offsets(ms)), ints(offsets(lens)))
    for w in (ws, ws, False):
        got = torch.full_like(out, 3.0)
        qmm.attn_prompt_bf16(*args, got, Hq, Hk, D, window=window, sinks=s, ws=w)
        if w is False:
            check_prompt(got, q, k, v, s, lens, ms, Hq, Hk, D, window)
        else:
            assert torch.equal(got, out)
    with pytest.raises(QmmError, match="WORKSPACE"):
        qmm.attn_prompt_bf16(*args, out, Hq, Hk, D, ws=ws[:-16])
    st = torch.cuda.Stream()                             # a workspace made for another stream
    st.wait_stream(torch.cuda.current_stream())
    got = torch.full_like(out, 3.0)
    st.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        qmm.attn_prompt_bf16(*args, got, Hq, Hk, D, window=window, sinks=s, stream=st)
    torch.cuda.synchronize()
    assert torch.equal(got, out)


def test_prompt_parts_not_finite(gpu):
    """A value that is not finite in one part: it reaches the rows that see it, in that dim."""
    lens, ms, D = [2300], [40], 128
    out, q, k, v, _ = run_prompt(lens, ms, 2, 1, D)
    v2 = v.clone()
    v2[100, 0, 5], v2[2280, 0, 9] = float("inf"), float("nan")
    got = torch.full_like(out, 3.0)
    qmm.attn_prompt_bf16(q, k, v2, ints([0, 40]), ints([0, 2300]), got, 2, 1, D)
    want = out.float()
    want[:40, :, 5] = float("inf")
    want[20:40, :, 9] = float("nan")
    w, o = want[:40], got.float()[:40]
    assert torch.equal(o.isnan(), w.isnan()) and torch.equal(o.isinf(), w.isinf())
    fin = w.isfinite()
    assert torch.equal(o[fin], w[fin])


@pytest.mark.parametrize("D", [64, 128, 256])
def test_prompt_parts_without_weight(gpu, D):
    """A NaN value at a key whose weight is 0 in 32 bits, which an earlier part alone has seen, is NaN as without parts."""
    lens, n = [4000], 40
    q = torch.ones(n, 2, D, dtype=torch.bfloat16, device="cuda")
    k = torch.zeros(4000, 1, D, dtype=torch.bfloat16, device="cuda")
    k[3900:] = 8.0                                       # scores 32 sqrt(D) above the others': their weights are below 2^-369
    v = torch.randn(4000, 1, D, generator=torch.Generator().manual_seed(15)).bfloat16().cuda()
    v[70, 0, 3] = float("nan")
    assert qmm.attn_prompt_ws_bytes(n, 4000, 1, 2, D) > 0
    for w in (None, False):
        out = torch.zeros(n, 2, D, dtype=torch.bfloat16, device="cuda")
        qmm.attn_prompt_bf16(q, k, v, ints([0, n]), ints([0, 4000]), out, 2, 1, D, scale=4 * D ** -0.5, ws=w)
        assert out[:, :, 3].isnan().all() and not torch.cat([out[:, :, :3], out[:, :, 4:]], 2).isnan().any(), w


def test_prompt_workspace_of_another_stream(gpu):
    """The workspace that is made for a call on another stream is not memory that the current stream's work still reads."""
    lens, ms, D = [4600], [70], 64
    out, q, k, v, _ = run_prompt(lens, ms, 4, 2, D)
    size = qmm.attn_prompt_ws_bytes(q.shape[0], k.shape[0], 1, 4, D)
    assert size > 0
    cu, cuk, got = ints([0, 70]), ints([0, 4600]), torch.full_like(out, 3.0)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    t = torch.full((size,), 7, dtype=torch.uint8, device="cuda")
    torch.cuda._sleep(20_000_000)                        # some 10 ms
    kept = t.clone()
    del t
    qmm.attn_prompt_bf16(q, k, v, cu, cuk, got, 4, 2, D, stream=st)
    torch.cuda.synchronize()
    assert (kept == 7).all() and torch.equal(got[:70], out[:70])


# ---------------------------------------------------------------- together
def block(s):
    """Positions, cache, attention of one step, as a decoder block runs them."""
    qmm.rope_axes(s["qkv"][:, :s["nq"] + s["nk"]], s["qk"], s["pos"], s["freq"], s["axis"], s["R"], s["Hq"] + s["Hk"], s["D"])
    qmm.kv_write_mxfp4(s["qk"][:, s["nq"]:], s["v16"], s["kv"], s["cu"], s["lens"], s["table"], s["R"])
    if s["prompt"]:
        qmm.kv_read_mxfp4(s["kv"], s["cuk"], s["lens"], s["table"], s["ko"], s["vo"], s["N"])
        qmm.attn_prompt_bf16(s["qk"][:, :s["nq"]], s["ko"], s["vo"], s["cu"], s["cuk"], s["out"], s["Hq"], s["Hk"], s["D"])
    else:
        qmm.attn_kv_mxfp4(s["qk"][:, :s["nq"]], s["kv"], s["cu"], s["lens"], s["table"], s["out"], s["R"], s["Hq"], 16, s["cap"], s["ws"])
    qmm.quantize_mxfp4(s["out"], s["xq"], s["R"], s["nq"])


def state(lens, ms, kv, table, prompt, seed):
    g = torch.Generator().manual_seed(seed)
    Hq, Hk, D = 8, 2, 128
    R, N = sum(ms), sum(lens)
    nq, nk = Hq * D, Hk * D
    qkv = torch.randn(R, nq + 2 * nk, generator=g).cuda()
    bf = lambda n, w: torch.zeros(n, w, dtype=torch.bfloat16, device="cuda")           # noqa: E731
    at = [n - m + i for n, m in zip(lens, ms) for i in range(m)]
    return dict(qkv=qkv, qk=bf(R, nq + nk), v16=qkv[:, nq + nk:].bfloat16(), pos=ints([at, at, at]), freq=torch.rand(64, generator=g).cuda(),
                axis=(torch.arange(64) % 3).byte().cuda(), kv=kv, table=table, cu=ints(offsets(ms)), lens=ints(lens), cuk=ints(offsets(lens)), R=R, N=N, Hq=Hq,
                Hk=Hk, D=D, nq=nq, nk=nk, ko=bf(N, nk), vo=bf(N, nk), out=bf(R, nq), cap=512, prompt=prompt, xq=qmm.XMXBuf(R, nq),
                ws=torch.empty(qmm.attn_kv_ws_bytes(R, Hq, D, 512), dtype=torch.uint8, device="cuda"), l=lens, m=ms)


def check_block(s):
    turned, bound = attn_ref.rope(host(s["qkv"][:, :s["nq"] + s["nk"]]).reshape(s["R"], -1, s["D"]), s["pos"].cpu().numpy(), host(s["freq"]),
                                  s["axis"].cpu().numpy().astype(int), "halves", 1.0)
    got = host(s["qk"]).reshape(turned.shape)
    assert (np.abs(got - turned) <= bound + 2.0 ** -8 * np.abs(turned)).all()
    q = got[:, :s["Hq"]].astype(np.float64)
    r = 0
    for b, (n, m) in enumerate(zip(s["l"], s["m"])):
        for h in range(s["Hq"]):
            k, v = gather(fetched(s["kv"], s["table"]), b, n, h // 4)
            want, bo = attn_ref.attention(q[r:r + m, h], k, v, n - m + np.arange(m), s["D"] ** -0.5, 0, None, 9, 2.0 ** -8, n / 16 + 24)
            err = np.abs(host(s["out"])[r:r + m].reshape(m, s["Hq"], s["D"])[:, h] - want)
            assert (err <= bo + 2.0 ** -8 * np.abs(want)).all(), (b, h)
        r += m


def test_block_prompt_then_decode_eager_and_replayed(gpu):
    """A prompt, its rest behind what is cached, then a decode step: eager, and each captured and replayed with other eager work between."""
    g = torch.Generator().manual_seed(20)
    kv, table = cache(g, [200, 130], 2, 128, 32)
    steps = [state([120, 60], [120, 60], kv, table, True, 1), state([199, 125], [79, 65], kv, table, True, 2), state([200, 128], [1, 3], kv, table, False, 3)]
    for s in steps:
        block(s)
        check_block(s)
    kept = [{x: s[x].clone() for x in ("qk", "out")} | {"q": s["xq"].q.clone(), "e": s["xq"].e.clone()} for s in steps]
    graphs = []
    for s in steps:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            block(s)
        graphs.append(gr)
    for again in range(3):
        for s in steps:
            for x in ("qk", "out"):
                s[x].fill_(again)
        for gr, s, want in zip(graphs, steps, kept):
            gr.replay()
            torch.cuda.synchronize()
            assert torch.equal(s["qk"], want["qk"]) and torch.equal(s["out"], want["out"])
            assert torch.equal(s["xq"].q, want["q"]) and torch.equal(s["xq"].e, want["e"])
        block(steps[2])
        torch.cuda.synchronize()
        assert torch.equal(steps[2]["out"], kept[2]["out"])


def test_two_calls_at_once(gpu):
    """Two decode steps on two streams, with a workspace each."""
    g = torch.Generator().manual_seed(21)
    kv, table = cache(g, [300, 512], 2, 128, 32)
    fill = state([300, 500], [300, 500], kv, table, True, 4)
    block(fill)
    s = [state([300, 500], [1, 2], kv, table, False, 5), state([300, 500], [4, 1], kv, table, False, 6)]
    for x in s:
        x["kv"] = qmm.KVMXBuf(kv.pages, 32, 2, 128)
        for t in ("kq", "ke", "vq", "ve"):
            getattr(x["kv"], t).copy_(getattr(kv, t))
        block(x)
        x["want"] = x["out"].clone()
    torch.cuda.synchronize()
    for _ in range(5):
        streams = [torch.cuda.Stream() for _ in s]
        for x, st in zip(s, streams):
            x["out"].fill_(0)
            st.wait_stream(torch.cuda.current_stream())
        for _ in range(4):
            for x, st in zip(s, streams):
                with torch.cuda.stream(st):
                    block(x)
        torch.cuda.synchronize()
        for x in s:
            assert torch.equal(x["out"], x["want"])


def test_offsets_and_lengths_that_mean_nothing(gpu):
    """Offsets and lengths lie on the device: whatever they are, nothing outside the tensors is touched."""
    g = torch.Generator().manual_seed(14)
    _, kv, table, q, _ = attend(g, [60], [4], 2, 1, 64, 16, extra=0)
    x = q.view(4, -1)[:, :64].contiguous()
    big, low = 0x7fffffff, -0x80000000
    for cu in ([big, low], [low, big], [2, 1], [-3, 2], [4, 9]):
        for n in (big, low, 0, 60):
            out, wide = torch.full((6, 128), 3.0, dtype=torch.bfloat16, device="cuda"), torch.full((6, 64), 3.0, dtype=torch.bfloat16, device="cuda")
            fresh = qmm.KVMXBuf(kv.pages, 16, 1, 64)
            qmm.kv_write_mxfp4(x, x, fresh, ints(cu), ints([n]), table, 4)
            qmm.kv_read_mxfp4(fresh, ints(cu), ints([n]), table, wide[1:5], wide[1:5].clone(), 4)
            qmm.attn_kv_mxfp4(q, kv, ints(cu), ints([n]), table, out[1:5], 4, 2, 4, 64, None)
            ws = torch.empty(qmm.attn_kv_ws_bytes(4, 2, 64, 4096), dtype=torch.uint8, device="cuda")
            qmm.attn_kv_mxfp4(q, kv, ints(cu), ints([n]), table, out[1:5], 4, 2, 4, 4096, ws)
            assert (out[[0, 5]] == 3).all() and (wide[[0, 5]] == 3).all()


def test_no_rows(gpu):
    kv, e = qmm.KVMXBuf(2, 16, 1, 64), torch.empty(0, 64, device="cuda", dtype=torch.bfloat16)
    cu, ln, table = ints([0, 0]), ints([0]), ints([[0]])
    qmm.kv_write_mxfp4(e, e, kv, cu, ln, table, 0)
    qmm.kv_read_mxfp4(kv, cu, ln, table, e, e, 0)
    qmm.attn_kv_mxfp4(e, kv, cu, ln, table, e, 0, 1, 1, 16, None)
    qmm.attn_prompt_bf16(e, e, e, cu, None, e, 1, 1, 64)
    qmm.rope_axes(e, e, ints([]), torch.ones(32, device="cuda"), None, 0, 1, 64)
    torch.cuda.synchronize()


def test_foreign_tensors_are_refused(gpu):
    kv = qmm.KVMXBuf(2, 16, 1, 64)
    x = torch.zeros(2, 64, device="cuda", dtype=torch.bfloat16)
    cu, ln, table = ints([0, 2]), ints([2]), ints([[0]])
    for bad in (dict(k=x.cpu()), dict(k=x[:1]), dict(k=x.t()), dict(cu=cu.cpu()), dict(cu=cu.long()), dict(cu=cu[:1]), dict(table=table[0]), dict(k=x.half()),
                dict(k=x.float())):
        a = dict(k=x, cu=cu, table=table) | bad
        with pytest.raises(QmmError):
            qmm.kv_write_mxfp4(a["k"], x, kv, a["cu"], ln, a["table"], 2)
    with pytest.raises(QmmError):
        qmm.attn_kv_mxfp4(x, kv, cu, ln, table, x.clone(), 2, 1, 2, 5000, torch.empty(8, dtype=torch.uint8, device="cuda"))
    with pytest.raises(QmmError):
        qmm.attn_prompt_bf16(x.float(), x, x, cu, None, x.clone(), 1, 1, 64)
