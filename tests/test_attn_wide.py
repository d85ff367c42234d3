"""Attention over the cache where q or out is f32: its matrix products take bf16 factors, so that q and the weights go in as three parts of 8
bits each.  A bound that counts the roundings of that path alone (attn_ref.attention's allows a weight's third part to be lost), inputs on
which a third part shows, and on the CPU the proof that the bound rejects two parts."""
import numpy as np
import pytest
import torch

import attn_ref
from hipster_amd import qmm
from test_attn_gpu import SHAPES, attend, cache, fetched, gather, host, ints, offsets

U, STEP, EXP = 2.0 ** -24, 2.0 ** -23, 2.0 ** -22       # a rounding of f32; a matrix instruction's sum; the hardware's 2^x


def parts(x, n):
    """The first n of the parts of 8 significant bits, toward zero, that an f32 is the sum of."""
    rest, out = np.asarray(x, np.float32), np.zeros(np.shape(x))
    for _ in range(n):
        p = (rest.view(np.uint32) & np.uint32(0xffff0000)).view(np.float32)
        out, rest = out + p, rest - p
    return out


def attention(q, k, v, pos, scale, window, sink, adds, steps, joins, split=None):
    """One head in float64: (o, bound without the output's rounding).  split (of q, of the weights): that many parts of each, not all.

    adds: matrix instructions whose products are not all zero in a score; steps: of 32 keys that one wave takes of a chunk; joins: of waves and
    chunks that have keys to join (none: 2^0 and times 1 are exact).  A score: its sums, the scale's rounding and the product's.  A weight: its
    difference to the maximum, 2^x, and, for every step but the first and every join, which may move the maximum, one more of both and a
    product.  Three instructions a step add the weights' parts times the values; the weights' sum adds eight a step, those of other
    lanes (2) and one a join.  The end: a quotient and a product."""
    m, n = q.shape[0], k.shape[0]
    o, bound = np.zeros((m, v.shape[1])), np.zeros((m, v.shape[1]))
    for i in range(m):
        j = np.arange(n)
        see = (j <= pos[i]) & ((j > pos[i] - window) if window else True)
        if not see.any():
            continue
        ks, vs = k[see], v[see]
        qi = q[i] if split is None else parts(q[i], split[0])
        t = (ks @ qi) * scale
        mag = np.abs(ks) @ np.abs(q[i]) * abs(scale)
        top = max(t.max(), sink) if sink is not None else t.max()
        w = np.exp(t - top)
        L = w.sum() + (np.exp(sink - top) if sink is not None else 0.0)
        o[i] = (w if split is None else parts(w, split[1])) @ vs / L
        w /= L
        span = np.abs(t - top).max()
        eps = (adds * STEP * mag + 2 * U * np.abs(t)).max() + U * span + EXP + (steps - 1 + joins) * (EXP + U) + 2 * U * span
        if sink is not None:                                                # its factor log2(e) and product, and one more join
            eps += 2 * U * abs(sink) + U * abs(t.max() - sink) + EXP + U
        bound[i] = (w @ np.abs(vs)) * (eps + 3 * steps * STEP + 2 * joins * U) + np.abs(o[i]) * (eps + (8 * steps + 2 + 2 * joins + 2) * U)
    return o, bound


def counts(n, max_len, D):
    """Steps a wave takes of a chunk and joins, at most: chunks of 256 keys or more, four or eight waves."""
    return -(-min(n, 1024) // 128), 8 + (0 if max_len <= (512 if D == 256 else 1024) else -(-max_len // 256))


# ---- inputs on which the third part shows ----
def inputs(rng, n, D, m, what):
    """Keys with one value that is not zero, so that scores round little, and queries of all 24 bits.  "scores": up to 8, beside a sink as
    heavy as all keys, so that a score's error is the output's.  "weights": from 1 down to a half, values of 1."""
    k, v = np.zeros((n, D), np.float32), np.ones((n, D), np.float32)
    q = rng.uniform(0.55, 1.0, (m, D)).astype(np.float32)
    if what == "scores":
        k[:, D // 2 + 1] = 8.0
        v = rng.choice([1, 1.5, 2, 3, 4, 6], (n, D)).astype(np.float32)
        return q, k, v, 6.2 + float(np.log(n))
    k[:, D // 2 + 1] = rng.choice([0.25, 0.375, 0.5, -0.125, -0.25, 0.125], n)
    return q, k, v, None


CASES = [(D, what) for D in (64, 128, 256) for what in ("scores", "weights")]


@pytest.mark.parametrize("D,what", CASES)
def test_the_bound_rejects_two_parts(D, what):
    """Many rows are off by more than the bound if q or the weights lose their third part, and far within it with all three."""
    q, k, v, sink = inputs(np.random.default_rng(D), 30, D, 40, what)
    a = (q, k.astype(np.float64), v.astype(np.float64), np.full(40, 29), 1.0, 0, sink, 3, 1, 0)
    o, bound = attention(*a)
    for split in ((3, 3), (2, 3) if what == "scores" else (3, 2)):
        over = (np.abs(attention(*a, split=split)[0] - o) / (bound + U * np.abs(o))).max(1)
        assert (over < 0.1).all() if split == (3, 3) else (over > 1).mean() > 0.4, (split, over)


def test_three_parts_are_all():
    x = np.random.default_rng(3).normal(size=4000).astype(np.float32) * np.exp2(np.random.default_rng(4).integers(-60, 60, 4000)).astype(np.float32)
    assert np.array_equal(parts(x, 3), x.astype(np.float64)) and not np.array_equal(parts(x, 2), x.astype(np.float64))


# ---- the kernels ----
def filled(g, B, n, Hk, D, k, v):
    """A cache in which every head of every sequence has these n keys and values."""
    kv, table = cache(g, [n] * B, Hk, D, 16)
    kk, vv = (torch.from_numpy(np.tile(x[None, :, None, :], (B, 1, Hk, 1)).reshape(B * n, Hk * D)).cuda() for x in (k, v))
    qmm.kv_write_mxfp4(kk, vv, kv, ints(offsets([n] * B)), ints([n] * B), table, B * n)
    return kv, table


@pytest.mark.gpu
@pytest.mark.parametrize("D,what", CASES)
@pytest.mark.parametrize("B,share,max_len", [(1, 4, 64), (1, 4, 4000), (200, 7, 64), (200, 9, 64), (120, 9, 4000)])
def test_a_third_part_is_not_lost(gpu, D, what, B, share, max_len):
    """Groups of 16 rows and, with more units than are resident, of more; one chunk and several."""
    n, m, Hk = 30, 5, 8
    rng = np.random.default_rng(D + B)
    g = torch.Generator().manual_seed(D)
    q, k, v, sink = inputs(rng, n, D, B * m * Hk * share, what)
    kv, table = filled(g, B, n, Hk, D, k, v)
    held = fetched(kv, table)
    assert np.array_equal(np.stack(gather(held, B - 1, n, Hk - 1)), np.stack([k, v]))           # the cache holds them exactly
    out, *_ = attend(g, [n] * B, [m] * B, Hk * share, Hk, D, 16, "f32", "f32", scale=1.0, sinks=False if sink is None else torch.full((Hk * share,), sink, device="cuda"), max_len=max_len, max_rows=m, kv=kv, table=table,
                     q=torch.from_numpy(q).view(B * m, Hk * share, D).cuda(), extra=0)
    pos = np.repeat(np.tile(n - m + np.arange(m), B), Hk * share)
    pick = rng.permutation(len(pos))[:600]
    sink = None if sink is None else float(np.float32(sink))
    want, bound = attention(q[pick], k.astype(np.float64), v.astype(np.float64), pos[pick], 1.0, 0, sink, 3, 1, 0)            # one step has all keys
    got = host(out).reshape(-1, D)[pick]
    assert (np.abs(got - want) <= bound + U * np.abs(want)).all(), (np.abs(got - want) / (bound + U * np.abs(want))).max()


@pytest.mark.gpu
@pytest.mark.parametrize("qt", ["f32", "bf16"])
@pytest.mark.parametrize("window", [0, 300])
@pytest.mark.parametrize("lens,ms,Hq,Hk,D,page", SHAPES + [([2100, 900], [3, 5], 4, 1, 64, 64), ([1700], [2], 4, 2, 256, 32)])
def test_attend_in_f32(gpu, lens, ms, Hq, Hk, D, page, window, qt):
    """Shapes of every kind, f32 out, within the tighter bound."""
    g = torch.Generator().manual_seed(sum(lens) + D + 1)
    out, kv, table, q, s = attend(g, lens, ms, Hq, Hk, D, page, qt, "f32", window, True)
    got, qh, c, r = host(out).reshape(-1, Hq, D), host(q).astype(np.float64).reshape(-1, Hq, D), fetched(kv, table), 0
    for b, (n, m) in enumerate(zip(lens, ms)):
        for h in range(Hq if m else 0):
            k, v = gather(c, b, n, h // (Hq // Hk))
            want, bound = attention(qh[r:r + m, h], k, v, n - m + np.arange(m), D ** -0.5, window, float(s[h]), D // 32 * (3 if qt == "f32" else 1),
                                    *counts(n, max(lens), D))
            err, lim = np.abs(got[r:r + m, h] - want), bound + attn_ref.HALF["f32"] * np.abs(want)
            assert (err <= lim).all(), (b, n, m, h, (err / lim).max())
        r += m
