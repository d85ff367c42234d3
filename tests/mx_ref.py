"""MXFP4 and the operators around it from their definitions, in numpy float64 (plain and slow: the tests' oracle)."""
import numpy as np

LEVELS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def steps(K):
    return -(-K // 128)


def quantise(x):
    """x f32 [R][K] -> codes [R][128 steps], scale bytes [R][4 steps] of the padded row (a block at a time)."""
    x = np.asarray(x, np.float64)
    R, K = x.shape
    v = np.zeros((R, steps(K) * 128))
    v[:, :K] = x
    v = v.reshape(R, -1, 32)
    amax = np.abs(v).max(2)
    bad = ~np.isfinite(amax) | np.isnan(v).any(2)
    safe = np.where(bad | (amax == 0), 1.0, amax)
    E = np.maximum(np.frexp(safe)[1] - 1 - 2, -127)
    E = np.where(amax == 0, -127, E)
    t = np.abs(np.where(bad[:, :, None], 0.0, v)) / np.exp2(E)[:, :, None]
    # nearest level, the tie to the even code
    d = np.abs(t[..., None] - LEVELS)
    best = d.min(-1)
    code = np.argmax(d == best[..., None], -1)                       # the lower of a tie
    upper = np.minimum(code + 1, 7)
    tie = (np.take_along_axis(d, upper[..., None], -1)[..., 0] == best) & (upper != code)
    code = np.where(tie & (code % 2 == 1), upper, code)
    code = code | (np.signbit(v) << 3)
    code = np.where(bad[:, :, None], 0, code)
    return code.reshape(R, -1).astype(np.uint8), np.where(bad, 255, E + 127).astype(np.uint8)


def pack(code):
    return (code[:, 0::2] | (code[:, 1::2] << 4)).astype(np.uint8)


def values(code, byte):
    """float64 values [R][padded K]."""
    v = np.where(code & 8, -1.0, 1.0) * LEVELS[code & 7]
    s = np.where(byte == 255, np.nan, np.exp2(byte.astype(np.float64) - 127))
    with np.errstate(invalid="ignore"):
        return v * np.repeat(s, 32, axis=1)


def random_rows(rng, R, K, spread=3):
    """Codes and scale bytes of R random rows of K values, padding zero: block scales 2^+-spread."""
    code = np.zeros((R, steps(K) * 128), np.uint8)
    code[:, :K] = rng.integers(0, 16, (R, K))
    byte = np.zeros((R, steps(K) * 4), np.uint8)
    nb = -(-K // 32)
    byte[:, :nb] = 127 + rng.integers(-spread, spread + 1, (R, nb))
    return code, byte


def product_bound(a, w, K):
    """(a w^T, bound of an f32 result's error).  One matrix instruction adds 128 products to its sum within
    2^-23 of the magnitudes it sees (twice a rounding); a chain of steps does it once each, and up to 8 partial
    sums add a rounding each."""
    mag = np.abs(a) @ np.abs(w).T
    return a @ w.T, (steps(K) + 8) * 2.0 ** -23 * mag


def route(logits, nexp, topk, score="softmax", bias=None, groups=1, keep=1, best=1, renorm=True, scale=1.0, shared=None):
    """ids and float64 weights, one token and one choice at a time."""
    T = logits.shape[0]
    slots = topk + (shared is not None)
    ids, w = np.full((T, slots), -1, np.int32), np.zeros((T, slots))
    for t in range(T):
        l = logits[t, :nexp].astype(np.float64)
        ok = l > -np.inf                                              # False for NaN
        s = np.zeros(nexp)
        if ok.any():
            with np.errstate(over="ignore"):
                if score == "softmax":
                    top = l[ok].max()
                    s[ok] = np.where(l[ok] == top, 1.0, np.exp(l[ok] - top if np.isfinite(top) else np.full(ok.sum(), -np.inf)))
                    s[ok] /= s[ok].sum()
                else:
                    s[ok] = 1.0 / (1.0 + np.exp(-l[ok]))
        c = s + (0 if bias is None else bias.astype(np.float64))
        c = np.where(ok & ~np.isnan(c), c, -np.inf)
        if keep < groups:
            g = -np.sort(-c.reshape(groups, -1), axis=1)[:, :best]
            val = np.where(np.isinf(g[:, -1]), g[:, 0], g.sum(1))
            kept = np.argsort(-val, kind="stable")[:keep]
            c = np.where(np.isin(np.arange(nexp) // (nexp // groups), kept), c, -np.inf)
        order = [e for e in np.argsort(-c, kind="stable")[:topk] if c[e] > -np.inf]
        p = s[order]
        tot = p.sum()
        ids[t, :len(order)] = order
        w[t, :len(order)] = (p / tot if tot > 0 else 0 * p) * scale if renorm else p * scale
        if shared == "gate":
            w[t, topk] = 1.0 / (1.0 + np.exp(-np.float64(logits[t, nexp])))
        elif shared == "one":
            w[t, topk] = 1.0
    return ids, w


def act(z, name):
    if name == "none":
        return z
    s = 1.0 / (1.0 + np.exp(-z))
    return s if name == "sigmoid" else z * s


def postnorm(x, y, wy, w, gate, name, alpha, eps):
    """(xo, xn, bounds of both): f32 arithmetic with U = 2^-24 a rounding.  A sum of squares is off by at most
    its longest path of additions (16 values, 5 tree steps, 32 wave sums), which the root halves, and mean, root and
    quotient round: rms within 32 U.  p has rms, two products, the gate (exp, 1 +, quotient and product: 6 U) and its
    product.  xn repeats this on an xo that is itself off."""
    U = 2.0 ** -24
    x, y, w = (np.asarray(v, np.float64) for v in (x, y, w))
    rms = lambda v: np.sqrt((v * v).mean(1, keepdims=True) + eps)     # noqa: E731
    p = y / rms(y) * np.asarray(wy, np.float64) if wy is not None else y
    if gate is not None:
        p = p * act(np.asarray(gate, np.float64), name)
    xo = x + alpha * p
    bo = U * np.abs(xo) + 44 * U * np.abs(alpha * p)
    r = rms(xo)
    xn = xo / r * w
    shift = np.sqrt((bo * bo).mean(1, keepdims=True)) / r             # of rms, from the errors of xo
    bn = np.abs(w) / r * bo + np.abs(xn) * (36 * U + shift)
    return xo, xn, bo, bn
