"""Attention's operators from their definitions, in numpy float64 (plain and slow: the tests' oracle), with bounds of an f32 result's error.

Bounds count: a rounding is half a step (bf16 2^-8, f32 2^-24, relative); a bf16 matrix instruction adds its products to its sum within
2^-23 of the magnitudes it sees; the hardware's 2^x is within 2^-22."""
import numpy as np

import mx_ref

U = 2.0 ** -24
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8}


def quantise(x):
    """x f32 [..][D] -> packed codes [..][D / 2], scale bytes [..][D / 32]."""
    D = x.shape[-1]
    code, byte = mx_ref.quantise(np.asarray(x, np.float32).reshape(-1, D))
    return mx_ref.pack(code[:, :D]).reshape(*x.shape[:-1], D // 2), byte[:, :D // 32].reshape(*x.shape[:-1], D // 32)


def values(q, e):
    """float64 values of packed codes [..][D / 2] with scale bytes [..][D / 32]."""
    if q.size == 0:
        return np.zeros((*q.shape[:-1], 2 * q.shape[-1]))
    code = np.stack([q & 15, q >> 4], -1).reshape(*q.shape[:-1], -1)
    v = mx_ref.values(code.reshape(-1, code.shape[-1]), e.reshape(-1, e.shape[-1]))
    return v.reshape(code.shape)


def rope(x, pos, freq, axis, style, scale):
    """x [T][H][D], pos [axes][T] -> (y, bound without the output's rounding).  Cosine and sine are within 2^-22, times scale
    one rounding; two products and a sum round each: within 2^-22 + 3 U of |a| + |b|."""
    y, P = x.astype(np.float64).copy(), len(freq)
    ang = pos[axis if axis is not None else np.zeros(P, int)].T.astype(np.float64) * freq.astype(np.float64)       # below 2^53: exact enough
    c, s = np.cos(ang)[:, None] * scale, np.sin(ang)[:, None] * scale
    ia, ib = (np.arange(P), np.arange(P) + P) if style == "halves" else (2 * np.arange(P), 2 * np.arange(P) + 1)
    a, b = y[:, :, ia], y[:, :, ib]
    bound = np.zeros_like(y)
    bound[:, :, ia] = bound[:, :, ib] = (np.abs(a) + np.abs(b)) * abs(scale) * (2.0 ** -22 + 3 * U)
    y[:, :, ia], y[:, :, ib] = a * c - b * s, b * c + a * s
    return y, bound


def attention(q, k, v, pos, scale, window, sink, terms, wround, steps):
    """One head: q [m][D] at positions pos, k, v [n][D] -> (o, bound without the output's rounding).

    terms: matrix instructions of a score (each 2^-23 of sum |q k|), wround: rounding of a weight, steps: those of the sums.
    A score is scaled with two roundings, its difference to the maximum is one; weights are rescaled with 2^x at most `steps` times."""
    m, n = q.shape[0], k.shape[0]
    o, bound = np.zeros((m, v.shape[1])), np.zeros((m, v.shape[1]))
    for i in range(m):
        j = np.arange(n)
        see = (j <= pos[i]) & ((j > pos[i] - window) if window else True)
        if not see.any():
            continue
        ks, vs = k[see], v[see]
        t = (ks @ q[i]) * scale
        mag = np.abs(ks) @ np.abs(q[i]) * abs(scale)
        top = max(t.max(), sink) if sink is not None else t.max()
        w = np.exp(t - top)
        L = w.sum() + (np.exp(sink - top) if sink is not None else 0.0)
        w /= L
        eps = (terms * 2 * U * mag + 3 * U * (np.abs(t) + np.abs(t - top))).max() + (2 + steps) * 2.0 ** -22
        o[i] = w @ vs
        A = w @ np.abs(vs)
        bound[i] = A * (eps + wround + steps * 2 * U) + np.abs(o[i]) * (eps + steps * U + 4 * U)
    return o, bound
