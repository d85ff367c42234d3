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
