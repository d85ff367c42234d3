"""qmm_moe_route_groups against tests/mx_ref.py: ids equal, weights within their one rounding to f32 (2^-24) and the
float64 arithmetic of both sides (1e-13)."""
import numpy as np
import pytest
import torch

import mx_ref
from hipster_amd import qmm
from hipster_amd._lib import QmmError
from tests.gpu_util import dev, host

pytestmark = pytest.mark.gpu

TOL = 2.0 ** -24 + 1e-13


def run(logits, nexp, topk, bias=None, pad=2, **kw):
    T = logits.shape[0]
    slots = topk + (kw.get("shared") is not None)
    ids = torch.full((T + pad, slots), -9, dtype=torch.int32, device="cuda")
    w = torch.full((T + pad, slots), -9.0, device="cuda")
    qmm.moe_route_groups(dev(logits), ids, w, T, nexp, topk, bias=None if bias is None else dev(bias), **kw)
    ids, w = host(ids), host(w)
    assert (ids[T:] == -9).all() and (w[T:] == -9).all()
    return ids[:T], w[:T]


def check(logits, nexp, topk, **kw):
    ids, w = run(logits, nexp, topk, **kw)
    rid, rw = mx_ref.route(logits, nexp, topk, **kw)
    assert np.array_equal(ids, rid)
    assert (np.abs(w - rw) <= TOL * np.abs(rw) + 2.0 ** -150).all()
    return ids, w


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,k,groups,keep,best", [(1, 512, 10, 1, 1, 1), (1, 1, 1, 1, 1, 1), (3, 7, 7, 1, 1, 1), (9, 60, 4, 1, 1, 1), (130, 64, 6, 8, 3, 1),
                                                    (65, 256, 8, 8, 4, 2), (33, 160, 6, 5, 2, 2), (17, 1024, 16, 64, 5, 2), (20, 96, 3, 3, 1, 2),
                                                    (6, 64, 2, 64, 2, 1), (4, 64, 2, 64, 2, 2), (5, 1000, 16, 1, 1, 2), (40, 384, 8, 12, 12, 2)])
def test_rules(gpu, T, E, k, groups, keep, best, score):
    rng = np.random.default_rng(T + E)
    for i, (bias, shared, renorm, scale) in enumerate(((False, None, True, 1.0), (True, "gate", True, 2.5), (True, "one", False, 0.3))):
        logits = (rng.standard_normal((T, E + 1 + i)) * 2).astype(np.float32)          # a wider row than needed too
        b = (rng.standard_normal(E) * 0.2).astype(np.float32) if bias else None
        check(logits, E, k, score=score, bias=b, groups=groups, keep=keep, best=best, renorm=renorm, scale=np.float32(scale).item(), shared=shared)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_ties_go_to_the_lower_id(gpu, score):
    rng = np.random.default_rng(1)
    logits = rng.integers(-2, 3, (200, 256)).astype(np.float32)                        # a few values only
    check(logits, 256, 10, score=score)
    check(logits, 256, 10, score=score, groups=16, keep=3, best=2)
    ids, _ = check(np.zeros((3, 512), np.float32), 512, 10, score=score)
    assert (ids == np.arange(10)).all()
    ids, _ = check(np.zeros((3, 512), np.float32), 512, 10, score=score, groups=8, keep=2, best=2)
    assert (ids == np.arange(10)).all()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_masked_and_extreme_logits(gpu, score):
    rng = np.random.default_rng(2)
    l = rng.standard_normal((12, 64)).astype(np.float32)
    l[0] = -np.inf                                                                     # no expert at all
    l[1, 1:] = -np.inf                                                                 # one
    l[2, ::2] = np.nan
    l[3, :56] = -np.inf                                                                # one group of eight
    l[4] = np.finfo(np.float32).min
    l[5, 7] = np.inf
    l[6, [3, 9]] = np.inf
    l[7] = np.linspace(-200, 200, 64)
    l[8] = 1e-30 * np.arange(64)
    l[9] = 88.0
    l[10, 5:] = np.nan
    for kw in (dict(), dict(groups=8, keep=2, best=2), dict(groups=8, keep=3, best=1, shared="one"), dict(renorm=False, scale=2.0)):
        ids, w = check(l, 64, 6, score=score, **kw)
        assert (ids[0, :6] == -1).all() and (w[0, :6] == 0).all() and (ids[1, 1:6] == -1).all()
    b = np.zeros(64, np.float32)
    b[4], b[5] = np.nan, -np.inf
    ids, _ = check(l, 64, 6, score=score, bias=b)
    assert not np.isin(ids, (4, 5)).any()


def test_negative_choice_values(gpu):
    """A bias that pushes every choice value below zero: the order of negative doubles, and masked experts still last."""
    rng = np.random.default_rng(3)
    l = rng.standard_normal((50, 128)).astype(np.float32)
    l[:, 100:] = -np.inf
    b = (-3 - rng.random(128)).astype(np.float32)
    ids, _ = check(l, 128, 8, score="sigmoid", bias=b, groups=4, keep=4)
    assert (ids < 100).all()
    check(l, 128, 8, score="sigmoid", bias=b, groups=4, keep=2, best=2)


def test_agrees_with_the_plain_routing(gpu):
    """Softmax without groups is qmm_moe_route_n's rule (its f32 arithmetic within 1e-5)."""
    rng = np.random.default_rng(4)
    l = rng.standard_normal((64, 513)).astype(np.float32)
    ids, w = run(l, 512, 10, shared="gate")
    i2, w2 = torch.zeros(64, 11, dtype=torch.int32, device="cuda"), torch.zeros(64, 11, device="cuda")
    qmm.moe_route_n(dev(l), i2, w2, 64, 512, 513, 10)
    assert np.array_equal(ids, host(i2))
    np.testing.assert_allclose(w, host(w2), rtol=1e-5, atol=1e-7)


def test_long_call_and_graph(gpu):
    rng = np.random.default_rng(5)
    T, E, k = 5003, 256, 8
    l = rng.standard_normal((T, E)).astype(np.float32)
    kw = dict(score="sigmoid", groups=8, keep=4, best=2, scale=2.5)
    check(l, E, k, **kw)
    dl, ids, w = dev(l), torch.zeros(T, k, dtype=torch.int32, device="cuda"), torch.zeros(T, k, device="cuda")
    qmm.moe_route_groups(dl, ids, w, T, E, k, **kw)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qmm.moe_route_groups(dl, ids, w, T, E, k, **kw)
    for i in range(3):
        l = rng.standard_normal((T, E)).astype(np.float32)
        dl.copy_(torch.from_numpy(l))
        graph.replay()
        assert np.array_equal(host(ids), mx_ref.route(l, E, k, **kw)[0])
        torch.cuda.synchronize()


def test_refusals(gpu):
    l, ids, w = torch.zeros(2, 64, device="cuda"), torch.zeros(2, 4, dtype=torch.int32, device="cuda"), torch.zeros(2, 4, device="cuda")
    for bad in (dict(score="relu"), dict(shared="gate"), dict(groups=3), dict(groups=8, keep=9), dict(best=3), dict(bias=torch.zeros(63, device="cuda"))):
        with pytest.raises(QmmError):
            qmm.moe_route_groups(l, ids, w, 2, 64, 4, **bad)
    with pytest.raises(QmmError):
        qmm.moe_route_groups(l, ids, w, 3, 64, 4)
    with pytest.raises(QmmError):
        qmm.moe_route_groups(l.double(), ids, w, 2, 64, 4)
