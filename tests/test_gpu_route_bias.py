"""The order by score + bias, where neither decides alone: biases as large as the scores' differences.

Only tokens whose order FP32 cannot change are compared: a score is off by at most 64 x 2^-24 of itself (as in
test_gpu_route.py) and its sum with the bias by 2^-24 of that, so values (and groups' scores) further apart than
twice both keep their order."""
import numpy as np
import pytest
import torch
from test_gpu_route import TOL, check, reference

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
E, TOPK = 64, 6


def clear(x, score, bias, kw):
    """The tokens whose order is clear of rounding."""
    s = np.empty_like(x, np.float64)
    ids, w = reference(x, E, score)
    np.put_along_axis(s, ids, w, 1)
    c = s + bias
    off = TOL * s.max(1) + 2.0 ** -24 * np.abs(c).max(1)
    ok = np.diff(np.sort(c, 1), axis=1).min(1) > 2 * off
    if kw.get("n_group", 1) > 1:
        by = -np.sort(-c.reshape(len(x), kw["n_group"], -1), 2)
        of = by[..., 0] if kw["group_score"] == "max" else by[..., 0] + by[..., 1]
        ok &= np.diff(np.sort(of, 1), axis=1).min(1) > 4 * off + 2.0 ** -23 * np.abs(of).max(1)
    return x[ok]


def inputs(score, kw):
    rng = np.random.default_rng(12)
    x = rng.normal(size=(600, E)).astype(np.float32)
    # as large as the spread of the scores
    bias = (rng.normal(size=E) * (0.01 if score == "softmax" else 0.15)).astype(np.float32).astype(np.float64)
    return clear(x, score, bias, kw), bias


CASES = [("softmax", {}), ("softmax", dict(n_group=8, topk_group=4, group_score="top2")), ("softmax", dict(n_group=8, topk_group=3, group_score="max")),
         ("sigmoid", {}), ("sigmoid", dict(n_group=8, topk_group=4, group_score="top2")), ("sigmoid", dict(n_group=8, topk_group=3, group_score="max"))]


@pytest.mark.parametrize("score,kw", CASES)
def test_scores_and_bias_order_together(score, kw):
    x, bias = inputs(score, kw)
    ids = lambda x, bias: np.sort(reference(x, TOPK, score, bias, **kw)[0], 1)  # noqa: E731
    both = ids(x, bias)
    assert len(x) > 300
    assert (both != ids(x, None)).any(1).mean() > 0.8                 # the bias alters most selections,
    assert (both != ids(np.zeros_like(x), bias)).any(1).mean() > 0.8   # and so do the scores
    check(torch.tensor(x, device=DEV), TOPK, bias=bias, score=score, renormalize=True, scaling=2.5, **kw)
    check(torch.tensor(x, device=DEV), TOPK, bias=bias, score=score, n_forced=2, **kw)
