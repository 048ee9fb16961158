"""route_experts on the GPU against a plain NumPy routing in 64 bits.

Selections are compared exactly, so the random logits are drawn from a grid whose scores differ by far
more than FP32 rounds (ties are tested apart, with equal logits). Weights: a softmax's terms have at
most 2 units of 2^-23 from expf and |l - max| 2^-24 from its argument, its sum at most 16 + 5 roundings
(a lane's values, then five shuffles), the division and the scaling one each, the renormalising sum
of at most 5 shuffles and its division 6 more: 64 x 2^-24 relative covers |l - max| <= 16."""
import numpy as np
import pytest
import torch

from fleet.routing import route_experts

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TOL = 64 * 2.0 ** -24


def reference(x, topk, score="softmax", bias=None, n_group=1, topk_group=1, group_score="max", renormalize=False,
              scaling=1.0, n_forced=0):
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    T, E = x.shape
    with np.errstate(all="ignore"):
        if score == "sigmoid":
            s = 1 / (1 + np.exp(-x))
        else:
            m = x.max(1, keepdims=True)
            e = np.where(np.isneginf(m), 0.0, np.where(x == m, 1.0, np.exp(x - m)))
            s = e / np.maximum(e.sum(1, keepdims=True), 1e-300)
    c = s if bias is None else s + bias
    c = np.where(np.isnan(c), -np.inf, c)
    if n_group > 1:
        by = -np.sort(-c.reshape(T, n_group, -1), 2)
        of = by[..., 0] if group_score == "max" or by.shape[2] == 1 else by[..., 0] + by[..., 1]
        out = np.argsort(-of, 1, kind="stable")[:, topk_group:]
        c = c.reshape(T, n_group, -1).copy()
        dropped = np.zeros(c.shape, bool)
        np.put_along_axis(dropped, out[:, :, None], True, 1)
        dropped = dropped.reshape(T, E)
        c = c.reshape(T, E)
    else:
        dropped = np.zeros((T, E), bool)
    # the kept experts first, by the selection, ties to the lowest index
    ids = np.lexsort((np.broadcast_to(np.arange(E), (T, E)), -c, dropped), axis=1)[:, :topk]
    w = np.take_along_axis(s, ids, 1)
    if renormalize:
        total = w.sum(1, keepdims=True)
        w = np.where(total == 0, 0.0, w / np.where(total == 0, 1, total))
    ids = np.concatenate([ids, np.broadcast_to(np.arange(E, E + n_forced), (T, n_forced))], 1)
    return ids, np.concatenate([w * scaling, np.ones((T, n_forced))], 1)


def grid_logits(T, E, seed, dtype=torch.float32):
    """Distinct logits per token, 1/16 apart (exact in BF16 for E <= 128, distinct scores in FP32)."""
    rng = np.random.default_rng(seed)
    x = np.stack([rng.permutation(E) for _ in range(T)]) / 16.0 - E / 32.0
    return torch.tensor(x, dtype=dtype, device=DEV)


def check(x, topk, bias=None, **kw):
    ids, w = route_experts(x, topk, bias=None if bias is None else torch.tensor(bias, dtype=torch.float32, device=DEV), **kw)
    want_ids, want_w = reference(x.float().cpu().numpy(), topk, bias=bias, **kw)
    assert ids.dtype == torch.int32 and w.dtype == torch.float32 and ids.shape == w.shape == want_ids.shape
    assert np.array_equal(ids.cpu().numpy(), want_ids)
    got = w.cpu().numpy().astype(np.float64)
    assert (np.abs(got - want_w) <= TOL * np.abs(want_w) + 1e-37).all()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,topk", [(1, 64, 6), (3, 8, 8), (7, 1, 1), (9, 33, 5), (300, 60, 4), (5, 100, 32), (33, 160, 6),
                                      (17, 256, 8), (2, 257, 8), (4, 512, 16), (5000, 64, 6)])
def test_topk(T, E, topk, score):
    # 1/16 apart over at most 256 values keeps |l - max| <= 16; a sigmoid saturates past 16 instead
    x = grid_logits(T, E, T + E) / max(1, E // 128)
    check(x, topk, score=score)
    check(x, topk, score=score, renormalize=True, scaling=2.5, n_forced=2)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("group_score", ["max", "top2"])
@pytest.mark.parametrize("T,E,n_group,topk_group,topk", [(1, 64, 8, 3, 6), (40, 160, 8, 3, 6), (33, 256, 8, 4, 8), (5, 60, 4, 1, 15),
                                                         (6, 96, 32, 2, 5), (11, 12, 12, 5, 5), (3, 512, 16, 16, 9), (9, 40, 5, 2, 7)])
def test_groups(T, E, n_group, topk_group, topk, group_score, score):
    x = grid_logits(T, E, 7 * T + E) / max(1, E // 64)
    check(x, topk, score=score, n_group=n_group, topk_group=topk_group, group_score=group_score, renormalize=True)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_bias_orders_but_does_not_weigh(score):
    rng = np.random.default_rng(4)
    x = grid_logits(50, 64, 3) / 2
    # sixteenths of the smallest score gap: the order of c is the same in 32 and 64 bits
    bias = np.round(rng.normal(size=64) * 64) / 64
    check(x, 6, bias=bias, score=score, n_group=8, topk_group=4, group_score="top2", renormalize=True, scaling=2.5)
    check(x, 6, bias=np.where(np.arange(64) < 32, -np.inf, 0.0), score=score)


def test_bf16_logits_and_strides():
    big = grid_logits(40, 100, 8, torch.bfloat16)
    for x in (big, big[:, 3:99], big[::2, 1:65], big[:1, :64].expand(9, 64)):
        check(x, 6)
    one = grid_logits(40, 65, 9)[:, 1:]
    check(one, 6, score="sigmoid", n_group=8, topk_group=2)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_ties_go_to_the_lowest_index(score):
    for E in (8, 64, 100, 256):
        x = torch.zeros(3, E, device=DEV)
        x[1, E // 2:] = 1.0
        x[2, ::3] = -1.0
        check(x, 8, score=score)
    x = torch.zeros(2, 64, device=DEV)
    x[1, 40] = x[1, 8] = 2.0
    check(x, 6, score=score, n_group=8, topk_group=3)
    check(x, 6, score=score, n_group=8, topk_group=3, group_score="top2")


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_infinities_and_nan(score):
    inf, nan = float("inf"), float("nan")
    x = grid_logits(7, 64, 11) / 4
    x[0, 5:] = -inf                       # fewer experts than topk have a score
    x[1] = -inf                           # none has
    x[2, 7] = nan
    x[3] = nan
    x[4, 9] = inf
    x[5, ::8] = torch.finfo(torch.float32).min
    if score == "softmax":
        x[4, 33] = inf                    # they share the probability
    for kw in ({}, dict(renormalize=True), dict(n_group=8, topk_group=4), dict(n_group=8, topk_group=4, group_score="top2")):
        check(x, 6, score=score, **kw)


def test_outputs_no_tokens_and_refusals():
    x = grid_logits(4, 64, 1)
    ids, w = torch.empty(4, 8, dtype=torch.int32, device=DEV), torch.empty(4, 8, device=DEV)
    got = route_experts(x, 6, n_forced=2, ids=ids, weights=w)
    assert got[0] is ids and got[1] is w and torch.equal(ids, route_experts(x, 6, n_forced=2)[0])
    assert route_experts(x[:0], 6)[0].shape == (0, 6)
    for bad in (lambda: route_experts(x.t(), 2), lambda: route_experts(x[0], 2), lambda: route_experts(x, 6, ids=ids),
                lambda: route_experts(x, 6, bias=torch.zeros(63, device=DEV)), lambda: route_experts(x, 6, bias=torch.zeros(64)),
                lambda: route_experts(x, 6, weights=w.double())):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        route_experts(x.half(), 6)
    from fleet.mk import MkError
    for kw in (dict(topk=0), dict(topk=33), dict(topk=6, n_group=5), dict(topk=20, n_group=8, topk_group=2), dict(topk=6, n_forced=-1)):
        with pytest.raises((MkError, RuntimeError)):
            route_experts(x, **kw)
