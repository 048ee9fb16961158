"""Routing of a batch of tokens to experts (mk_route, csrc/mk_route.cu).

The persistent kernel's router serves its one token; this is the router of a batch, with the score
functions, balance bias, expert groups and renormalisation that checkpoints of this family name in
their configurations. Its ids and weights are what fleet.w4.W4Experts takes.
"""
import ctypes
from functools import lru_cache
from operator import index as index_of

import torch

from fleet import mk

SCORES = {"softmax": 0, "sigmoid": 1}
GROUP_SCORES = {"max": 0, "top2": 1}
LOGITS = {torch.float32: 0, torch.bfloat16: 1}


@lru_cache(maxsize=256)
def _params(experts, topk, n_forced, n_group, topk_group, group_score, score, renormalize, dtype, scaling):
    if score not in SCORES or group_score not in GROUP_SCORES:
        raise ValueError(f"score {score!r} is one of {list(SCORES)}, group_score {group_score!r} of {list(GROUP_SCORES)}")
    if dtype not in LOGITS:
        raise TypeError(f"logits are float32 or bfloat16, not {dtype}")
    p = mk.MkRoute(experts, topk, n_forced, n_group, topk_group, GROUP_SCORES[group_score], SCORES[score],
                   int(renormalize), LOGITS[dtype], scaling)
    return p, ctypes.addressof(p)


def _given(t, shape, dtype, device, name):
    if tuple(t.shape) != shape or t.dtype != dtype or not t.is_contiguous() or t.device != device:
        raise ValueError(f"{name}: contiguous {dtype} {shape} on {device} expected, got {t.dtype} {tuple(t.shape)} on {t.device}")


def route_experts(logits, topk, *, score="softmax", bias=None, n_group=1, topk_group=1, group_score="max",
                  renormalize=False, scaling=1.0, n_forced=0, ids=None, weights=None, stream=None):
    """(ids [T, topk + n_forced] int32, weights [T, topk + n_forced] float32) of logits [T, E].

    Scores are softmax(logits) or 1 / (1 + exp(-logits)) (`score`). The selection goes by the scores
    plus `bias` [E] (float32; it does not enter the weights), among the experts of the `topk_group`
    best of `n_group` equal consecutive groups, a group being as good as its best expert
    (`group_score` "max") or its two best together ("top2"). Ties go to the lowest index. Weights are
    the selected experts' scores in descending order of the selection, divided by their sum if
    `renormalize`, times `scaling`. `n_forced` always-selected experts E, E + 1, ... with weight 1
    follow (the packed weights' folded shared experts). A logit of -inf scores 0, a NaN counts as -inf.

    logits float32 or bfloat16, rows of unit stride (any row stride); E <= 512, topk <= 32. Runs on
    `stream` (default: the current stream of the tensors' device); `ids` / `weights` are written if
    given."""
    if stream is not None:
        with mk.on_stream(logits, stream, bias, ids, weights):
            return route_experts(logits, topk, score=score, bias=bias, n_group=n_group, topk_group=topk_group,
                                 group_score=group_score, renormalize=renormalize, scaling=scaling, n_forced=n_forced,
                                 ids=ids, weights=weights)
    if logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError(f"logits [T, E] with unit stride along E expected, got {tuple(logits.shape)}, strides {logits.stride()}")
    T, E = logits.shape
    topk, n_forced = index_of(topk), index_of(n_forced)
    # plain numbers (a tensor would be cached by its identity), held until the call is over: the cache may drop
    # them meanwhile
    params = _params(E, topk, n_forced, index_of(n_group), index_of(topk_group), group_score, score, bool(renormalize),
                     logits.dtype, float(scaling))
    call, device, current_stream, context = mk.entry("mk_route")
    index = logits.get_device()
    if index < 0 or device() != index:
        return mk.off_device("mk_route", index, context, lambda: route_experts(
            logits, topk, score=score, bias=bias, n_group=n_group, topk_group=topk_group, group_score=group_score,
            renormalize=renormalize, scaling=scaling, n_forced=n_forced, ids=ids, weights=weights))
    b = 0
    if bias is not None:
        if (bias.dtype is not torch.float32 or bias.shape != (E,) or not bias.is_contiguous() or bias.get_device() != index):
            raise ValueError(f"bias: contiguous float32 [{E}] on {logits.device} expected, got {bias.dtype} {tuple(bias.shape)} on {bias.device}")
        b = bias.data_ptr()
    k = topk + n_forced
    shape = (T, k)
    if ids is None:
        ids = torch.empty_strided(shape, (k, 1), dtype=torch.int32, device=logits.device)
    else:
        _given(ids, shape, torch.int32, logits.device, "ids")
    if weights is None:
        weights = torch.empty_strided(shape, (k, 1), dtype=torch.float32, device=logits.device)
    else:
        _given(weights, shape, torch.float32, logits.device, "weights")
    rc = call(params[1], logits.data_ptr(), logits.stride(0), T, b, ids.data_ptr(), weights.data_ptr(), current_stream(index))
    if rc:
        mk._check(rc, "mk_route")
    return ids, weights
