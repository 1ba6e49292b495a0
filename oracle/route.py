"""Expert routing in 64 bits on numpy (test infrastructure, not product).

The reference has no routing code; the rules are those that include/mosaicist_sm100a.h states for
msc_moe_route and msc_moe_route_backward.
"""

from __future__ import annotations

import numpy as np


def scores(logits: np.ndarray, score: str) -> np.ndarray:
    """(T, E) -> (T, E) float64; NaN counts as -inf, an infinite maximum leaves only its equals."""
    x = np.where(np.isnan(logits.astype(np.float64)), -np.inf, logits.astype(np.float64))
    with np.errstate(over="ignore", invalid="ignore", divide="ignore"):
        if score == "sigmoid":
            return 1.0 / (1.0 + np.exp(-x))
        mx = x.max(axis=1, keepdims=True)
        e = np.where(x == mx, np.where(np.isneginf(x), 0.0, 1.0), np.exp(x - mx))
        e = np.where(np.isneginf(x), 0.0, e)
        total = e.sum(axis=1, keepdims=True)
        return np.where(total > 0, e / np.where(total > 0, total, 1.0), 0.0)


def route(logits, topk, score="softmax", bias=None, groups=1, topk_groups=1, group_top=1, renormalize=True, scale=1.0):
    """-> ids (T, topk) int32, weights (T, topk) float64."""
    T, E = logits.shape
    s = scores(logits, score)
    b = np.zeros(E) if bias is None else bias.astype(np.float64)
    by_logit = bias is None and (group_top == 1 or topk_groups == groups)
    x = np.where(np.isnan(logits.astype(np.float64)), -np.inf, logits.astype(np.float64))
    key = x.copy() if by_logit else s + b      # without a bias scores are in the order of the logits
    barred = np.isneginf(x) | np.isnan(b) | np.isneginf(b)
    key[barred] = -np.inf
    ids, weights = np.zeros((T, topk), np.int32), np.zeros((T, topk))
    per = E // groups
    for t in range(T):
        k = key[t].copy()
        if topk_groups < groups:
            best = -np.sort(-k.reshape(groups, per), axis=1)[:, :group_top]
            strength = np.where(np.isneginf(best).any(axis=1), -np.inf, best.sum(axis=1))
            kept = np.argsort(-strength, kind="stable")[:topk_groups]
            out = np.ones(groups, bool)
            out[kept] = False
            k[np.repeat(out, per)] = -np.inf
        ids[t] = np.argsort(-k, kind="stable")[:topk]
        w = np.where(np.isneginf(k[ids[t]]), 0.0, s[t, ids[t]])
        if renormalize:
            w = w / w.sum() if w.sum() > 0 else np.zeros_like(w)
        weights[t] = w * scale
    return ids, weights


def weights_of(logits, ids, score, renormalize, scale):
    """The weights as a function of the logits for a given choice (what the gradient is of)."""
    w = np.take_along_axis(scores(logits, score), ids, axis=1)
    return (w / w.sum(axis=1, keepdims=True) if renormalize else w) * scale


def route_backward(grad, logits, ids, weights, score, renormalize, scale):
    """Gradient of sum(grad * weights) by the logits, float64; weights of 0 do not move."""
    s = scores(logits, score)
    w = weights.astype(np.float64)
    g = np.where(w == 0, 0.0, grad.astype(np.float64))
    total = (g * w).sum(axis=1, keepdims=True)
    c = w * (g - total / scale) if renormalize else w * g
    if score == "sigmoid":
        c = c * (1.0 - np.take_along_axis(s, ids, axis=1))
    out = np.zeros_like(s)
    if score == "softmax" and not renormalize:
        out = -s * total
    for k in range(ids.shape[1]):
        out[np.arange(len(ids)), ids[:, k]] += c[:, k]
    return out
