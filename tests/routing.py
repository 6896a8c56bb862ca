"""Routing to experts in numpy, by the definition, in float64."""
import numpy as np


def scores(logits, scoring):
    x = logits.astype(np.float64)
    with np.errstate(over="ignore", invalid="ignore", divide="ignore"):
        if scoring == "sigmoid":
            return 1.0 / (1.0 + np.exp(-x))
        top = x.max(axis=1, keepdims=True)
        e = np.exp(x - np.where(top == -np.inf, 0.0, top))
        total = e.sum(axis=1, keepdims=True)
        return e / np.where(total == 0.0, 1.0, total)


def better(a, i, b, j):
    """Whether (value a, number i) goes before (b, j): numbers before NaN, larger before smaller, lower before higher."""
    if np.isnan(a) != np.isnan(b):
        return not np.isnan(a)
    if not np.isnan(a) and a != b:
        return a > b
    return i < j


def choose(choice, experts, topk, groups=1, top_groups=1, best=1):
    """ids of one token from its choice values (NaN allowed, -Inf: not there)."""
    left = [e for e in range(experts) if choice[e] != -np.inf]
    if groups > 1:
        per = experts // groups
        low = -1e300

        def group_score(g):
            v = sorted((low if np.isnan(c) else c for c in choice[g * per:(g + 1) * per]), reverse=True)
            return sum(v[:best])

        order = sorted(range(groups), key=lambda g: (-group_score(g), g))[:top_groups]
        left = [e for e in left if e // per in order]
    left.sort(key=lambda e: (np.isnan(choice[e]), 0.0 if np.isnan(choice[e]) else -choice[e], e))
    return left[:topk] + [-1] * (topk - len(left[:topk]))


def route(logits, scoring, topk, bias=None, groups=1, top_groups=1, best=1, renorm=0, scale=1.0):
    """(ids (n, topk), weights float64)."""
    n, experts = logits.shape
    p = scores(logits, scoring)
    # without a bias and with groups by their best expert the logits decide
    choice = logits.astype(np.float64) if bias is None and (groups == 1 or best == 1) else p + (0.0 if bias is None else bias)
    choice = np.where(logits == -np.inf, -np.inf, choice)
    ids = np.array([choose(choice[t], experts, topk, groups, top_groups, best) for t in range(n)], np.int32).reshape(n, topk)
    w = np.where(ids < 0, 0.0, np.take_along_axis(p, np.maximum(ids, 0), 1))
    if renorm:
        total = w.sum(axis=1, keepdims=True)
        w = w / np.where(total == 0.0, 1.0, total)
    return ids, w * scale


def order(ids, experts):
    """(offsets, places, pairs) of a stable sort by expert."""
    flat = ids.reshape(-1)
    there = (flat >= 0) & (flat < experts)
    pairs = np.full(flat.size, -1, np.int32)
    by = np.argsort(np.where(there, flat, experts), kind="stable")
    count = int(there.sum())
    pairs[:count] = by[:count]
    places = np.full(flat.size, -1, np.int32)
    places[pairs[:count]] = np.arange(count)
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat[there], minlength=experts))]).astype(np.int64)
    return offsets, places.reshape(ids.shape), pairs


def grad(logits, scoring, ids, dweights, renorm=0, scale=1.0):
    """The logits' gradient, through the weights' Jacobian."""
    n, experts = logits.shape
    p = scores(logits, scoring)
    out = np.zeros((n, experts))
    for t in range(n):
        at = [(s, e) for s, e in enumerate(ids[t]) if 0 <= e < experts]
        total = sum(p[t, e] for _, e in at) if renorm else 1.0
        total = total if total != 0.0 else 1.0
        dot = sum(dweights[t, s] * p[t, e] for s, e in at)
        dp = np.zeros(experts)
        for s, e in at:
            dp[e] += scale * (dweights[t, s] / total - (dot / total ** 2 if renorm else 0.0))
        if scoring == "sigmoid":
            out[t] = dp * p[t] * (1.0 - p[t])
        else:
            out[t] = p[t] * (dp - (dp * p[t]).sum())
    return out
