"""What follows a verify pass, restated on the CPU in 64 bits: sampling with
filters from given random numbers, and the walk down a drafted tree along the
sampled tokens (the accepted path that mlx-tree-spec
src/mlx_tree_spec/tree_verify.py:499-516 commits). TEST INFRASTRUCTURE ONLY.
"""

from __future__ import annotations

import numpy as np


def filtered(x, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token order, weights) of what the filters keep of one row of logits:
    tokens by (logit descending, index ascending), weights relative to the first."""
    x = np.asarray(x, dtype=np.float64)
    ids = np.flatnonzero(~np.isnan(x) & ~np.isneginf(x))
    order = ids[np.argsort(-x[ids], kind="stable")]
    if order.size == 0:
        return order, np.zeros(0)
    if not temperature > 0:
        return order[:1], np.ones(1)
    if top_k > 0:
        order = order[:top_k]
    top = x[order[0]]
    with np.errstate(invalid="ignore"):
        w = np.where(x[order] == top, 1.0, np.exp((x[order] - top) / temperature))
    if top_p < 1:
        n = max(1, int(np.searchsorted(np.cumsum(w), top_p * np.cumsum(w)[-1], side="left")) + 1)
        order, w = order[:n], w[:n]
    if min_p > 0:
        keep = w >= min_p
        keep[0] = True
        order, w = order[keep], w[keep]
    return order, w


def sample(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, log probability, margin): margin is how far u lies from the
    nearest border between two tokens' shares, so that a test can tell a wrong
    token from one that rounding of a 64-bit sum decides."""
    order, w = filtered(x, temperature, top_k, top_p, min_p)
    if order.size == 0:
        return -1, -np.inf, np.inf
    cum = np.cumsum(w) / np.sum(w)
    at = min(int(np.searchsorted(cum, min(max(float(u), 0.0), 1.0), side="right")), order.size - 1)
    return int(order[at]), float(np.log(w[at] / np.sum(w))), float(np.min(np.abs(cum - u)))


def tree_accept(tokens, parents, samples):
    """(path, next token) of one tree."""
    cur, path = 0, [0]
    while samples[cur] >= 0:
        below = [c for c in range(cur + 1, len(tokens)) if parents[c] == cur and tokens[c] == samples[cur]]
        if not below:
            break
        cur = below[0]
        path.append(cur)
    return path, int(samples[cur])
