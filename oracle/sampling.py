"""Plain statement of the sampler, in 64 bits on the CPU (numpy)."""

from __future__ import annotations

import numpy as np


def sample(row, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """-> (token, probability, slack, kept): the token of one row of logits, how far the nearest decision was from falling
    otherwise, relative to the kept weight (min-p's to the largest), and the kept weight, the largest weight being 1."""
    row = np.where(np.isnan(row), -np.inf, np.asarray(row, dtype=np.float64))
    order = np.argsort(-row, kind="stable")
    top = row[order[0]]
    if top == -np.inf:
        return -1, 0.0, 1.0, 0.0
    if not temperature > 0:
        return int(order[0]), 1.0, 1.0, 1.0
    with np.errstate(all="ignore"):
        x = np.where(row[order] == top, 0.0, (row[order] - top) / np.float64(temperature))
        w = np.exp(np.where(np.isnan(x), -np.inf, x))
    w = w[w > 2.0 ** -42]
    slack = float(np.min(np.abs(w - min_p))) if 0 < min_p < 1 else 1.0
    w = w[w >= min(min_p, 1.0)]
    if top_k > 0:
        w = w[:top_k]
    acc = np.cumsum(w)
    if top_p < 1:
        slack = min(slack, float(np.min(np.abs(acc[:-1] - top_p * acc[-1]), initial=1.0)) / acc[-1])
        w = w[:max(1, int(np.searchsorted(acc, top_p * acc[-1], side="left")) + 1)]
        acc = np.cumsum(w)
    slack = min(slack, float(np.min(np.abs(acc[:-1] - u * acc[-1]), initial=1.0)) / acc[-1])
    at = min(int(np.searchsorted(acc, u * acc[-1], side="right")), len(w) - 1)
    return int(order[at]), float(w[at] / acc[-1]), slack, float(acc[-1])
