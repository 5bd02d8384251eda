"""Float64 oracle of token sampling (include/k3_hip_sample_abi.h): one row by sorting."""
from __future__ import annotations

import numpy as np


def sample_row(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, margin): the token drawn, and how near any decision came to going the other
    way, relative to the kept weight (top-p's border, min-p's border, the draw's)."""
    l = np.asarray(logits, np.float64).copy()
    l[np.isnan(l)] = -np.inf
    top = l.max()
    if top == -np.inf:
        return -1, np.inf
    order = np.lexsort((np.arange(len(l)), -l))
    if not temperature > 0:
        return int(order[0]), np.inf
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.exp((l[order] - top) / temperature)
    w[l[order] == top] = 1.0
    w[(l[order] == -np.inf)] = 0.0
    if top == np.inf:
        w[l[order] != top] = 0.0
    mass = np.cumsum(w)
    margin = np.inf
    n = len(l)
    if 0 < top_k < n:
        n = int(top_k)
    if top_p < 1:
        want = max(top_p, 0.0) * mass[n - 1]
        n_p = 1 + int((mass[:n] < want).sum())
        if top_p > 0:
            margin = min(margin, np.abs(mass[:n] - want).min() / mass[n - 1])
        n = min(n, n_p)
    if min_p > 0:
        least = min(min_p, 1.0)
        away = np.abs(w - least)
        if least < 1:
            margin = min(margin, away.min() / least)
        n = min(n, int((w >= least).sum()))
    u = 1 - 2.0 ** -24 if not u < 1 else max(float(u), 0.0)
    target = u * mass[n - 1]
    if u > 0:
        margin = min(margin, np.abs(mass[:n] - target).min() / mass[n - 1])
    at = min(int((mass[:n] <= target).sum()), n - 1)
    return int(order[at]), margin
