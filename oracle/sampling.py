"""Sampling restated in numpy from its definition, in 64 bits: the check for ffai_amd.sampling.
Sorts every row; cumulative sums run in the stated orders."""

from __future__ import annotations

import numpy as np


def sample_row(l, u, t=1.0, k=0, p=1.0, mp=0.0):
    """l: one row of f32 logits; settings as f32 / int. Returns (token, logprob, kept tokens)."""
    l = np.asarray(l, np.float64).copy()
    l[np.isnan(l)] = -np.inf
    m = l.max()
    if m == -np.inf:
        return -1, -np.inf, np.array([], np.int64)

    def weights(inv):
        with np.errstate(all="ignore"):
            w = np.exp((l - m) * inv)
        w[l == -np.inf] = 0
        if m == np.inf:
            w[l < m] = 0
        w[l == m] = 1
        return w

    logz = np.log(weights(1.0).sum())

    def logprob(i):
        return (0.0 if l[i] == m else l[i] - m) - logz

    t = np.float32(t)
    if not t > 0:
        i = int(np.flatnonzero(l == m)[0])
        return i, logprob(i), np.array([i])
    w = weights(1.0 / np.float64(t))
    order = np.lexsort((np.arange(l.size), -l))
    order = order[l[order] > -np.inf]
    if k > 0:
        order = order[:k]
    mp = np.float32(mp)
    if mp > 0:
        order = order[w[order] >= min(float(mp), 1.0)]
    p = np.float32(p)
    if p < 1:
        c = np.cumsum(w[order])
        before = np.concatenate([[0.0], c[:-1]])
        order = order[:max(1, int((before < np.float64(p) * c[-1]).sum()))]
    kept = np.sort(order)
    c = np.cumsum(w[kept])
    u = np.float32(u)
    u = 0.0 if not u >= 0 else min(float(u), float(np.nextafter(np.float32(1), np.float32(0))))
    hit = np.flatnonzero((c > u * c[-1]) & (w[kept] > 0))
    i = int(kept[hit[0]]) if hit.size else int(kept[np.flatnonzero(w[kept] > 0)[-1]])
    return i, logprob(i), kept
