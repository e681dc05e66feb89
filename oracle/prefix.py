"""Attention over a shared prefix and own keys, in 64 bits and straight from the definition: the
check for ffai_amd.prefix. Slot by slot, row by row; nothing is blocked, split or reordered."""

from __future__ import annotations

import numpy as np


def prefix_attend(q, pk, pv, plens, ok, ov, olens, scale):
    """q (S, Hq, T, D); pk, pv (G, H, P, D); ok, ov (S, H, C, D); lengths per group and per slot
    (clamped to the capacities). Returns (out, mean_abs, reach): the attention, the same weights
    over |v|, and per row the largest sum |q_d k_d| over the keys it sees (what a score's rounding
    is relative to), as float64 arrays."""
    q, pk, pv, ok, ov = (np.asarray(x, np.float64) for x in (q, pk, pv, ok, ov))
    s_n, hq, t_n, d = q.shape
    per = s_n // pk.shape[0]
    rep = hq // pk.shape[1]
    out = np.zeros_like(q)
    mean = np.zeros_like(q)
    reach = np.zeros(q.shape[:3])
    for s in range(s_n):
        g = s // per
        n_p = int(np.clip(plens[g], 0, pk.shape[2]))
        n_o = int(np.clip(olens[s], 0, ok.shape[2]))
        for h in range(hq):
            for t in range(t_n):
                seen = min(n_o, max(0, n_o - t_n + t + 1))
                k = np.concatenate([pk[g, h // rep, :n_p], ok[s, h // rep, :seen]])
                v = np.concatenate([pv[g, h // rep, :n_p], ov[s, h // rep, :seen]])
                if len(k) == 0:
                    continue
                z = k @ q[s, h, t] * scale
                with np.errstate(invalid="ignore"):
                    w = np.exp(z - z.max())
                    w /= w.sum()
                    out[s, h, t] = w @ v
                    mean[s, h, t] = w @ np.abs(v)
                    reach[s, h, t] = (np.abs(k) @ np.abs(q[s, h, t])).max() * scale
    return out, mean, reach
