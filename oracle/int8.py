"""Linear layers in 8-bit integers, restated in numpy from the definition: the check for
ffai_amd.int8. Scales are the largest magnitude times the f32 number nearest to 1 / 127, quotients
IEEE f32, sums exact integers, the rest in f32 step by step."""

from __future__ import annotations

import numpy as np


def quantize_rows(x):
    """x (rows, dim) f32 -> (q int8, scale f32)."""
    x = np.asarray(x, np.float32)
    top = np.abs(x).max(axis=1) if x.shape[1] else np.zeros(len(x), np.float32)
    with np.errstate(all="ignore"):
        s = np.where(top == 0, np.float32(1), top * (np.float32(1) / np.float32(127))).astype(np.float32)
        r = np.rint(x / s[:, None])  # numpy's rint rounds halves to even
        q = np.where(np.isnan(r), 0, np.clip(r, -127, 127)).astype(np.int8)
    return q, s


def linear(q, s, w, w_scale, bias=None):
    """y in f32: acc * s and its product with w_scale each rounded, except that a bias joins the
    second product in one rounding (as float64, whose own rounding is 2^-29 of that)."""
    acc = q.astype(np.int64) @ w.astype(np.int64).T
    with np.errstate(all="ignore"):
        t = acc.astype(np.float32) * s[:, None]
        if bias is None:
            return t * w_scale[None]
        y = t.astype(np.float64) * w_scale[None].astype(np.float64) + bias[None].astype(np.float64)
        return y.astype(np.float32)
