"""What sampling refuses, and its oracle: no GPU needed (nothing is launched)."""

from __future__ import annotations

import math
import re

import numpy as np
import pytest
import torch

from ffai_amd import _lib as L
from ffai_amd.sampling import sample, workspace_bytes
from oracle.sampling import sample_row

OK = dict(logits=4096, dtype=L.F32, rows=3, vocab=100, stride=100, t=0, k=0, p=0, mp=0, u=4096,
          tok=4096, lp=4096, ws=4096, ws_bytes=1 << 40)


def call(**edit):
    a = dict(OK, **edit)
    rc = L.load().ffai_sample(a["logits"], a["dtype"], a["rows"], a["vocab"], a["stride"], a["t"],
                              1.0, a["k"], 0, a["p"], 1.0, a["mp"], 0.0, a["u"], a["tok"], a["lp"],
                              a["ws"], a["ws_bytes"], None)
    return rc, L.last_error()


@pytest.mark.parametrize("edit,why", [
    (dict(logits=0), "null"), (dict(u=0), "null"), (dict(tok=0), "null"), (dict(dtype=4), "dtype"),
    (dict(rows=-1), "rows"), (dict(rows=65536), "rows"), (dict(vocab=0), "vocab"),
    (dict(vocab=(1 << 20) + 1), "vocab"), (dict(stride=-1), "stride"), (dict(logits=4098), "aligned"),
    (dict(logits=4097, dtype=L.F16), "aligned"), (dict(t=4097), "4-byte"), (dict(k=4098), "4-byte"),
    (dict(p=4098), "4-byte"), (dict(mp=4098), "4-byte"), (dict(u=4098), "4-byte"),
    (dict(tok=4098), "4-byte"), (dict(lp=4098), "4-byte"), (dict(ws=4104), "16-byte")],
    ids=lambda v: next(iter(v)) if isinstance(v, dict) else None)
def test_bad_arguments(edit, why):
    rc, msg = call(**edit)
    assert rc == L.FFAI_ERR_INVALID and re.search(why, msg), (rc, msg)


def test_workspace_and_no_rows():
    assert call(ws=0)[0] == L.FFAI_ERR_WORKSPACE
    assert call(ws_bytes=workspace_bytes(3, 100) - 1)[0] == L.FFAI_ERR_WORKSPACE
    assert call(rows=0, logits=0, u=0, tok=0, ws=0)[0] == L.FFAI_OK  # nothing is launched
    assert workspace_bytes(0, 5) == 0


def test_binding_refuses():
    l, u = torch.zeros(3, 100), torch.zeros(3)
    for args, kw, why in (((l[0], u), {}, "logits"), ((l.int(), u), {}, "logits"),
                          ((l.t().contiguous().t(), u), {}, "contiguous"),
                          ((l, u[:2]), {}, "u must"), ((l, u.double()), {}, "u must"),
                          ((l, u), dict(top_k=torch.zeros(3)), "top_k"),
                          ((l, u), dict(top_p=torch.zeros(2)), "top_p"),
                          ((l, u), dict(min_p=torch.zeros(6)[::2]), "min_p"),
                          ((l, u), dict(temperature=torch.zeros(3, dtype=torch.float64)), "temperature"),
                          ((l, u), {}, "HIP device")):
        with pytest.raises(ValueError, match=why):
            sample(*args, **kw)


def test_oracle_by_hand():
    l = np.log(np.float32([0.1, 0.4, 0.2, 0.3]))
    assert sample_row(l, 0.0)[0] == 0 and sample_row(l, 0.11)[0] == 1
    assert sample_row(l, 0.999)[0] == 3 and sample_row(l, 0.5, t=0.0)[0] == 1
    assert sample_row(l, 0.9, k=1)[0] == 1
    assert list(sample_row(l, 0.0, k=2)[2]) == [1, 3]
    assert list(sample_row(l, 0.0, p=0.6)[2]) == [1, 3]      # 0.4 < 0.6, 0.7 is not
    assert list(sample_row(l, 0.0, p=0.75)[2]) == [1, 2, 3]
    assert list(sample_row(l, 0.0, p=0.0)[2]) == [1]
    assert list(sample_row(l, 0.0, mp=0.6)[2]) == [1, 3]     # 0.3 / 0.4
    assert list(sample_row(l, 0.0, k=3, mp=0.6, p=0.5)[2]) == [1]  # 0.4 >= 0.5 * 0.7
    assert abs(sample_row(l, 0.0)[1] - math.log(0.1)) < 1e-6
    assert sample_row([-np.inf, np.nan], 0.5)[0] == -1
    assert list(sample_row([1, 1, 1, 1], 0.5, k=2)[2]) == [0, 1]
