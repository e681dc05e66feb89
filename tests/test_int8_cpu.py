"""What the 8-bit linear layers refuse, and their oracle: no GPU needed (nothing is launched)."""

from __future__ import annotations

import ctypes
import re

import numpy as np
import pytest
import torch

from ffai_amd import _lib as L
from ffai_amd import int8
from oracle import int8 as oracle8

OK = dict(x=4096, x_dtype=L.F32, xs=256, rows=4, dim=256, w=4096, ws=256, sw=4096, bias=4096, n=8,
          y=4096, y_dtype=L.F32, ys=8, work=4096, work_bytes=1 << 40)


def linear(**edit):
    a = dict(OK, **edit)
    rc = L.load().ffai_int8_linear(a["x"], a["x_dtype"], a["xs"], a["rows"], a["dim"], a["w"],
                                   a["ws"], a["sw"], a["bias"], a["n"], a["y"], a["y_dtype"],
                                   a["ys"], a["work"], a["work_bytes"], None)
    return rc, L.last_error()


def product(**edit):
    a = dict(OK, **edit)
    rc = L.load().ffai_int8_product(a["x"], a["xs"], a.get("sx", 4096), a["rows"], a["dim"], a["w"],
                                    a["ws"], a["sw"], a["bias"], a["n"], a["y"], a["y_dtype"],
                                    a["ys"], None)
    return rc, L.last_error()


WEIGHTS = [
    (dict(w=0), "null"), (dict(sw=0), "null"), (dict(y=0), "null"), (dict(n=0), "out_dim"),
    (dict(n=(1 << 28) + 1), "out_dim"), (dict(w=4100), "16-byte"), (dict(ws=250), "multiple of 16"),
    (dict(ws=240), "in_dim"), (dict(ws=(1 << 22) + 16), "2\\^22"), (dict(sw=4097), "4-byte"),
    (dict(bias=4098), "4-byte"), (dict(y_dtype=5), "y dtype"), (dict(y=4098), "aligned"),
    (dict(ys=7), "overlap"), (dict(ys=-8), "overlap"), (dict(dim=0), "in_dim"),
    (dict(dim=131073), "in_dim"), (dict(rows=-1), "rows"),
]


@pytest.mark.parametrize("edit,why", WEIGHTS + [
    (dict(x=0), "null"), (dict(x_dtype=3), "x dtype"), (dict(x=4098), "aligned"),
    (dict(xs=255), "overlap"), (dict(xs=-1), "overlap"), (dict(work=4104), "16-byte")],
    ids=lambda v: next(iter(v)) if isinstance(v, dict) else None)
def test_linear_refuses(edit, why):
    rc, msg = linear(**edit)

    assert rc == L.FFAI_ERR_INVALID and re.search(why, msg), (rc, msg)


@pytest.mark.parametrize("edit,why", WEIGHTS + [
    (dict(x=0), "null"), (dict(sx=0), "null"), (dict(x=4100), "16-byte"), (dict(xs=272), "128"),
    (dict(xs=128), "in_dim"), (dict(xs=1 << 23), "2\\^22"), (dict(sx=4097), "4-byte")],
    ids=lambda v: next(iter(v)) if isinstance(v, dict) else None)
def test_product_refuses(edit, why):
    rc, msg = product(**edit)

    assert rc == L.FFAI_ERR_INVALID and re.search(why, msg), (rc, msg)


def test_quantize_refuses():
    q = L.load().ffai_int8_quantize_rows
    for args, why in (((4096, L.F32, 4, 256, 256, 4104, 256, 4096), "16-byte"),
                      ((4096, L.F32, 4, 256, 256, 4096, 272, 4096), "128"),
                      ((4096, L.F32, 4, 256, 256, 4096, 128, 4096), "dim"),
                      ((4096, L.F32, 4, 256, 256, 4096, 256, 4098), "4-byte"),
                      ((4096, L.F32, 4, 256, 256, 0, 256, 4096), "null"),
                      ((4096, L.F32, 4, 256, 256, 4096, 256, 0), "null"),
                      ((0, L.F32, 4, 256, 256, 4096, 256, 4096), "null"),
                      ((4096, 9, 4, 256, 256, 4096, 256, 4096), "dtype"),
                      ((4096, L.F32, 4, 256, 200, 4096, 256, 4096), "overlap")):
        assert q(*args, None) == L.FFAI_ERR_INVALID and why in L.last_error()


def test_no_rows_is_no_work():
    """Nothing is launched (this runs without a GPU) and nothing is read."""
    assert linear(rows=0, x=0, y=0, work=0)[0] == L.FFAI_OK
    assert product(rows=0, x=0, y=0, sx=0)[0] == L.FFAI_OK
    assert L.load().ffai_int8_quantize_rows(None, L.F32, 0, 5, 5, None, 0, None, None) == L.FFAI_OK


def test_workspace():
    rc, msg = linear(rows=20, work=0)
    assert rc == L.FFAI_ERR_WORKSPACE and "workspace" in msg
    n = ctypes.c_size_t()
    assert L.load().ffai_int8_linear_workspace_bytes(50, 129, ctypes.byref(n)) == L.FFAI_OK
    assert n.value == 50 * 256 + 208
    assert linear(rows=50, dim=129, xs=129, work_bytes=n.value - 1)[0] == L.FFAI_ERR_WORKSPACE
    # few rows are quantized where they are used, unless they are too long for that
    for rows, dim, none in ((1, 1, True), (16, 1024, True), (17, 1024, False), (16, 4080, False),
                            (1, 65408, True), (1, 65536, False)):
        assert L.load().ffai_int8_linear_workspace_bytes(rows, dim, ctypes.byref(n)) == L.FFAI_OK
        assert (n.value == 0) == none, (rows, dim, n.value)


def test_binding_refuses():
    w, s = torch.zeros(8, 32, dtype=torch.int8), torch.ones(8)
    lin = int8.Int8Linear.from_quantized(w, s)
    assert lin.qw.data_ptr() == w.data_ptr()
    for bad, why in (((w.float(), s), "int8"), ((w, s[:7]), "one value per row"),
                     ((w, s.double()), "f32"), ((w[0], s), "int8")):
        with pytest.raises(ValueError, match=why):
            int8.Int8Linear.from_quantized(*bad)
    with pytest.raises(ValueError, match="bias"):
        int8.Int8Linear.from_quantized(w, s, torch.zeros(3))
    with pytest.raises(ValueError, match="must be"):
        lin(torch.zeros(4, 31))
    with pytest.raises(ValueError, match="f32, f16"):
        lin(torch.zeros(4, 32, dtype=torch.int32), out_dtype=torch.float32)
    with pytest.raises(ValueError, match="HIP device"):
        lin(torch.zeros(4, 32))
    with pytest.raises(ValueError, match="HIP device"):
        int8.quantize_rows(torch.zeros(4, 32))
    qr = int8.QuantizedRows(torch.zeros(4, 64, dtype=torch.int8), torch.ones(4), 32)
    with pytest.raises(ValueError, match="quantize_rows"):
        lin(qr)  # rows not padded to 128
    with pytest.raises(ValueError, match="rows of 32"):
        lin(int8.QuantizedRows(torch.zeros(4, 128, dtype=torch.int8), torch.ones(4), 33))


def test_unaligned_weights_are_padded():
    w = torch.randint(-5, 5, (6, 21), dtype=torch.int8)
    lin = int8.Int8Linear.from_quantized(w, torch.ones(6))
    assert lin.qw.shape == (6, 32) and torch.equal(lin.qw[:, :21], w) and not lin.qw[:, 21:].any()


def test_oracle():
    x = np.float32([[0.5, 1.5, -2.5, 127.0], [0, 0, 0, 0]])
    q, s = oracle8.quantize_rows(x)
    assert q.tolist() == [[0, 2, -2, 127], [0, 0, 0, 0]] and s.tolist() == [1.0, 1.0]
    y = oracle8.linear(q, s, np.int8([[1, 2, 3, 4]]), np.float32([0.5]), np.float32([1]))
    assert y.tolist() == [[(4 - 6 + 508) * 0.5 + 1], [1.0]]


@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (5, 1024, 1024), (227, 1024, 4096), (1500, 1280, 3840),
                                   (24000, 5120, 1280), (1 << 20, 64, 7), (3, 64, 1 << 20)])
def test_plan(m, k, n):
    p = int8.plan_info(m, k, n)
    assert p["workgroups"] >= -(-m // p["tile_rows"]) * -(-n // p["tile_outputs"])
    assert p["waves"] in (1, 2, 4, 8, 16)
