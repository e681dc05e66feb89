"""Linear layers in 8-bit integers (ffai_amd.int8) against their definition. The quantization and
the integer sums are exact, so f32 results without a bias are equal bit for bit; with one, the
oracle's fused sum is rounded twice (f64, then f32), which can differ by one f32 step; 16-bit
results are the f32 ones rounded once."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from ffai_amd import _lib as L
from ffai_amd.int8 import Int8Linear, QuantizedRows, plan_info, quantize_rows
from oracle import int8 as oracle8

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def rand(gpu, *shape, seed=0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp(0.7 * torch.randn(shape[-1], generator=g))
    return x.to(dtype).to(gpu)


def layer(gpu, n, k, bias, seed=1):
    g = torch.Generator().manual_seed(seed)
    w = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8)
    s = torch.rand(n, generator=g) * 0.01 + 1e-4
    b = torch.randn(n, generator=g) if bias else None
    lin = Int8Linear.from_quantized(w.to(gpu), s.to(gpu), None if b is None else b.to(gpu))
    return lin, w.numpy(), s.numpy(), None if b is None else b.numpy()


def same(got, want, bias):
    """got: a tensor; want: the oracle's f32 values."""
    w = torch.from_numpy(want)
    g = got.cpu()
    if bias:
        low, high = (torch.from_numpy(np.nextafter(want, np.float32(v), dtype=np.float32))
                     for v in (-np.inf, np.inf))
        ok = (g == w.to(g.dtype)) | (g == low.to(g.dtype)) | (g == high.to(g.dtype))
    else:
        ok = g == w.to(g.dtype)
    ok |= torch.isnan(g) & torch.isnan(w)
    assert ok.all(), (~ok).nonzero()[:4]


@pytest.mark.parametrize("x", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,dim", [(1, 1), (3, 7), (5, 128), (2, 129), (7, 1000), (4, 2049),
                                      (3, 4100), (2, 8192), (2, 8200), (1025, 96), (1030, 515),
                                      (1025, 1031), (1026, 2050), (1025, 4099), (1027, 8193)])
def test_quantized_rows(gpu, x, rows, dim):
    t = rand(gpu, rows, dim, seed=rows, dtype=DT[x])
    if rows > 2:
        t[1] = 0
        t[2, 0] = 1e-3 if dim == 1 else 77.0
    qr = quantize_rows(t)
    q, s = oracle8.quantize_rows(t.float().cpu().numpy())
    assert qr.q.shape[1] % 128 == 0
    assert np.array_equal(qr.scale.cpu().numpy(), s)
    assert np.array_equal(qr.q[:, :dim].cpu().numpy(), q)
    assert not qr.q[:, dim:].any()


def test_halves_small_and_non_finite_rows(gpu):
    """Quotients that are exact halves go to the even integer; subnormal rows; infinities, NaN."""
    x = torch.zeros(8, 300)
    x[0, :255] = torch.arange(-127, 128) / 2.0 * 2
    x[0, 255] = 127.0
    x[1, :254] = torch.arange(-127, 127) + 0.5
    x[1, 254] = 127.0
    x[2] = 1e-41
    x[2, 5] = -3e-41
    x[3, 7] = float("inf")
    x[3, 8] = 3.0
    x[4, 9] = float("nan")
    x[5, 11], x[5, 12] = float("-inf"), float("nan")
    x[6] = 3.0e38
    x[7, 299] = -1e-45
    qr = quantize_rows(x.to(gpu))
    q, s = oracle8.quantize_rows(x.numpy())
    np.testing.assert_array_equal(qr.scale.cpu().numpy(), s)
    assert np.array_equal(qr.q[:, :300].cpu().numpy(), q)
    lin, w, sw, _ = layer(gpu, 33, 300, False)
    same(lin(x.to(gpu)), oracle8.linear(q, s, w, sw), False)


@pytest.mark.parametrize("rows,dim", [(9, 5000), (1030, 4096), (3, 16384)])
def test_quotients_next_to_a_half(gpu, rows, dim):
    """Rows whose quotients lie on halves, some units in the last place off them, and 1e-5 to 1e-4
    off: which integer each goes to is the division's."""
    g = np.random.default_rng(dim)
    top = np.float32(1) + g.random((rows, 1), dtype=np.float32)
    s = top * (np.float32(1) / np.float32(127))
    half = g.integers(-127, 127, (rows, dim)).astype(np.float32) + np.float32(0.5)
    x = (half * s).astype(np.float32)
    ulps = g.integers(-3, 4, (rows, dim)).astype(np.int32)
    x = (x.view(np.int32) + ulps).view(np.float32)
    x[:, 1::3] += (g.uniform(-1e-4, 1e-4, (rows, dim)).astype(np.float32) * s)[:, 1::3]
    x[:, :1] = top
    qr = quantize_rows(torch.from_numpy(x).to(gpu))
    q, scale = oracle8.quantize_rows(x)
    assert np.array_equal(qr.scale.cpu().numpy(), scale)
    assert np.array_equal(qr.q[:, :dim].cpu().numpy(), q)
    lin, w, sw, b = layer(gpu, 33, dim, False)
    for m in (1, 3, rows):  # and where they are quantized inside the product
        same(lin(torch.from_numpy(x[:m]).to(gpu)), oracle8.linear(q[:m], scale[:m], w, sw), False)


SIZES = [(1, 1, 1), (1, 128, 32), (2, 100, 31), (5, 1024, 1024), (16, 640, 48), (17, 130, 65),
         (1, 2081, 100), (16, 4000, 33), (16, 4100, 40), (3, 9001, 17), (1, 65408, 20), (2, 40000, 20),
         (33, 257, 70), (64, 128, 64), (65, 129, 63), (100, 1000, 130), (130, 64, 700),
         (300, 2100, 129), (257, 512, 257)]


@pytest.mark.parametrize("m,k,n", SIZES)
@pytest.mark.parametrize("x,out,bias", [("f32", "f32", False), ("bf16", "bf16", True),
                                        ("f16", "f16", False), ("bf16", "f32", True),
                                        ("f32", "f16", True)])
def test_against_the_definition(gpu, m, k, n, x, out, bias):
    t = rand(gpu, m, k, seed=m + k, dtype=DT[x])
    lin, w, sw, b = layer(gpu, n, k, bias)
    q, s = oracle8.quantize_rows(t.float().cpu().numpy())
    got = lin(t, out_dtype=DT[out])
    assert got.dtype == DT[out] and got.shape == (m, n)
    same(got, oracle8.linear(q, s, w, sw, b), bias)


@pytest.mark.parametrize("m,k,n", [(2000, 96, 2100), (4100, 200, 4099), (8200, 32, 2049),
                                   (700, 5000, 1300), (24000, 130, 70)])
def test_large_grids(gpu, m, k, n):
    """Every tile shape, with ragged last tiles on both sides."""
    t = rand(gpu, m, k, seed=3, dtype=torch.bfloat16)
    lin, w, sw, b = layer(gpu, n, k, True)
    q, s = oracle8.quantize_rows(t.float().cpu().numpy())
    got = lin(t, out_dtype=torch.float32).cpu()
    rows = np.r_[0:3, m // 2:m // 2 + 40, m - 40:m]
    same(got[rows], oracle8.linear(q[rows], s[rows], w, sw, b), True)
    cols = np.r_[0:3, n - 30:n]
    same(got[:, cols], oracle8.linear(q, s, w[cols], sw[cols], b[cols]), True)


def test_largest_sums(gpu):
    """The longest row that 32-bit sums hold, every product at its largest."""
    k = 131072
    x = torch.ones(3, k, device=gpu)
    x[1] = -1
    w = torch.full((5, k), 127, dtype=torch.int8, device=gpu)
    lin = Int8Linear.from_quantized(w, torch.ones(5, device=gpu))
    got = lin(x).cpu().numpy()
    one = np.float32(127 * 127 * k) * np.float32(np.float32(1) / np.float32(127))
    assert np.array_equal(got, np.float32([[one] * 5, [-one] * 5, [one] * 5]))


def test_rows_do_not_depend_on_their_batch(gpu):
    """A row's result is the same bits alone and in any batch (other tiles run)."""
    t = rand(gpu, 3000, 640, seed=5, dtype=torch.float16)
    lin, *_ = layer(gpu, 900, 640, True)
    whole = lin(t)
    for a, b in ((0, 1), (7, 20), (100, 165), (2000, 2300), (5, 1005)):
        assert torch.equal(lin(t[a:b]), whole[a:b])


def test_strides_and_shapes(gpu):
    """Rows of a wider buffer, three-dimensional x, an out that is a slice of a larger one."""
    lin, w, sw, b = layer(gpu, 70, 200, True)
    wide = rand(gpu, 40, 777, seed=7, dtype=torch.float16)
    x = wide[:, 3:203]  # off every vector alignment
    q, s = oracle8.quantize_rows(x.float().cpu().numpy())
    want = oracle8.linear(q, s, w, sw, b)
    same(lin(x), want, True)
    same(lin(x.reshape(4, 10, 200)).reshape(40, 70), want, True)
    same(lin(x.unflatten(0, (5, 8)).transpose(0, 1)).transpose(0, 1).reshape(40, 70), want, True)
    held = torch.full((40, 100), 9.0, device=gpu)
    out = held[:, 11:81]
    assert lin(x, out=out) is out
    same(out, want, True)
    assert (held[:, :11] == 9).all() and (held[:, 81:] == 9).all()
    # weights off 16 bytes are copied into rows that are not
    odd = Int8Linear.from_quantized(torch.from_numpy(w).to(gpu)[:, 1:], lin.scale)
    q2, s2 = oracle8.quantize_rows(x[:, 1:].float().cpu().numpy())
    same(odd(x[:, 1:]), oracle8.linear(q2, s2, w[:, 1:], sw), False)


def test_empty_and_shared_rows(gpu):
    lin, w, sw, b = layer(gpu, 40, 96, True)
    assert lin(torch.empty(0, 96, device=gpu)).shape == (0, 40)
    x = rand(gpu, 6, 96, seed=9)
    qr = quantize_rows(x)
    assert torch.equal(lin(qr), lin(x))  # several layers may share the quantized rows
    cut = QuantizedRows(qr.q[2:5], qr.scale[2:5], 96)
    assert torch.equal(lin(cut, out_dtype=torch.float16), lin(x, out_dtype=torch.float16)[2:5])
    one = x[:1].expand(4, 96)  # one row many times
    assert torch.equal(lin(one), lin(x[:1]).expand(4, 40))


def test_weights_quantized_here(gpu):
    """Int8Linear(weight): its weights are the oracle's, and the layer stays near the f32 one: each
    factor is off by at most half a step of its row's largest / 127."""
    x, wt = rand(gpu, 9, 333, seed=11), rand(gpu, 50, 333, seed=12)
    lin = Int8Linear(wt)
    q, s = oracle8.quantize_rows(wt.cpu().numpy())
    assert np.array_equal(lin.qw[:, :333].cpu().numpy(), q)
    assert np.array_equal(lin.scale.cpu().numpy(), s)
    qx, sx = oracle8.quantize_rows(x.cpu().numpy())
    same(lin(x), oracle8.linear(qx, sx, q, s), False)
    xd, wd = x.double().cpu().numpy(), wt.double().cpu().numpy()
    hx, hw = sx[:, None].astype(float) / 2, s[:, None].astype(float) / 2
    tol = hx * np.abs(wd).sum(1)[None] + np.abs(xd).sum(1)[:, None] * hw.T + 333 * hx * hw.T
    assert (np.abs(lin(x).double().cpu().numpy() - xd @ wd.T) <= tol * 1.001).all()


def test_streams_and_graph_replays(gpu):
    lin, w, sw, b = layer(gpu, 130, 300, True)
    x = rand(gpu, 20, 300, seed=13)
    first = lin(x)
    torch.cuda.synchronize()
    outs = []
    for s in [torch.cuda.Stream() for _ in range(2)] * 3:
        with torch.cuda.stream(s):
            outs.append(lin(x))
    torch.cuda.synchronize()
    assert all(torch.equal(first, o) for o in outs)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = lin(x)
        graphs.append((g, y))
    for i in range(4):
        x.copy_(torch.randn_like(x))
        g, y = graphs[i % 2]
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, lin(x))


def test_short_workspace_is_refused(gpu):
    lin, *_ = layer(gpu, 40, 96, False)
    x = rand(gpu, 22, 96)
    n = lin.workspace_bytes(22)
    lin(x, workspace=torch.empty(n, dtype=torch.uint8, device=gpu))
    with pytest.raises(L.FfaiError, match="workspace"):
        lin(x, workspace=torch.empty(n - 1, dtype=torch.uint8, device=gpu))


def test_rows_past_32_bit_offsets(gpu):
    """y and x whose last rows lie past 2^31 elements from the first."""
    m, k, n = 3, 256, 64
    x = torch.empty(m, 1 << 30, dtype=torch.float16, device=gpu)[:, :k]
    x.copy_(rand(gpu, m, k, seed=15))
    y = torch.empty(m, (1 << 30) + 64, dtype=torch.float16, device=gpu)[:, :n]
    lin, w, sw, b = layer(gpu, n, k, False)
    lin(x, out=y)
    q, s = oracle8.quantize_rows(x.float().cpu().numpy())
    same(y, oracle8.linear(q, s, w, sw), False)


def test_tiles_cover_the_grid():
    for m, k, n in SIZES + [(24000, 5120, 1280), (1500, 1280, 3840)]:
        p = plan_info(m, k, n)
        assert p["workgroups"] >= -(-m // p["tile_rows"]) * -(-n // p["tile_outputs"])


@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m,k,n,tile", [(3900, 200, 4010, 256), (2500, 130, 1030, 128),
                                        (600, 300, 1030, 64)])
def test_every_tile_into_every_type(gpu, m, k, n, tile, out):
    """Ragged on both sides, y with rows of a larger buffer whose other elements stay."""
    assert plan_info(m, k, n)["tile_rows"] == tile
    t = rand(gpu, m, k, seed=8, dtype=torch.float16)
    lin, w, sw, b = layer(gpu, n, k, True)
    y = torch.full((m, n + 5), 7.0, dtype=DT[out], device=gpu)
    lin(t, out=y[:, 3:3 + n])
    q, s = oracle8.quantize_rows(t.float().cpu().numpy())
    same(y[:, 3:3 + n], oracle8.linear(q, s, w, sw, b), True)
    assert (y[:, :3] == 7).all() and (y[:, 3 + n:] == 7).all()


def test_many_rows_past_32_bit_offsets(gpu):
    m, k, n, stride = 20, 256, 64, 1 << 27
    x = torch.empty(m, stride, dtype=torch.float16, device=gpu)[:, :k]
    x.copy_(rand(gpu, m, k, seed=16))
    y = torch.empty(m, stride + 64, dtype=torch.float16, device=gpu)[:, :n]
    lin, w, sw, b = layer(gpu, n, k, True)
    lin(x, out=y)
    q, s = oracle8.quantize_rows(x.float().cpu().numpy())
    same(y, oracle8.linear(q, s, w, sw, b), True)


def test_few_rows_on_streams_and_in_graphs(gpu):
    lin, w, sw, b = layer(gpu, 130, 2300, True)
    x = rand(gpu, 7, 2300, seed=17)
    first = lin(x)
    torch.cuda.synchronize()
    outs = []
    for s in [torch.cuda.Stream() for _ in range(2)] * 3:
        with torch.cuda.stream(s):
            outs.append(lin(x))
    torch.cuda.synchronize()
    assert all(torch.equal(first, o) for o in outs)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = lin(x)
    for i in range(3):
        x.copy_(torch.randn_like(x))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, lin(x))


def test_scales_are_the_devices_amax_over_127(gpu):
    """Weights quantized by elementary device operations have the same scales and integers."""
    w = rand(gpu, 3000, 700, seed=23)
    qr = quantize_rows(w)
    s = w.abs().amax(1) / 127
    assert torch.equal(qr.scale, s)
    assert torch.equal(qr.q[:, :700].float(), torch.round(w / s[:, None]))
