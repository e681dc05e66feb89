"""Sampling (ffai_amd.sampling) against its definition in 64 bits: tokens are equal. The
log-probability is an f32 number from a sum of n f32 exponentials (each within 2^-22 of its own
value, and of exponents off by up to |l - m| 2^-23), so log of it is off by at most
(4 + 2 * 30) 2^-24 + 2^-40 for terms that matter (those further than 30 below the maximum weigh
less than n e^-30), and rounded once: 2^-18 + 2^-24 |logprob| + n e^-30."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from ffai_amd import _lib as L
from ffai_amd.sampling import sample, workspace_bytes
from oracle.sampling import sample_row

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def per_row(x, r):
    return x if not isinstance(x, torch.Tensor) else x[r].item()


def check(logits, u, got=None, t=None, k=None, p=None, mp=None):
    if got is None:
        got = sample(logits, u, temperature=t, top_k=k, top_p=p, min_p=mp)
    tok, lp = (x.cpu().numpy() for x in got)
    rows = logits.float().cpu().numpy()
    uu = u.cpu().numpy()
    for r in range(len(rows)):
        want, wlp, kept = sample_row(rows[r], uu[r], 1.0 if t is None else per_row(t, r),
                                     0 if k is None else per_row(k, r),
                                     1.0 if p is None else per_row(p, r),
                                     0.0 if mp is None else per_row(mp, r))
        assert tok[r] == want, (r, tok[r], want, len(kept))
        if want < 0:
            assert lp[r] == -np.inf
        else:
            tol = 2.0 ** -18 + 2.0 ** -24 * abs(wlp) + rows.shape[1] * math.exp(-30)
            assert abs(lp[r] - wlp) <= tol, (r, lp[r], wlp)


def make(gpu, rows, vocab, sigma=2.5, seed=0, dtype=torch.float32, low=0.03):
    g = torch.Generator().manual_seed(seed)
    l = torch.randn(rows, vocab, generator=g) * sigma
    if low:
        l[torch.rand(rows, vocab, generator=g) < low] = -math.inf
        l[:, vocab // 2] = 1.0
    return l.to(dtype).to(gpu), torch.rand(rows, generator=g).to(gpu)


VOCABS = [1, 2, 3, 4, 5, 7, 8, 9, 63, 1000, 4095, 4096, 4097, 8193, 51865]


@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kw", [dict(), dict(t=0.3), dict(t=0.0), dict(k=1), dict(k=40, p=0.8),
                                dict(p=0.9), dict(mp=0.05, t=1.7), dict(k=300, p=0.95, mp=1e-4)],
                         ids=lambda k: "-".join(k) or "plain")
def test_against_the_definition(gpu, vocab, dtype, kw):
    l, u = make(gpu, 7, vocab, seed=vocab, dtype=DT[dtype])
    check(l, u, **kw)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_settings_of_each_row(gpu, dtype):
    rows = 48
    l, u = make(gpu, rows, 20011, seed=1, dtype=DT[dtype])
    l *= torch.linspace(0.05, 3, rows, device=gpu)[:, None].to(l.dtype)
    g = torch.Generator().manual_seed(5)
    pick = lambda *v: torch.tensor(v)[torch.randint(len(v), (rows,), generator=g)]  # noqa: E731
    check(l, u, t=pick(0.0, 0.2, 1.0, 1.0, 2.0, -1.0).float().to(gpu),
          k=pick(0, 1, 7, 90, 1500, 5000, 30000, -4).int().to(gpu),
          p=pick(0.0, 0.1, 0.7, 0.99, 1.0, 1.0, 1.5).float().to(gpu),
          mp=pick(0.0, 0.0, 1e-3, 0.2, 1.0, 2.0, -1.0).float().to(gpu))


@pytest.mark.parametrize("kw", [dict(p=0.5), dict(p=0.97), dict(k=4000), dict(k=19000, p=0.7),
                                dict(mp=0.3), dict(mp=0.01, p=0.9), dict(k=1800, mp=0.2, p=0.6),
                                dict(t=50.0, p=0.8), dict(t=0.001, k=5000)],
                         ids=lambda k: "-".join(f"{a}{b}" for a, b in k.items()))
@pytest.mark.parametrize("sigma", [0.05, 1.0, 200.0])
def test_many_tokens_kept(gpu, kw, sigma):
    """Flat rows: thousands of kept tokens, boundaries deep in the row."""
    l, u = make(gpu, 9, 20011, sigma=sigma, seed=int(sigma * 100))
    check(l, u, **kw)


@pytest.mark.parametrize("kw", [dict(), dict(p=0.3), dict(p=0.9, t=0.5), dict(k=10), dict(k=2500),
                                dict(k=7001, p=0.5), dict(mp=0.5), dict(mp=0.1, p=0.8)],
                         ids=lambda k: "-".join(f"{a}{b}" for a, b in k.items()) or "plain")
@pytest.mark.parametrize("values", [1, 2, 5, 40])
@pytest.mark.parametrize("vocab", [300, 15000])
def test_equal_logits(gpu, kw, values, vocab):
    """Few distinct values, thousands of each: the lower index comes first."""
    g = torch.Generator().manual_seed(values)
    l = torch.randint(0, values, (6, vocab), generator=g).float() * 0.37
    l[0] = -0.0
    l[0, ::3] = 0.0  # equal to -0
    check(l.to(gpu), torch.rand(6, generator=g).to(gpu), **kw)


def test_both_ends_of_u(gpu):
    l, _ = make(gpu, 6, 5000, sigma=0.5, seed=3)
    u = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, -0.5, 2.0, float("nan")], device=gpu)
    for kw in (dict(), dict(k=20), dict(p=0.9), dict(p=0.99, k=4000)):
        check(l, u, **kw)


def test_masked_infinite_and_nan_logits(gpu):
    inf, nan, low = math.inf, math.nan, torch.finfo(torch.float32).min
    l, u = make(gpu, 10, 6000, seed=4)
    l[0] = -inf
    l[1] = -inf
    l[1, 4321] = -3.0
    l[2, 17], l[2, 5000] = inf, inf
    l[3, ::2] = nan
    l[4] = nan
    l[5] = low
    l[5, 100:103] = 1.0
    l[6] = low
    l[7, :] = -inf
    l[7, 5999] = inf
    l[8, 1:] = -inf
    l[9, 40] = 1e30
    for kw in (dict(), dict(t=0.0), dict(k=3), dict(p=0.9), dict(mp=0.1), dict(k=5500, p=0.99)):
        check(l, u, **kw)


def test_odd_settings(gpu):
    l, u = make(gpu, 4, 3000, seed=6)
    for kw in (dict(t=math.nan), dict(t=math.inf), dict(t=1e-42), dict(t=-0.0), dict(t=3e38),
               dict(p=math.nan, k=9), dict(mp=math.nan, k=9), dict(p=-1.0), dict(p=1e-30),
               dict(p=1.0 - 2.0 ** -24), dict(k=2 ** 31 - 1), dict(k=-5), dict(k=3000), dict(k=2999),
               dict(mp=1.0), dict(mp=7.0), dict(mp=1e-38)):
        check(l, u, **kw)


def test_many_rows_and_a_large_vocabulary(gpu):
    l, u = make(gpu, 300, 7777, seed=7)
    check(l, u, k=30, p=0.9, t=0.8)
    l, u = make(gpu, 3, 1 << 20, sigma=1.0, seed=8, dtype=torch.float16)
    for kw in (dict(), dict(k=50), dict(p=0.9), dict(k=1000), dict(k=100000, p=0.5)):
        check(l, u, **kw)


def test_strides_and_outputs(gpu):
    """Rows of a wider buffer, off every vector alignment; the caller's outputs; no
    log-probabilities; one row for all."""
    wide = torch.randn(9, 5050, device=gpu, dtype=torch.float16)
    l = wide[1:8, 3:4004]
    u = torch.rand(7, device=gpu)
    check(l, u, k=50, p=0.9)
    held = torch.full((20,), 99, dtype=torch.int32, device=gpu)
    tok, lp = sample(l, u, top_k=50, top_p=0.9, logprobs=False, out=held[5:12])
    assert lp is None and tok.data_ptr() == held[5:].data_ptr()
    assert torch.equal(tok, sample(l, u, top_k=50, top_p=0.9)[0])
    assert (held[:5] == 99).all() and (held[12:] == 99).all()
    one = l[:1].expand(7, -1)
    check(one, u, p=0.8)
    assert sample(l[:0], u[:0])[0].shape == (0,)


def test_same_tokens_whatever_the_batch(gpu):
    l, u = make(gpu, 40, 51865, sigma=1.5, seed=9)
    for kw in (dict(temperature=0.9), dict(top_k=50, top_p=0.9), dict(top_p=0.95), dict(min_p=0.02)):
        whole = sample(l, u, **kw)
        again = sample(l, u, **kw)
        part = sample(l[11:14], u[11:14], **kw)
        for a, b, c in zip(whole, again, part):
            assert torch.equal(a, b) and torch.equal(a[11:14], c)


def test_streams_and_graph_replays(gpu):
    l, u = make(gpu, 12, 9001, seed=10)
    t = torch.full((12,), 0.7, device=gpu)
    kw = dict(temperature=t, top_k=60, top_p=0.9)
    first = sample(l, u, **kw)
    torch.cuda.synchronize()
    outs = []
    for s in [torch.cuda.Stream() for _ in range(2)] * 3:
        with torch.cuda.stream(s):
            outs.append(sample(l, u, **kw))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for o in outs for a, b in zip(first, o))
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = sample(l, u, **kw)
        graphs.append((g, o))
    for i in range(4):
        l.copy_(torch.randn_like(l) * 2), u.copy_(torch.rand_like(u)), t.fill_(0.5 + 0.2 * i)
        g, o = graphs[i % 2]
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(o, sample(l, u, **kw)))
        check(l, u, got=o, t=t, k=60, p=0.9)


def test_frequencies(gpu):
    """Evenly spread u draw each token in proportion: within one draw a token of n p (the uniform
    grid's discrepancy), and nothing outside the kept set."""
    probs = torch.tensor([0.4, 0.05, 0.3, 0.2, 0.05])
    n = 4000
    l = torch.log(probs).expand(n, 5).contiguous().to(gpu)
    u = ((torch.arange(n) + 0.5) / n).float().to(gpu)
    got = torch.bincount(sample(l, u)[0], minlength=5).cpu()
    assert ((got - n * probs).abs() <= 2).all(), got
    got = torch.bincount(sample(l, u, top_k=3)[0], minlength=5).cpu()
    assert got[1] == 0 and got[4] == 0 and (got[[0, 2, 3]] - n * probs[[0, 2, 3]] / 0.9).abs().max() <= 2


def test_short_workspace_is_refused(gpu):
    l, u = make(gpu, 5, 5000)
    n = workspace_bytes(5, 5000)
    sample(l, u, workspace=torch.empty(n, dtype=torch.uint8, device=gpu))
    with pytest.raises(L.FfaiError, match="workspace"):
        sample(l, u, workspace=torch.empty(n - 1, dtype=torch.uint8, device=gpu))


@pytest.mark.parametrize("vocab,rows", [(51865, 3), (131072, 2), (200001, 1), (300000, 2)])
@pytest.mark.parametrize("kw", [dict(p=0.85), dict(p=0.999), dict(p=0.5, t=1.7), dict(mp=0.02),
                                dict(p=0.99999, t=0.8), dict(p=1 - 2.0 ** -24, t=0.9),
                                dict(p=0.99999, mp=0.001),
                                dict(p=0.9, mp=0.01), dict(p=0.9, mp=0.3, t=0.4), dict(p=1e-9),
                                dict(p=-1.0), dict(p=0.6, t=math.inf)], ids=str)
@pytest.mark.parametrize("sigma", [0.3, 3.0])
def test_nuclei_and_minima_of_many_tokens(gpu, vocab, rows, kw, sigma):
    """More tokens than a list holds, spread over several workgroups a row; logits of 16 bits, so
    that many are equal, and (small sigma) more in the boundary's bins than are listed."""
    for dtype in (torch.float32, torch.bfloat16):
        l, u = make(gpu, rows, vocab, sigma=sigma, seed=vocab + rows, dtype=dtype)
        check(l, u, **kw)


def test_one_workspace_for_changing_settings(gpu):
    """What a call leaves in the workspace is nothing to the next: rows that were wide nuclei are
    settled by their list, greedy, unfiltered or minima in the next, and the other way round."""
    rows, vocab = 6, 60000
    l, u = make(gpu, rows, vocab, sigma=1.5, seed=8)
    peaked = l.clone()
    peaked[:, 7] = 30.0
    masked = l.clone()
    masked[1::2] = -math.inf
    infinite = l.clone()
    infinite[::2, 99] = math.inf
    work = torch.empty(workspace_bytes(rows, vocab), dtype=torch.uint8, device=gpu)
    work.fill_(255)
    mixed = dict(t=torch.tensor([0.0, 1.0, 0.7, 1.0, 2.0, 1.0], device=gpu),
                 k=torch.tensor([0, 40, 0, 0, 3000, 0], dtype=torch.int32, device=gpu),
                 p=torch.tensor([0.9, 0.9, 0.8, 1.0, 0.9, 0.95], device=gpu),
                 mp=torch.tensor([0.0, 0.0, 0.0, 0.01, 0.0, 0.001], device=gpu))
    for x in (l, peaked, masked, infinite, l, infinite, peaked, l):
        for kw in (dict(p=0.9), mixed, dict(mp=0.05), dict(), dict(k=30, p=0.9), dict(p=0.8, mp=0.01)):
            got = sample(x, u, temperature=kw.get("t"), top_k=kw.get("k"), top_p=kw.get("p"),
                         min_p=kw.get("mp"), workspace=work)
            check(x, u, got=got, **kw)


def test_wide_nuclei_in_a_graph(gpu):
    rows, vocab = 5, 52000
    l, u = make(gpu, rows, vocab, sigma=1.0, seed=21)
    sample(l, u, top_p=0.9, min_p=0.001)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        tok, lp = sample(l, u, top_p=0.9, min_p=0.001)
    for i in range(4):
        a, b = make(gpu, rows, vocab, sigma=0.5 + i, seed=30 + i)
        l.copy_(a)
        u.copy_(b)
        g.replay()
        want = sample(l, u, top_p=0.9, min_p=0.001)
        torch.cuda.synchronize()
        assert torch.equal(tok, want[0]) and torch.equal(lp, want[1])
        check(l, u, got=(tok, lp), p=0.9, mp=0.001)
