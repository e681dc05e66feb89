"""Attention over a shared prefix (ffai_amd.prefix) against the definition in 64 bits.

Tolerances. Let A = sum_j p_j |v_j| (p the exact softmax weights), e = 2^-24, n the visible keys, r
the largest sum_d |q_d k_d| * scale of the row. A score sums D exact products in f32 and is scaled
once: off by at most (D + 4) e r; its exponential and the multiplication by log2 e add at most
(8 + 2 r) e; the sums of n weights and products at most n e each, and each of the (at most 130)
joins of pieces a few e. A weight carried in parts is off by at most 2^-22. So with
delta = (D + 4 + 2) e r + (2 n + 300) e + 2^-22, the f32 result is off by at most 2 delta A (weights
and their sum), and is rounded once more by e |o|. A 16-bit result rounds each weight by at most
u = eps / 2 (u A in all; f16 weights below 2^-14 round by at most 2^-25 of the largest, n 2^-25
max |v| in all) and itself by u |o|."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from ffai_amd import _lib as L
from ffai_amd import flash_attn as fa
from ffai_amd.kv_cache import KVCache
from ffai_amd.prefix import PrefixAttention, prefix_attention
from oracle.prefix import prefix_attend

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def make(dev, groups, per, hkv, rep, t, d, plens, olens, pcap, ocap, q="bf16", kv="bf16", seed=0,
         stale=float("nan"), k_gain=1.0):
    g = torch.Generator().manual_seed(seed)

    def rand(*shape):
        return torch.randn(shape, generator=g)

    s = groups * per
    x = {"q": rand(s, hkv * rep, t, d).to(DT[q])}
    for name, n, cap, lens in (("p", groups, pcap, plens), ("o", s, ocap, olens)):
        for m in "kv":
            y = (rand(n, hkv, cap, d) * (k_gain if m == "k" else 1.0)).to(DT[kv])
            for i in range(n):  # what lies past a length is no one's business
                y[i, :, max(0, min(cap, lens[i])):] = stale
            x[name + m] = y
        x[name + "lens"] = torch.tensor(lens, dtype=torch.int32)
    return {k: v.to(dev) for k, v in x.items()}


def caches(x):
    return (KVCache.from_tensors(x["pk"], x["pv"], x["plens"]),
            KVCache.from_tensors(x["ok"], x["ov"], x["olens"]))


def check(got, x, scale, out_dtype):
    c = {k: v.float().cpu().numpy() if v.is_floating_point() else v.cpu().numpy()
         for k, v in x.items()}
    want, mean, reach = prefix_attend(c["q"], c["pk"], c["pv"], c["plens"], c["ok"], c["ov"],
                                      c["olens"], scale)
    d = want.shape[3]
    n = c["pk"].shape[2] + c["ok"].shape[2]
    e = 2.0 ** -24
    delta = (d + 6) * e * reach[..., None] + (2 * n + 300) * e + 2.0 ** -22
    tol = 2 * delta * mean + e * np.abs(want) + 1e-30
    if out_dtype != torch.float32:
        u = torch.finfo(out_dtype).eps / 2
        tol = tol + u * mean + u * np.abs(want)
        if out_dtype == torch.float16:
            tol = tol + n * 2.0 ** -25 * max(np.nanmax(np.abs(c["pv"]), initial=0),
                                             np.nanmax(np.abs(c["ov"]), initial=0)) + 2.0 ** -25
    got = got.double().cpu().numpy()
    finite = np.isfinite(want)
    assert np.array_equal(np.isfinite(got), finite)
    err = np.abs(got[finite] - want[finite])
    assert (err <= np.broadcast_to(tol, want.shape)[finite]).all(), err.max(initial=0)


IO = [("bf16", "bf16", "bf16"), ("f16", "f16", "f16"), ("bf16", "bf16", "f32"),
      ("f16", "f16", "f32"), ("f32", "bf16", "f32"), ("f32", "f16", "f32")]
# groups, per, hkv, rep, t, d, plens, olens, pcap, ocap
SHAPES = {
    "one of everything": (1, 1, 1, 1, 1, 64, [1], [1], 1, 1),
    "prefix alone": (1, 3, 2, 1, 1, 64, [65], [0, 0, 0], 65, 7),
    "own alone": (1, 3, 2, 1, 1, 128, [0], [1, 63, 64], 1, 64),
    "some rows see nothing": (2, 2, 1, 2, 3, 64, [0, 2], [0, 2, 1, 5], 4, 6),
    "tile edges": (4, 1, 1, 3, 1, 64, [63, 64, 65, 129], [127, 128, 0, 66], 130, 128),
    "lengths out of range": (2, 1, 1, 1, 1, 128, [99, -3], [-1, 1000], 70, 70),
    "beams": (1, 5, 16, 1, 1, 64, [37], [3, 20, 33, 47, 61], 37, 448),
    "rows past 16": (1, 17, 1, 1, 1, 128, [130], list(range(1, 18)), 131, 20),
    "rows past 32, a ragged block": (2, 11, 1, 3, 1, 64, [200, 77], list(range(40, 62)), 200, 64),
    "several tokens": (1, 4, 2, 1, 5, 64, [100], [5, 69, 64, 130], 100, 130),
    "several tokens, grouped": (2, 2, 2, 4, 3, 128, [70, 40], [3, 64, 66, 90], 70, 90),
    "rows of one slot past 32": (1, 2, 1, 8, 5, 64, [90], [5, 77], 90, 80),
    "a prompt's continuation": (1, 2, 1, 1, 70, 128, [33], [70, 140], 40, 140),
    "many pieces": (1, 2, 1, 2, 1, 128, [2500], [700, 1], 2501, 1100),
}


@pytest.mark.parametrize("shape", SHAPES, ids=[s.replace(" ", "_") for s in SHAPES])
@pytest.mark.parametrize("io", IO, ids=["-".join(i) for i in IO])
@pytest.mark.parametrize("roomy", [False, True], ids=["tight", "roomy"])
def test_against_the_definition(gpu, shape, io, roomy):
    """`roomy`: the same sequences in caches of a large capacity, which run in pieces with a merge
    where the tight ones run in one launch."""
    q, kv, out = io
    gr, per, hkv, rep, t, d, pl, ol, pc, oc = SHAPES[shape]
    if roomy:
        pc, pl = pc + 3000, [min(n, pc) for n in pl]  # (a length past the tight capacity ends there)
        oc, ol = oc + 3000, [min(n, oc) for n in ol]
    x = make(gpu, gr, per, hkv, rep, t, d, pl, ol, pc, oc, q, kv)
    got = prefix_attention(x["q"], *caches(x), scale=d ** -0.5, out_dtype=DT[out])
    assert got.dtype == DT[out] and got.shape == x["q"].shape
    check(got, x, d ** -0.5, DT[out])


# shapes whose prefix runs in shared tiles (blocks of 128 rows): a block with an idle wave, ragged
# blocks, one query token and several, groups of unlike lengths, one empty
MANY = {
    "an idle wave": (1, 70, 16, 1, 1, 64, [5600], list(range(1, 71)), 5601, 72),
    "ragged blocks, grouped": (1, 50, 4, 4, 1, 128, [9500], list(range(70, 120)), 9600, 120),
    "tokens and groups": (4, 10, 4, 3, 3, 128, [5700, 0, 64, 5631], [3 + i for i in range(40)], 5700, 44),
}


@pytest.mark.parametrize("shape", MANY, ids=[s.replace(" ", "_") for s in MANY])
@pytest.mark.parametrize("io", [IO[0], IO[1], IO[2], IO[5]], ids=lambda i: "-".join(i))
def test_many_rows(gpu, shape, io):
    q, kv, out = io
    gr, per, hkv, rep, t, d, pl, ol, pc, oc = MANY[shape]
    x = make(gpu, gr, per, hkv, rep, t, d, pl, ol, pc, oc, q, kv, seed=19)
    plan = PrefixAttention(*caches(x), hkv * rep, t, q_dtype=DT[q], out_dtype=DT[out], scale=d ** -0.5)
    assert plan.plan()["row_block"] > 32
    got = plan(x["q"])
    check(got, x, d ** -0.5, DT[out])
    assert torch.equal(got, plan(x["q"]))


@pytest.mark.parametrize("cap", [80, 4000])
def test_one_slots_infinities_stay_its_own(gpu, cap):
    """One query token a slot: a slot whose every V is infinite or NaN among ordinary ones."""
    x = make(gpu, 1, 5, 2, 1, 1, 64, [70], [66, 40, 3, 0, 80], 70, cap, "bf16", "bf16", seed=6)
    x["ov"][1, :, 3] = float("inf")
    x["ov"][2, 0, 1, 3] = float("nan")
    x["ok"][4, 1, 7] = float("nan")
    got = prefix_attention(x["q"], *caches(x), scale=0.125)
    check(got, x, 0.125, torch.bfloat16)
    assert torch.isfinite(got[[0, 3]]).all() and torch.isinf(got[1]).all()
    assert torch.isnan(got[2, 0, 0, 3]) and torch.isfinite(got[2, 1]).all()
    assert torch.isnan(got[4, 1]).all() and torch.isfinite(got[4, 0]).all()


@pytest.mark.parametrize("kv", ["bf16", "f16"])
@pytest.mark.parametrize("gain", [0.01, 8.0])
def test_flat_and_sharp_rows(gpu, kv, gain):
    """Nearly uniform weights, and rows that one key takes."""
    x = make(gpu, 1, 6, 2, 2, 1, 64, [300], [10, 40, 64, 1, 0, 77], 300, 80, "f32", kv, seed=3,
             k_gain=gain)
    check(prefix_attention(x["q"], *caches(x), scale=0.5), x, 0.5, torch.float32)


@pytest.mark.parametrize("io", [("f16", "f16", "f16"), ("f32", "bf16", "f32")])
@pytest.mark.parametrize("cap", [66, 4000])
def test_non_finite_values_of_keys_that_a_row_does_not_see(gpu, io, cap):
    """A later token's K and V may hold anything, and so may another slot's: only the rows that see
    them are touched."""
    q, kv, out = io
    x = make(gpu, 1, 2, 1, 2, 4, 64, [70], [66, 40], 70, cap, q, kv, seed=5)
    x["ok"][0, :, 64] = float("nan")
    x["ov"][0, :, 65, 5] = float("inf")
    x["ov"][1, :, 39, 7] = float("nan")
    x["ov"][1, :, 38, 9] = float("-inf")
    got = prefix_attention(x["q"], *caches(x), scale=0.125, out_dtype=DT[out])
    check(got, x, 0.125, DT[out])
    assert torch.isfinite(got[0, :, :2]).all() and torch.isnan(got[0, :, 2:]).all()
    assert torch.isnan(got[1, :, 3, 7]).all() and torch.isinf(got[1, :, 2, 9]).all()


def test_strides(gpu):
    """q as the (slots, t, heads, d) rows of a packed q/k/v projection, out in the merged layout
    with rows of a larger buffer, caches as layers and slot slices of larger ones."""
    s, h, t, d = 4, 6, 2, 64
    x = make(gpu, 2, 2, h, 1, t, d, [70, 12], [3, 66, 20, 9], 70, 66, "f16", "f16", seed=7)
    big = torch.randn(s, t, 3 * h * d, device=gpu, dtype=torch.float16)
    big[:, :, :h * d] = x["q"].transpose(1, 2).reshape(s, t, h * d)
    q = big[:, :, :h * d].view(s, t, h, d).transpose(1, 2)
    stack = KVCache(s + 3, h, 80, d, dtype=torch.float16, device=gpu, layers=3)
    stack.k.fill_(float("nan")), stack.v.fill_(float("nan"))
    lay = stack.layer(1)
    lay.k[2:2 + s, :, :66] = x["ok"]
    lay.v[2:2 + s, :, :66] = x["ov"]
    lay.lens[2:2 + s] = x["olens"]
    own = KVCache.from_tensors(lay.k[2:2 + s], lay.v[2:2 + s], lay.lens[2:2 + s])
    held = torch.full((s + 2, t, h * d + 8), 7.0, device=gpu, dtype=torch.float16)
    out = held[1:1 + s, :, 8:].view(s, t, h, d).transpose(1, 2)
    got = prefix_attention(q, caches(x)[0], own, scale=0.125, out=out)
    assert got.data_ptr() == out.data_ptr()
    check(got, x, 0.125, torch.float16)
    assert (held[0] == 7).all() and (held[-1] == 7).all() and (held[:, :, :8] == 7).all()


def test_equals_one_cache_that_holds_both(gpu):
    """A shared prefix plus own keys against fa.attention over each slot's whole sequence."""
    x = make(gpu, 1, 5, 4, 1, 1, 64, [100], [28, 1, 77, 40, 60], 100, 80, seed=9, stale=0.0)
    k = torch.cat([x["pk"].expand(5, -1, -1, -1), x["ok"]], 2).contiguous()
    v = torch.cat([x["pv"].expand(5, -1, -1, -1), x["ov"]], 2).contiguous()
    lens = (x["olens"] + 100).int()
    want = fa.attention(x["q"], k, v, scale=0.125, kv_lens=lens, out_dtype=torch.float32)
    got = prefix_attention(x["q"], *caches(x), scale=0.125, out_dtype=torch.float32)
    # both within the definition's bound; fa.attention rounds its weights to bf16
    assert (got - want).abs().max() <= 2 * torch.finfo(torch.bfloat16).eps * 4


def test_same_bits_and_other_streams(gpu):
    x = make(gpu, 2, 8, 4, 2, 1, 128, [1500, 900], list(range(30, 46)), 1500, 64, seed=11)
    plan = PrefixAttention(*caches(x), 8, scale=0.088)
    first = plan(x["q"])
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for i in range(6):
        with torch.cuda.stream(side[i % 2]):
            outs.append(plan(x["q"]))
    torch.cuda.synchronize()
    assert all(torch.equal(first, o) for o in outs)


def test_graph_replays_follow_the_lengths(gpu):
    """A captured step: append, attend, with the lengths advancing on the device between replays,
    two graphs over the same caches; every replay equals the eager call."""
    torch.manual_seed(1)
    x = make(gpu, 1, 3, 2, 1, 1, 64, [50], [60, 1, 63], 50, 90, seed=13, stale=0.0)
    pre, own = caches(x)
    plan = PrefixAttention(pre, own, 2, scale=0.125)
    kn, vn = (torch.randn(3, 1, 128, device=gpu, dtype=torch.bfloat16) for _ in range(2))
    plan.step(x["q"], kn, vn)
    torch.cuda.synchronize()
    graphs = []
    s = torch.cuda.Stream()
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out = plan.step(x["q"], kn, vn)
        graphs.append((g, out))
    for i in range(6):
        kn.copy_(torch.randn_like(kn)), vn.copy_(torch.randn_like(vn))
        before = own.lens.clone()
        g, out = graphs[i % 2]
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(own.lens, before + 1)
        assert torch.equal(out, plan(x["q"]))
        check(out, x, 0.125, torch.bfloat16)


def test_offsets_past_32_bits(gpu):
    """Slots and positions whose elements lie past 2^31 from the cache's start."""
    cap, d, h = 1 << 19, 64, 33
    k = torch.empty(2, h, cap, d, dtype=torch.bfloat16, device=gpu)  # 2.2e9 elements
    v = torch.empty_like(k)
    g = torch.Generator().manual_seed(2)
    small = {}
    for name, t in (("ok", k), ("ov", v)):
        y = torch.randn(2, h, 70, d, generator=g).bfloat16().to(gpu)
        t[:, :, :70] = y
        small[name] = y
    x = make(gpu, 1, 2, h, 1, 1, d, [40], [70, 67], 40, 70, seed=15)
    x.update(small)
    own = KVCache.from_tensors(k, v, x["olens"])
    got = prefix_attention(x["q"], caches(x)[0], own, scale=0.125)
    check(got, x, 0.125, torch.bfloat16)


def test_a_whole_beam_step(gpu):
    """Prompt into the prefix cache, beams forked, stepped and reordered: what the beams see is
    what one whole sequence per beam would hold."""
    torch.manual_seed(3)
    beams, h, d, prompt = 4, 3, 64, 37
    pre = KVCache(1, h, prompt, d, device=gpu)
    two = [KVCache(beams, h, 16, d, device=gpu) for _ in range(2)]
    kp, vp = (torch.randn(1, prompt, h * d, device=gpu, dtype=torch.bfloat16) for _ in range(2))
    pre.append(kp, vp)
    hist = [[] for _ in range(beams)]
    plans = [PrefixAttention(pre, c, h, scale=0.125) for c in two]
    cur = 0
    for step in range(5):
        q = torch.randn(beams, h, 1, d, device=gpu, dtype=torch.bfloat16)
        kn, vn = (torch.randn(beams, 1, h * d, device=gpu, dtype=torch.bfloat16) for _ in range(2))
        out = plans[cur].step(q, kn, vn)
        hist = [hist[b] + [(kn[b], vn[b])] for b in range(beams)]
        n = len(hist[0])
        ok, ov = (torch.stack([torch.cat([t[i] for t in hist[b]]) for b in range(beams)])
                  .view(beams, n, h, d).transpose(1, 2) for i in range(2))
        x = {"q": q, "pk": pre.k, "pv": pre.v, "plens": pre.lens, "ok": ok, "ov": ov,
             "olens": torch.full((beams,), n, dtype=torch.int32)}
        check(out, x, 0.125, torch.bfloat16)
        parent = torch.randint(0, beams, (beams,), device=gpu, dtype=torch.int32)
        two[1 - cur].gather_from(two[cur], parent)
        hist = [list(hist[p]) for p in parent.tolist()]
        cur = 1 - cur


def test_shared_output_of_a_plan(gpu):
    """A plan's caches may be refilled with another sequence between calls: nothing is kept."""
    x = make(gpu, 1, 2, 1, 1, 1, 64, [20], [5, 9], 20, 12, seed=17, stale=0.0)
    plan = PrefixAttention(*caches(x), 1, scale=0.125)
    check(plan(x["q"]), x, 0.125, torch.bfloat16)
    x["pk"].normal_(), x["ov"].normal_(), x["plens"].fill_(3), x["olens"].fill_(12)
    check(plan(x["q"]), x, 0.125, torch.bfloat16)


def test_a_short_workspace_is_refused(gpu):
    x = make(gpu, 1, 2, 1, 1, 1, 64, [3000], [5, 9], 3000, 12)
    plan = PrefixAttention(*caches(x), 1)
    plan(x["q"], workspace=torch.empty(plan.workspace_bytes, dtype=torch.uint8, device=gpu))
    with pytest.raises(L.FfaiError, match="workspace"):
        plan(x["q"], workspace=torch.empty(plan.workspace_bytes - 1, dtype=torch.uint8, device=gpu))


# so many heads that a workgroup takes several slots: their rows side by side in one or two blocks
# of 16 columns, each slot's own tiles masked for the others
SIDE = {
    "one row a slot": (2, 24, 32, 1, 1, 64, [70, 0], [i % 81 for i in range(48)], 70, 80),
    "four rows, two blocks": (2, 24, 32, 4, 1, 64, [130, 3], [(7 * i) % 65 for i in range(48)], 130, 64),
    "tokens": (1, 40, 64, 1, 2, 128, [65], [(3 * i) % 64 for i in range(40)], 65, 63),
}


@pytest.mark.parametrize("shape", SIDE, ids=[s.replace(" ", "_") for s in SIDE])
@pytest.mark.parametrize("io", IO, ids=["-".join(i) for i in IO])
def test_slots_side_by_side(gpu, shape, io):
    q, kv, out = io
    gr, per, hkv, rep, t, d, pl, ol, pc, oc = SIDE[shape]
    x = make(gpu, gr, per, hkv, rep, t, d, pl, ol, pc, oc, q, kv, seed=31)
    plan = PrefixAttention(*caches(x), hkv * rep, t, q_dtype=DT[q], out_dtype=DT[out], scale=d ** -0.5)
    assert plan.workspace_bytes == 0 and plan.plan()["row_block"] > rep * t
    got = plan(x["q"])
    check(got, x, d ** -0.5, DT[out])
    # two slots of non-finite values: the others' results are what they were
    odd = torch.tensor([3, 22], device=gpu)
    for name, value in (("ov", float("inf")), ("ok", float("nan")), ("ov", float("nan"))):
        x[name][odd] = value
        again = plan(x["q"])
        keep = torch.ones(len(ol), dtype=torch.bool, device=gpu)
        keep[odd] = False
        assert torch.equal(again[keep], got[keep])
