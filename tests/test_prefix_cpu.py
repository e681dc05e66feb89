"""What attention over a shared prefix refuses, and its plan: no GPU needed (nothing is launched)."""

from __future__ import annotations

import ctypes
import re

import pytest
import torch

from ffai_amd import _lib as L
from ffai_amd.kv_cache import KVCache
from ffai_amd.prefix import PrefixAttention


def cache(slots=2, heads=4, cap=10, d=64, dtype=torch.bfloat16):
    k = torch.zeros(slots, heads, cap, d, dtype=dtype)
    return KVCache.from_tensors(k, torch.zeros_like(k), torch.zeros(slots, dtype=torch.int32))


def fwd(a_prefix, an_own, heads_q=4, q_len=1, q_dtype=L.BF16, out_dtype=L.BF16, scale=1.0, **edit):
    """The C call on made-up operands: only for calls that are refused before any launch."""
    d = an_own.head_dim
    a = dict(q=4096, out=8192, qs=(heads_q * q_len * d, q_len * d, d), os=None, ws=4096,
             ws_bytes=1 << 40)
    a.update(edit)
    a["os"] = a["os"] or a["qs"]
    pv, ov = a_prefix.view(), an_own.view()
    for name, view in (("pre", pv), ("own", ov)):
        for field, value in edit.get(name, {}).items():
            if field == "strides":
                view.strides[:] = value
            else:
                setattr(view, field, value)
    rc = L.load().ffai_prefix_attn_fwd(
        ctypes.byref(pv), ctypes.byref(ov), a["q"], q_dtype, heads_q, q_len,
        (ctypes.c_int64 * 3)(*a["qs"]), scale, a["out"], out_dtype,
        (ctypes.c_int64 * 3)(*a["os"]), a["ws"], a["ws_bytes"], None)
    return rc, L.last_error()


BAD = [
    (dict(heads_q=6), "heads_q"), (dict(heads_q=0), "heads_q"), (dict(q_len=0), "q_len"),
    (dict(q=0), "null"), (dict(out=0), "null"), (dict(scale=0.0), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(q_dtype=L.F16), "q must be"), (dict(out_dtype=L.F16), "out must be"),
    (dict(q_dtype=L.F32, out_dtype=L.BF16), "out must be"), (dict(q_dtype=9), "q must be"),
    (dict(q=4097), "aligned"), (dict(out=8193), "aligned"), (dict(ws=4104), "workspace"),
    (dict(qs=(-1, 64, 64)), "negative"), (dict(os=(256, 32, 64)), "overlap"),
    (dict(pre=dict(k=4097)), "16-byte"), (dict(own=dict(v=4104)), "16-byte"),
    (dict(own=dict(k=None)), "null"), (dict(pre=dict(lens=None)), "null"),
    (dict(own=dict(strides=(2560, 640, 60))), "position stride"),
    (dict(own=dict(strides=(2560, 640, 1 << 24))), "position stride"),
    (dict(pre=dict(strides=(2564, 640, 64))), "multiples of 8"),
    (dict(own=dict(dtype=7)), "dtype"), (dict(own=dict(dtype=L.F16)), "differ"),
    (dict(own=dict(heads=2)), "differ"), (dict(own=dict(head_dim=128)), "differ"),
    (dict(own=dict(slots=3)), "multiple"), (dict(own=dict(capacity=0)), "capacity"),
    (dict(own=dict(capacity=(1 << 30) + 1)), "capacity"), (dict(q_len=1 << 22), "2\\^24"),
]


@pytest.mark.parametrize("edit,why", BAD, ids=[f"{i}-{next(iter(b[0]))}" for i, b in enumerate(BAD)])
def test_bad_arguments(edit, why):
    rc, msg = fwd(cache(2), cache(4), **edit)
    assert rc == L.FFAI_ERR_INVALID and re.search(why, msg), (rc, msg)


def test_workspace_is_checked():
    for ws in (dict(ws=0), dict(ws_bytes=0)):
        rc, msg = fwd(cache(2, cap=4000), cache(4), **ws)
        assert rc == L.FFAI_ERR_WORKSPACE and "workspace" in msg


@pytest.mark.parametrize("kw", [dict(dtype=torch.float32), dict(d=96), dict(d=256)])
def test_declined(kw):
    pre, own = cache(2, **kw), cache(4, **kw)
    n = ctypes.c_size_t()
    rc = L.load().ffai_prefix_attn_workspace_bytes(ctypes.byref(pre.view()), ctypes.byref(own.view()),
                                                   4, 1, ctypes.byref(n))
    assert rc == L.FFAI_DECLINED
    with pytest.raises(ValueError, match="not served"):
        PrefixAttention(pre, own, 4)


def test_binding_refuses():
    pre, own = cache(2), cache(4)
    plan = PrefixAttention(pre, own, 8, 3)
    for q in (torch.zeros(4, 8, 3, 64), torch.zeros(4, 8, 2, 64, dtype=torch.bfloat16),
              torch.zeros(4, 4, 3, 64, dtype=torch.bfloat16)):
        with pytest.raises(ValueError, match="q must be"):
            plan(q)
    with pytest.raises(ValueError, match="HIP device"):  # host memory never reaches a kernel
        plan(torch.zeros(4, 8, 3, 64, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="k_new"):
        plan.step(torch.zeros(4, 8, 3, 64, dtype=torch.bfloat16), torch.zeros(4, 1, 256),
                  torch.zeros(4, 1, 256))
    with pytest.raises(ValueError, match="one layer"):
        PrefixAttention(pre, KVCache(4, 4, 8, 64, device="cpu", layers=2), 4)
    with pytest.raises(ValueError, match="f32, f16"):
        PrefixAttention(pre, own, 4, q_dtype=torch.int32)


@pytest.mark.parametrize("edit,why", [
    (dict(v=torch.zeros(2, 4, 9, 64)), "alike"), (dict(k=torch.zeros(2, 4, 64)), "alike"),
    (dict(lens=torch.zeros(2)), "int32"), (dict(lens=torch.zeros(3, dtype=torch.int32)), "int32"),
    (dict(lens=torch.zeros(4, dtype=torch.int32)[::2]), "contiguous"),
    (dict(k=torch.zeros(2, 4, 10, 64, dtype=torch.int8), v=torch.zeros(2, 4, 10, 64, dtype=torch.int8)),
     "f32, f16"),
    (dict(k=torch.zeros(2, 4, 64, 10).transpose(2, 3), v=torch.zeros(2, 4, 64, 10).transpose(2, 3)),
     "contiguous"),
])
def test_from_tensors_refuses(edit, why):
    a = dict(k=torch.zeros(2, 4, 10, 64), v=torch.zeros(2, 4, 10, 64),
             lens=torch.zeros(2, dtype=torch.int32))
    a.update(edit)
    with pytest.raises(ValueError, match=why):
        KVCache.from_tensors(**a)


def test_from_tensors_views_what_it_is_given():
    k = torch.randn(5, 4, 16, 64)
    lens = torch.arange(5, dtype=torch.int32)
    c = KVCache.from_tensors(k[1:3, :, 2:12], k[1:3, :, 2:12], lens[1:3])
    v = c.view()
    assert (c.slots, c.heads, c.capacity, c.head_dim) == (2, 4, 10, 64)
    assert v.k == k[1:3, :, 2:12].data_ptr() and list(v.strides) == list(k.stride()[:3])


@pytest.mark.parametrize("groups,per,hkv,rep,t,pcap,ocap", [
    (1, 1, 1, 1, 1, 1, 1), (1, 5, 16, 1, 1, 37, 448), (8, 5, 16, 1, 1, 224, 224),
    (1, 16, 2, 6, 1, 4096, 512), (1, 128, 8, 4, 1, 16384, 1024), (3, 8, 20, 1, 5, 1111, 400),
    (1, 1, 1, 8, 7, 100000, 3), (1, 1, 1, 40, 1, 10, 10)])
@pytest.mark.parametrize("d", [64, 128])
def test_plan_covers_every_key_and_row(groups, per, hkv, rep, t, pcap, ocap, d):
    """One launch over whole slots with no workspace; or pieces of whole tiles, at least one a side
    and at most one per four tiles, and a workspace that holds every piece of every row."""
    pre, own = cache(groups, hkv, pcap, d), cache(groups * per, hkv, ocap, d)
    plan = PrefixAttention(pre, own, hkv * rep, t)
    p = plan.plan()
    assert p["rows"] == per * rep * t
    assert 1 <= p["row_block"] <= 128
    if plan.workspace_bytes == 0:
        slots = p["row_block"] // (rep * t)
        assert slots >= 1 and p["own_pieces"] == 0
        assert p["workgroups"] == groups * hkv * -(-per // slots)
        return
    assert 1 <= p["prefix_pieces"] <= max(1, -(-pcap // 256))
    assert 1 <= p["own_pieces"] <= max(1, -(-ocap // 256))
    rows = groups * per * hkv * rep * t
    pieces = p["prefix_pieces"] + p["own_pieces"]
    assert plan.workspace_bytes >= rows * pieces * (d + 2) * 4


def test_short_sequences_take_no_workspace():
    assert PrefixAttention(cache(1, 16, 37), cache(5, 16, 448), 16).workspace_bytes == 0
    assert PrefixAttention(cache(1, 16, 4096), cache(5, 16, 448), 16).workspace_bytes > 0
