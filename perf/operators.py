"""One step of many continuations of shared prompts, operator by operator: what each costs, and what
it computes in plain form.

The kinds:

* ``prefix``: attention of slots that share a prompt. Slots come in groups; a slot's queries see the
  keys of its group's prefix, held once, and its own keys, held per slot (a beam's or a sample's
  tokens since the prompt). Ragged lengths on both sides; several query tokens at once are causal
  over the slot's last keys. Whole-number lengths live on the device.
* ``int8``: a linear layer in 8-bit integers: the rows of x are quantized with a scale each, the
  weights hold a scale for each output channel, and the integer products sum exactly.
* ``sample``: one token per row of logits, from given uniform numbers, with per-row temperature,
  top-k, min-p and top-p, and the token's log-probability under the unfiltered logits.

``own`` says whose code ``run`` calls: the plain forms below, or the library.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # --- attention over a shared prefix
        # whisper-medium's beam step early in a window: a short prompt, f32 rows in and out as the
        # decoder's f16 GEMVs take and give them; the smallest call, all latency
        {"name": "prefix_b5_h16_p37", "kind": "prefix", "groups": 1, "per": 5, "heads_kv": 16,
         "rep": 1, "d": 64, "t": 1, "prefix": 37, "lo": 3, "hi": 61, "cap": 448,
         "q": "f32", "kv": "f16", "out": "f32"},
        # the beams of eight windows, each window with the previous one's text as its prompt
        {"name": "prefix_g8_b5_h16_p224", "kind": "prefix", "groups": 8, "per": 5, "heads_kv": 16,
         "rep": 1, "d": 64, "t": 1, "prefix": 224, "lo": 20, "hi": 223, "cap": 224,
         "q": "bf16", "kv": "bf16", "out": "f32"},
        # five tokens at once per slot (drafted ones being checked), whisper-large's heads
        {"name": "prefix_g3_b8_h20_t5_p1111", "kind": "prefix", "groups": 3, "per": 8,
         "heads_kv": 20, "rep": 1, "d": 64, "t": 5, "prefix": 1111, "lo": 5, "hi": 397, "cap": 400,
         "q": "f16", "kv": "f16", "out": "f16"},
        # sixteen answers to one 4096-token prompt, grouped heads
        {"name": "prefix_b16_gqa12_p4096", "kind": "prefix", "groups": 1, "per": 16, "heads_kv": 2,
         "rep": 6, "d": 128, "t": 1, "prefix": 4096, "lo": 100, "hi": 511, "cap": 512,
         "q": "bf16", "kv": "bf16", "out": "bf16"},
        # a full batch behind one long shared document
        {"name": "prefix_b128_gqa32_p16384", "kind": "prefix", "groups": 1, "per": 128,
         "heads_kv": 8, "rep": 4, "d": 128, "t": 1, "prefix": 16384, "lo": 33, "hi": 1024,
         "cap": 1024, "q": "bf16", "kv": "bf16", "out": "bf16"},
        # --- 8-bit linear layers
        # five beams through a 1024-wide projection: latency
        {"name": "int8_m5_k1024_n1024", "kind": "int8", "m": 5, "k": 1024, "n": 1024, "bias": True,
         "x": "f32", "out": "f32"},
        # a 227-token prompt through the up projection of a 1024-wide MLP
        {"name": "int8_m227_k1024_n4096", "kind": "int8", "m": 227, "k": 1024, "n": 4096,
         "bias": True, "x": "f16", "out": "f16"},
        # one window's frames through the packed q/k/v projection, 1280 wide
        {"name": "int8_m1500_k1280_n3840", "kind": "int8", "m": 1500, "k": 1280, "n": 3840,
         "bias": True, "x": "bf16", "out": "bf16"},
        # sixteen windows' frames through the down projection of a 1280-wide MLP
        {"name": "int8_m24000_k5120_n1280", "kind": "int8", "m": 24000, "k": 5120, "n": 1280,
         "bias": False, "x": "bf16", "out": "bf16"},
        # --- sampling
        # five candidates of one window at a temperature of the ladder
        {"name": "sample_r5_v51865", "kind": "sample", "rows": 5, "vocab": 51865, "logits": "f32",
         "mode": "temperature"},
        # a batch with top-k and top-p
        {"name": "sample_r64_v51865", "kind": "sample", "rows": 64, "vocab": 51865,
         "logits": "f32", "mode": "top_k"},
        # a large batch over a large vocabulary, each row with settings of its own
        {"name": "sample_r256_v131072", "kind": "sample", "rows": 256, "vocab": 131072,
         "logits": "bf16", "mode": "mixed"},
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], its logarithm uniform."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("prefix", "int8", "sample"))
    if kind == "prefix":
        d = rng.choice((64, 128))
        if d == 64:
            hkv, rep = rng.choice(((6, 1), (8, 1), (12, 1), (16, 1), (20, 1), (4, 4)))
        else:
            hkv, rep = rng.choice(((1, 8), (2, 6), (4, 4), (8, 4), (8, 1), (2, 3)))
        groups = _log(rng, 1, 8)
        per = _log(rng, 1, 128 // groups)
        t = rng.choice((1, 1, 1, rng.randint(2, 8)))
        # at most the largest listed case's 128 slots x 1024 own keys x 8 heads of 128, and its
        # scores (plain form: slots x heads x rows x keys)
        hi = _log(rng, t, 1024)
        prefix = rng.choice((_log(rng, 1, 16384), _log(rng, 16, 4096), 0))
        while groups * per * hkv * rep * t * (prefix + hi) > 128 * 32 * 16384 or \
                groups * hkv * d * prefix > 16 * 128 * 16384 or \
                groups * per * hkv * d * hi > 128 * 1024 * 8 * 128:
            prefix //= 2
            hi = max(t, hi // 2)
        dt = rng.choice(("bf16", "f16"))
        q, out = rng.choice(((dt, dt), (dt, "f32"), ("f32", "f32")))
        return {"kind": kind, "groups": groups, "per": per, "heads_kv": hkv, "rep": rep, "d": d,
                "t": t, "prefix": prefix, "lo": rng.randint(t, max(t, hi // 2)), "hi": hi,
                "cap": hi + rng.choice((0, 1, 37)), "q": q, "kv": dt, "out": out}
    if kind == "int8":
        m, k, n = _log(rng, 1, 4000), _log(rng, 64, 6000), _log(rng, 64, 6000)
        x = rng.choice(("f32", "f16", "bf16"))
        return {"kind": kind, "m": m, "k": k, "n": n, "bias": rng.random() < 0.5, "x": x,
                "out": rng.choice(("f32", x))}
    return {"kind": kind, "rows": _log(rng, 1, 256), "vocab": _log(rng, 1000, 131072),
            "logits": rng.choice(("f32", "f16", "bf16")),
            "mode": rng.choice(("temperature", "top_k", "top_p", "mixed"))}


# ---------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------

def _spread(lo, hi, n):
    """n lengths from lo to hi, both among them where n allows."""
    return [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)] if n > 1 else [hi]


def _prefix_lens(c):
    """Prompts of a batch differ in length: from three quarters of the longest up."""
    return _spread(c["prefix"] - c["prefix"] // 4, c["prefix"], c["groups"])


def _prepare_prefix(c, g):
    s, hkv, d = c["groups"] * c["per"], c["heads_kv"], c["d"]
    kv = DT[c["kv"]]

    def rand(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)

    lens = torch.tensor(_spread(c["lo"], c["hi"], s), dtype=torch.int32, device="cuda")
    lens = lens[torch.randperm(s, generator=g, device="cuda")].contiguous()
    p = max(1, c["prefix"])  # a cache holds at least one position; the length may be 0
    st = {"q": rand(s, hkv * c["rep"], c["t"], d).to(DT[c["q"]]),
          "pk": rand(c["groups"], hkv, p, d).to(kv), "pv": rand(c["groups"], hkv, p, d).to(kv),
          "plens": torch.tensor(_prefix_lens(c), dtype=torch.int32, device="cuda"),
          # positions past a slot's length hold what an earlier sequence left there
          "ok": rand(s, hkv, c["cap"], d).to(kv), "ov": rand(s, hkv, c["cap"], d).to(kv),
          "olens": lens}
    return st


def _prepare_int8(c, g):
    def rand(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)

    # activations with a few channels much larger than the others, as trained networks have them
    gain = torch.exp(0.7 * rand(c["k"]))
    x = (rand(c["m"], c["k"]) * gain).to(DT[c["x"]])
    w = rand(c["n"], c["k"]) / math.sqrt(c["k"])
    sw = w.abs().amax(1) / 127
    qw = torch.round(w / sw[:, None]).to(torch.int8)
    return {"x": x, "qw": qw, "sw": sw, "b": rand(c["n"]) if c["bias"] else None}


def _prepare_sample(c, g):
    rows, vocab = c["rows"], c["vocab"]

    def uni(*shape):
        return torch.rand(shape, generator=g, device="cuda", dtype=torch.float32)

    # rows from sure (a few tokens far above the rest) to undecided; some tokens ruled out
    sigma = 0.5 + 3.0 * uni(rows, 1)
    l = torch.randn((rows, vocab), generator=g, device="cuda") * sigma
    l = torch.where(uni(rows, vocab) < 8.0 / vocab, l + 6.0 * uni(rows, 1), l)
    l = torch.where(uni(rows, vocab) < 0.03, torch.full_like(l, -math.inf), l)
    st = {"l": l.to(DT[c["logits"]]), "u": uni(rows), "t": 0.2 + 1.1 * uni(rows), "top_k": None,
          "top_p": None, "min_p": None}
    mode = c["mode"]
    if mode in ("top_k", "mixed"):
        st["top_k"] = 1 + (uni(rows) * 99).to(torch.int32)
    if mode in ("top_k", "top_p", "mixed"):
        st["top_p"] = 0.7 + 0.3 * uni(rows)
    if mode == "mixed":  # each row with settings of its own, some with none (temperature 0: greedy)
        st["min_p"] = torch.where(uni(rows) < 0.5, 0.1 * uni(rows), torch.zeros(rows, device="cuda"))
        st["top_k"] = torch.where(uni(rows) < 0.5, st["top_k"], torch.zeros_like(st["top_k"]))
        st["top_p"] = torch.where(uni(rows) < 0.5, st["top_p"], torch.ones(rows, device="cuda"))
        st["t"] = torch.where(uni(rows) < 0.1, torch.zeros(rows, device="cuda"), st["t"])
    return st


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    make = {"prefix": _prepare_prefix, "int8": _prepare_int8, "sample": _prepare_sample}
    return {"case": case, **make[case["kind"]](case, g)}


# ---------------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------------

def _plain_prefix(s):
    c = s["case"]
    gr, per, hkv, rep, t, d = (c[k] for k in ("groups", "per", "heads_kv", "rep", "t", "d"))
    n = gr * per
    q = s["q"].float().reshape(n, hkv, rep * t, d) * d ** -0.5
    qg = q.reshape(gr, per, hkv, rep * t, d).transpose(1, 2).reshape(gr, hkv, per * rep * t, d)
    sp = qg @ s["pk"].float().transpose(2, 3).contiguous()
    so = q @ s["ok"].float().transpose(2, 3).contiguous()
    # row i of a slot stands at own position olens - t + i and sees own keys up to there
    far = torch.arange(sp.shape[3], device=sp.device) >= s["plens"][:, None]
    last = s["olens"][:, None] - t + torch.arange(t, device=so.device)
    hid = torch.arange(so.shape[3], device=so.device) > last[:, :, None]
    hid = hid.repeat(1, rep, 1)[:, None]
    sp = sp.masked_fill(far[:, None, None], -math.inf)
    so = so.masked_fill(hid, -math.inf)
    sp = sp.reshape(gr, hkv, per, rep * t, -1).transpose(1, 2).reshape(n, hkv, rep * t, -1)
    top = torch.maximum(sp.amax(3, keepdim=True), so.amax(3, keepdim=True))
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    sp, so = torch.exp(sp - top), torch.exp(so - top)
    den = sp.sum(3, keepdim=True) + so.sum(3, keepdim=True)
    spg = sp.reshape(gr, per, hkv, rep * t, -1).transpose(1, 2)
    spg = spg.reshape(gr, hkv, per * rep * t, -1)
    o = (spg @ s["pv"].float()).reshape(gr, hkv, per, rep * t, d).transpose(1, 2)
    o = o.reshape(n, hkv, rep * t, d)
    o = (o + so @ s["ov"].float()) / torch.where(den > 0, den, torch.ones_like(den))
    return o.reshape(n, hkv * rep, t, d).to(DT[c["out"]])


def _plain_int8(s):
    x = s["x"].float()
    top = x.abs().amax(1, keepdim=True)
    sx = torch.where(top > 0, top / 127, torch.ones_like(top))
    qx = torch.round(x / sx)
    y = (qx @ s["qw"].float().t().contiguous()) * sx * s["sw"]
    if s["b"] is not None:
        y = y + s["b"]
    return y.to(DT[s["case"]["out"]])


def _plain_sample(s):
    l = s["l"].double()
    rows, vocab = l.shape
    m = l.amax(1, keepdim=True)
    total = torch.exp(l - m).sum(1)
    greedy = s["t"] <= 0
    temp = torch.where(greedy, torch.ones_like(s["t"]), s["t"]).double()
    w = torch.exp((l - m) / temp[:, None])
    keep = torch.ones_like(l, dtype=torch.bool)
    if s["top_k"] is not None or s["top_p"] is not None or s["min_p"] is not None:
        order = torch.sort(s["l"], dim=1, descending=True, stable=True).indices
        sw = torch.gather(w, 1, order)
        kept = torch.ones_like(keep)
        if s["top_k"] is not None:
            k = torch.where(s["top_k"] > 0, s["top_k"], torch.full_like(s["top_k"], vocab))
            kept &= torch.arange(vocab, device=l.device) < k[:, None]
        if s["min_p"] is not None:
            kept &= sw >= s["min_p"].double()[:, None]
        if s["top_p"] is not None:
            sk = torch.where(kept, sw, torch.zeros_like(sw))
            before = torch.cumsum(sk, 1) - sk
            p = s["top_p"].double()[:, None]
            kept &= (before < p * sk.sum(1, keepdim=True)) | (p >= 1)
        keep = torch.zeros_like(keep).scatter_(1, order, kept)
    w = torch.where(keep, w, torch.zeros_like(w))
    cum = torch.cumsum(w, 1)
    # the first index whose cumulative weight passes u times the whole
    hit = (cum > s["u"].double()[:, None] * cum[:, -1:]) & (w > 0)
    tok = torch.where(greedy, l.argmax(1), hit.int().argmax(1))
    first = (l == m).int().argmax(1)  # the lowest index of the maximum
    tok = torch.where(greedy, first, tok)
    lp = torch.gather(l - m, 1, tok[:, None])[:, 0] - torch.log(total)
    return tok.int(), lp.float()


def _own_prefix(s):
    from ffai_amd.kv_cache import KVCache
    from ffai_amd.prefix import PrefixAttention
    c = s["case"]
    if "plan" not in s:  # the caches and the plan over them, which a decoding program keeps
        s["plan"] = PrefixAttention(KVCache.from_tensors(s["pk"], s["pv"], s["plens"]),
                                    KVCache.from_tensors(s["ok"], s["ov"], s["olens"]),
                                    c["heads_kv"] * c["rep"], c["t"], q_dtype=DT[c["q"]],
                                    out_dtype=DT[c["out"]], scale=c["d"] ** -0.5)
    return s["plan"](s["q"])


def _own_int8(s):
    from ffai_amd.int8 import Int8Linear
    if "layer" not in s:  # the layer over its quantized weights, which a program keeps
        s["layer"] = Int8Linear.from_quantized(s["qw"], s["sw"], s["b"])
    return s["layer"](s["x"], out_dtype=DT[s["case"]["out"]])


def _own_sample(s):
    from ffai_amd.sampling import sample
    return sample(s["l"], s["u"], temperature=s["t"], top_k=s["top_k"], top_p=s["top_p"],
                  min_p=s["min_p"])


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"prefix": _own_prefix, "int8": _own_int8, "sample": _own_sample}[kind](state)
    return {"prefix": _plain_prefix, "int8": _plain_int8, "sample": _plain_sample}[kind](state)


# ---------------------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------------------

def _size(name):
    return {"f32": 4, "f16": 2, "bf16": 2}[name]


def work(case):
    c = case
    if c["kind"] == "prefix":
        s, t, hq = c["groups"] * c["per"], c["t"], c["heads_kv"] * c["rep"]
        pl, ol = _prefix_lens(c), _spread(c["lo"], c["hi"], s)
        rows = s * hq * t * c["d"]
        seen = sum(c["per"] * t * n for n in pl)
        seen += sum(max(0, n - t + i + 1) for n in ol for i in range(t))
        return {"bytes": rows * (_size(c["q"]) + _size(c["out"])) +
                2 * (sum(pl) + sum(ol)) * c["heads_kv"] * c["d"] * _size(c["kv"]),
                "flops": 4 * hq * c["d"] * seen}
    if c["kind"] == "int8":
        m, k, n = c["m"], c["k"], c["n"]
        return {"bytes": m * k * _size(c["x"]) + n * k + 4 * n * (2 if c["bias"] else 1) +
                m * n * _size(c["out"]), "flops": 2 * m * n * k}
    # per token: a difference, a scaling, two exponentials (counted as one each) and two sums
    return {"bytes": c["rows"] * (c["vocab"] * _size(c["logits"]) + 28),
            "flops": 6 * c["rows"] * c["vocab"]}


# ---------------------------------------------------------------------------------------------
# In 64 bits, from the definitions
# ---------------------------------------------------------------------------------------------

def _exact_prefix(c, s):
    out = []
    t, rep = c["t"], c["rep"]
    for i, n in enumerate(s["olens"].tolist()):
        g = i // c["per"]
        np_ = int(s["plens"][g])
        k = torch.cat((s["pk"][g, :, :np_], s["ok"][i, :, :n]), 1).double()
        v = torch.cat((s["pv"][g, :, :np_], s["ov"][i, :, :n]), 1).double()
        q = s["q"][i].double().reshape(c["heads_kv"], rep, t, c["d"])
        z = torch.einsum("hrtd,hkd->hrtk", q, k) / math.sqrt(c["d"])
        seen = torch.arange(np_ + n, device=z.device)[None, :] <= \
            (np_ + n - t + torch.arange(t, device=z.device))[:, None]
        z = torch.where(seen, z, torch.full_like(z, -math.inf))
        out.append(torch.einsum("hrtk,hkd->hrtd", torch.softmax(z, 3), v)
                   .reshape(c["heads_kv"] * rep, t, c["d"]))
    return torch.stack(out)


def _exact_int8(c, s):
    x = s["x"].double()
    big = s["x"].float().abs().max(1).values.double()
    # the scale and the quotient are f32 numbers by definition: the f64 quotient rounded once more
    # is the correctly rounded f32 one
    sx = torch.where(big > 0, (big / 127.0).float(), torch.ones_like(big, dtype=torch.float32))
    q = torch.round((x / sx.double()[:, None]).float()).double()
    y = torch.mm(q, s["qw"].double().T) * sx.double()[:, None] * s["sw"].double()[None]
    return y if s["b"] is None else y + s["b"].double()


def _exact_sample(c, s):
    toks, lps = [], []
    par = {k: None if s[k] is None else s[k].double().cpu().numpy()
           for k in ("t", "top_k", "top_p", "min_p", "u")}
    for r, l in enumerate(s["l"].double().cpu().numpy()):
        m = l.max()
        if par["t"][r] <= 0:
            tok = int(np.flatnonzero(l == m)[0])
        else:
            w = np.exp((l - m) / par["t"][r])
            rank = np.lexsort((np.arange(l.size), -l))
            if par["top_k"] is not None and par["top_k"][r] > 0:
                rank = rank[:int(par["top_k"][r])]
            if par["min_p"] is not None:
                rank = rank[w[rank] >= par["min_p"][r]]
            if par["top_p"] is not None and par["top_p"][r] < 1:
                cw = np.cumsum(w[rank])
                rank = rank[:1 + int(np.searchsorted(cw, par["top_p"][r] * cw[-1]))]
            rank = np.sort(rank)
            cw = np.cumsum(w[rank])
            tok = int(rank[np.searchsorted(cw, par["u"][r] * cw[-1], side="right")])
        toks.append(tok)
        lps.append(l[tok] - m - np.log(np.exp(l - m).sum()))
    return (torch.tensor(toks, dtype=torch.int32), torch.tensor(lps, dtype=torch.float64))


def exact(case, seed):
    s = prepare(case, seed)
    make = {"prefix": _exact_prefix, "int8": _exact_int8, "sample": _exact_sample}
    return make[case["kind"]](case, s)
