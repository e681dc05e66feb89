"""Linear layers in 8-bit integers, attention over a shared prefix and sampling as a generation loop
runs them together: a prompt's keys once, several answers to it, a token per answer and step. Each
stage is held against the 64-bit definition on the inputs that the stage got (integer products and
tokens exactly, attention within its rounding bound), and captured steps against eager ones."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from ffai_amd.int8 import Int8Linear
from ffai_amd.kv_cache import KVCache
from ffai_amd.prefix import PrefixAttention
from ffai_amd.sampling import sample
from oracle import int8 as oracle8
from oracle.prefix import prefix_attend
from oracle.sampling import sample_row

pytestmark = pytest.mark.gpu

GROUPS, PER, HEADS, KV, D, VOCAB, PROMPT, CAP = 2, 3, 4, 2, 64, 9001, 70, 24
DIM, SLOTS = HEADS * D, GROUPS * PER
SETTINGS = dict(temperature=0.8, top_k=40, top_p=0.9, min_p=0.01)
NUCLEUS = dict(temperature=1.3, top_p=0.95)


class Model:
    """One layer of a decoder: token -> embedding -> q, k, v -> attention -> logits -> token."""

    def __init__(self, dev, dtype, seed=0):
        g = torch.Generator().manual_seed(seed)

        def rand(*shape, gain=1.0):
            return (torch.randn(shape, generator=g) * gain).to(dev)

        self.dev, self.dtype = dev, dtype
        self.embed = rand(VOCAB, DIM).to(dtype)
        self.qkv = Int8Linear(rand(DIM + 2 * KV * D, DIM, gain=DIM ** -0.5), rand(DIM + 2 * KV * D, gain=0.1))
        self.out = Int8Linear(rand(DIM, DIM, gain=DIM ** -0.5))
        self.vocab = Int8Linear(rand(VOCAB, DIM, gain=2 * DIM ** -0.5))
        self.prefix = KVCache(GROUPS, KV, PROMPT, D, dtype=dtype, device=dev)
        self.prompt = torch.randint(VOCAB, (GROUPS, PROMPT), generator=g).to(dev)
        x = self.qkv(self.embed[self.prompt])
        _, k, v = self.split(x)
        self.prefix.append(k, v)
        self.prefix.lens.copy_(torch.tensor([PROMPT, PROMPT - 7], dtype=torch.int32))
        self.start()

    def start(self):
        self.own = KVCache(SLOTS, KV, CAP, D, dtype=self.dtype, device=self.dev)
        self.attend = PrefixAttention(self.prefix, self.own, HEADS, q_dtype=self.dtype, scale=D ** -0.5)
        self.tokens = torch.arange(SLOTS, dtype=torch.int32, device=self.dev) * 11
        self.u = torch.empty(SLOTS, device=self.dev)

    @staticmethod
    def split(x):
        return x[..., :DIM], x[..., DIM:DIM + KV * D], x[..., DIM + KV * D:]

    def step(self, settings, seen=None):
        """self.tokens becomes the next tokens; seen: the stages' inputs and outputs go there."""
        x = self.embed[self.tokens.long()]
        h = self.qkv(x)
        q, k, v = self.split(h)
        q = q.view(SLOTS, HEADS, 1, D)
        a = self.attend.step(q, k.unsqueeze(1), v.unsqueeze(1))
        y = self.out(a.view(SLOTS, DIM), out_dtype=torch.float32)
        logits = self.vocab(y + x.float())
        _, lp = sample(logits, self.u, out=self.tokens, **settings)
        if seen is not None:
            seen.update(x=x, h=h, q=q, k=k, v=v, a=a, y=y, logits=logits, tokens=self.tokens.clone(),
                        lp=lp)
        return lp


def np32(t):
    return t.float().cpu().numpy()


def check_linear(layer, x, got):
    q, s = oracle8.quantize_rows(np32(x))
    b = None if layer.bias is None else np32(layer.bias)
    want = oracle8.linear(q, s, layer.qw[:, :layer.in_dim].cpu().numpy(), np32(layer.scale), b)
    w = [torch.from_numpy(want)]
    if b is not None:  # the sum with the bias is one rounding: its neighbours in f32 too
        w += [torch.from_numpy(np.nextafter(want, np.float32(v), dtype=np.float32))
              for v in (-np.inf, np.inf)]
    g = got.cpu()
    assert torch.stack([g == c.to(g.dtype) for c in w]).any(0).all()


def check_attention(m, q, got):
    c = [np32(m.prefix.k), np32(m.prefix.v), m.prefix.lens.cpu().numpy(), np32(m.own.k),
         np32(m.own.v), m.own.lens.cpu().numpy()]
    want, mean, reach = prefix_attend(np32(q), *c, D ** -0.5)
    # f32 scores, weights rounded to the 16-bit type for the second product, a 16-bit result
    n, e, u = PROMPT + CAP, 2.0 ** -24, torch.finfo(m.dtype).eps / 2
    delta = (D + 6) * e * reach[..., None] + (2 * n + 300) * e + 2.0 ** -22
    tol = 2 * delta * mean + u * mean + (u + e) * np.abs(want) + 1e-30
    if m.dtype == torch.float16:  # weights below its least normal
        tol = tol + n * 2.0 ** -25 * max(np.abs(c[1]).max(), np.abs(c[4]).max()) + 2.0 ** -25
    assert (np.abs(got.double().cpu().numpy() - want) <= tol).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("settings", [SETTINGS, NUCLEUS, {}], ids=["filtered", "nucleus", "plain"])
def test_steps_against_the_definitions(gpu, dtype, settings):
    m = Model(gpu, dtype)
    g = torch.Generator().manual_seed(3)
    for i in range(4):
        m.u.copy_(torch.rand(SLOTS, generator=g))
        seen = {}
        m.step(settings, seen)
        assert m.own.lens.tolist() == [i + 1] * SLOTS
        check_linear(m.qkv, seen["x"], seen["h"])
        # the step's keys and values are in the caches
        assert torch.equal(m.own.k[:, :, i].reshape(SLOTS, -1), seen["k"])
        assert torch.equal(m.own.v[:, :, i].reshape(SLOTS, -1), seen["v"])
        check_attention(m, seen["q"], seen["a"])
        check_linear(m.out, seen["a"].view(SLOTS, DIM), seen["y"])
        check_linear(m.vocab, seen["y"] + seen["x"].float(), seen["logits"])
        for r in range(SLOTS):
            want, wlp, _ = sample_row(np32(seen["logits"][r]), m.u[r].item(),
                                      settings.get("temperature", 1.0), settings.get("top_k", 0),
                                      settings.get("top_p", 1.0), settings.get("min_p", 0.0))
            assert seen["tokens"][r].item() == want
            tol = 2.0 ** -18 + 2.0 ** -24 * abs(wlp) + VOCAB * math.exp(-30)
            assert abs(seen["lp"][r].item() - wlp) <= tol


@pytest.mark.parametrize("settings", [SETTINGS, NUCLEUS], ids=["filtered", "nucleus"])
def test_captured_steps(gpu, settings):
    """Replays of a captured step, an answer's reorder between two of them, against eager steps from
    the same start."""
    m = Model(gpu, torch.bfloat16)
    g = torch.Generator().manual_seed(5)
    us = [torch.rand(SLOTS, generator=g).to(gpu) for _ in range(7)]
    parent = torch.tensor([2, 2, 0, 5, 3, 3], dtype=torch.int32, device=gpu)

    def run(step):
        tokens, lps = [], []
        spare = KVCache(SLOTS, KV, CAP, D, dtype=torch.bfloat16, device=gpu)
        for i, u in enumerate(us):
            m.u.copy_(u)
            lp = step()
            if i == 3:
                spare.gather_from(m.own, parent)
                m.own.k.copy_(spare.k), m.own.v.copy_(spare.v), m.own.lens.copy_(spare.lens)
                m.tokens.copy_(m.tokens[parent.long()])
            torch.cuda.synchronize()
            tokens.append(m.tokens.tolist())
            lps.append(lp.clone())
        return tokens, torch.stack(lps)

    want, want_lp = run(lambda: m.step(settings))
    m.start()
    m.u.copy_(us[0])
    m.step(settings)  # warm: the capture finds its allocations made
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lp = m.step(settings)
    m.own.lens.zero_()
    m.tokens.copy_(torch.arange(SLOTS, dtype=torch.int32) * 11)

    def replay():
        graph.replay()
        return lp

    got, got_lp = run(replay)
    assert got == want and torch.equal(got_lp, want_lp)
