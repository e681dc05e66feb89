"""Sampling a token per row of logits on the device, through include/ffai_sample.h.

What follows gemv.Int8Vocab in a step that samples (the reference does it on the host,
crates/ffai-mercury/src/asr/decoder.rs:650-847): temperature, top-k, min-p and top-p from given
uniform numbers, and the token's log-probability. The header says exactly which token that is.
"""

from __future__ import annotations

import ctypes
import functools
from typing import Optional, Union

import torch

from . import _lib as L
from .flash_attn import _DT

Setting = Union[None, float, int, torch.Tensor]


@functools.lru_cache(maxsize=256)
def workspace_bytes(rows: int, vocab: int) -> int:
    n = ctypes.c_size_t(0)
    L.check(L.load().ffai_sample_workspace_bytes(rows, vocab, ctypes.byref(n)))
    return n.value


def _setting(x: Setting, off, dtype, rows: int, device, name: str):
    """(pointer, value for all rows) of one setting."""
    if x is None:
        return None, off
    if not isinstance(x, torch.Tensor):
        return None, x
    if x.dtype != dtype or x.shape != (rows,) or x.device != device or not x.is_contiguous():
        raise ValueError(f"{name} must be a number or a contiguous {dtype} tensor of {rows} on {device}")
    return x.data_ptr(), off


def sample(logits: torch.Tensor, u: torch.Tensor, *, temperature: Setting = None,
           top_k: Setting = None, top_p: Setting = None, min_p: Setting = None,
           logprobs: bool = True, out: Optional[torch.Tensor] = None,
           workspace: Optional[torch.Tensor] = None):
    """logits (rows, vocab) f32, f16 or bf16; u (rows,) f32 in [0, 1). Each setting is a number for
    every row, a tensor of one per row (temperature, top_p, min_p f32; top_k int32), or None
    (temperature 1, no filter). Returns (tokens int32 (rows,), log-probabilities f32 (rows,) or
    None). Temperature 0 takes the first maximum; a row with nothing to choose from gives -1.
    `out`: an int32 tensor for the tokens. `workspace` (workspace_bytes(rows, vocab), contents of no
    matter): memory that no call in flight on another stream uses."""
    if logits.dim() != 2 or logits.dtype not in _DT:
        raise ValueError("logits must be (rows, vocab) f32, f16 or bf16")
    rows, vocab = logits.shape
    if vocab > 1 and logits.stride(1) != 1:
        raise ValueError("logits must be contiguous within a row")
    device = logits.device
    if u.dtype != torch.float32 or u.shape != (rows,) or u.device != device or not u.is_contiguous():
        raise ValueError(f"u must be a contiguous f32 tensor of {rows} on {device}")
    t = _setting(temperature, 1.0, torch.float32, rows, device, "temperature")
    k = _setting(top_k, 0, torch.int32, rows, device, "top_k")
    p = _setting(top_p, 1.0, torch.float32, rows, device, "top_p")
    mp = _setting(min_p, 0.0, torch.float32, rows, device, "min_p")
    if out is None:
        out = torch.empty(rows, dtype=torch.int32, device=device)
    elif out.dtype != torch.int32 or out.shape != (rows,) or out.device != device or \
            not out.is_contiguous():
        raise ValueError(f"out must be a contiguous int32 tensor of {rows} on {device}")
    lp = torch.empty_like(u) if logprobs else None
    if workspace is None:
        n = workspace_bytes(rows, vocab)
        workspace = torch.empty(n, dtype=torch.uint8, device=device)
    elif workspace.device != device or not workspace.is_contiguous():
        raise ValueError(f"workspace must be contiguous, on {device}")
    else:
        n = workspace.nbytes
    L.call_on(device, L.load().ffai_sample, logits.data_ptr(), _DT[logits.dtype], rows, vocab,
              logits.stride(0), *t, *k, *p, *mp, u.data_ptr(), out.data_ptr(),
              None if lp is None else lp.data_ptr(), workspace.data_ptr(), n)
    return out, lp
