"""Attention of many slots over a shared prefix and their own keys, through include/ffai_prefix.h.

The reference restores a whole decoder state per beam
(crates/ffai-mercury/src/asr/decoder.rs:559-583): every beam holds its own copy of the prompt's
keys. Here a prompt's K/V rows live once in a prefix cache (one slot per group of sequences, filled
by ``KVCache.append``), and each sequence's own ``KVCache`` slot holds only what came since; a beam
step's ``gather_from`` then moves the own rows alone.

    prefix = KVCache(groups, heads, prompt_capacity, head_dim, dtype)
    own = KVCache(groups * beams, heads, capacity, head_dim, dtype)
    attend = PrefixAttention(prefix, own, heads_q, scale=head_dim ** -0.5)
    own.append(k_new, v_new); out = attend(q)
"""

from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _lib as L
from .flash_attn import _DT
from .kv_cache import KVCache


class PrefixAttention:
    """The attention of `q_len` query rows per slot over `prefix` (one slot per group; slot s of
    `own` belongs to group s // (own.slots // prefix.slots)) and `own`, both 16-bit caches of one
    layer. Called with q (slots, heads_q, q_len, head_dim) of `q_dtype` it returns the same shape
    in `out_dtype`. The caches' lengths are read on the device at each call, so the object stays
    valid while they grow; it holds the caches, not their contents."""

    def __init__(self, prefix: KVCache, own: KVCache, heads_q: int, q_len: int = 1, *,
                 q_dtype: Optional[torch.dtype] = None, out_dtype: Optional[torch.dtype] = None,
                 scale: float = 1.0):
        if prefix.layers is not None or own.layers is not None:
            raise ValueError("attend one layer: PrefixAttention(prefix.layer(l), own.layer(l), ...)")
        if prefix.k.device != own.k.device:
            raise ValueError("prefix and own caches must be on one device")
        self.prefix, self.own = prefix, own
        self.heads_q, self.q_len, self.scale = int(heads_q), int(q_len), float(scale)
        self.q_dtype = own.k.dtype if q_dtype is None else q_dtype
        self.out_dtype = self.q_dtype if out_dtype is None else out_dtype
        if self.q_dtype not in _DT or self.out_dtype not in _DT:
            raise ValueError("q_dtype and out_dtype are f32, f16 or bf16")
        self.shape = (own.slots, self.heads_q, self.q_len, own.head_dim)
        self.device = own.k.device
        # the descriptors, built once: a call only fills in pointers
        self._views = (prefix.view(), own.view())
        self._refs = tuple(ctypes.byref(v) for v in self._views)
        n = ctypes.c_size_t(0)
        rc = L.load().ffai_prefix_attn_workspace_bytes(*self._refs, self.heads_q, self.q_len,
                                                       ctypes.byref(n))
        if L.check(rc) == L.FFAI_DECLINED:
            raise ValueError(f"not served: {L.last_error()}")
        self.workspace_bytes = n.value
        self._strides = {}

    def _stride_array(self, t: torch.Tensor):
        s = t.stride()
        a = self._strides.get(s)
        if a is None:
            if s[3] != 1:
                raise ValueError("head_dim must be contiguous (stride 1)")
            a = self._strides[s] = (ctypes.c_int64 * 3)(*s[:3])
        return a

    def plan(self) -> dict:
        """The launch plan: query rows that share a prefix K/V head, key pieces of the prefix and
        of a slot's own keys, workgroups, prefix rows per workgroup."""
        info = (ctypes.c_int32 * 5)()
        L.check(L.load().ffai_prefix_attn_plan_info(*self._refs, self.heads_q, self.q_len, info))
        return dict(zip(("rows", "prefix_pieces", "own_pieces", "workgroups", "row_block"), info))

    def forward(self, q: torch.Tensor, out: Optional[torch.Tensor] = None,
                workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
        """`workspace` (at least `workspace_bytes`, contents of no matter): memory that no call in
        flight on another stream, nor another graph replayed beside this one, uses."""
        if q.shape != self.shape or q.dtype != self.q_dtype or q.device != self.device:
            raise ValueError(f"q must be {self.shape} {self.q_dtype} on {self.device}, "
                             f"not {tuple(q.shape)} {q.dtype} on {q.device}")
        if out is None:
            out = torch.empty(self.shape, dtype=self.out_dtype, device=self.device)
        elif out.shape != self.shape or out.dtype != self.out_dtype or out.device != self.device:
            raise ValueError(f"out must be {self.shape} {self.out_dtype} on {self.device}")
        work, n = None, 0
        if workspace is not None:
            if workspace.device != self.device or not workspace.is_contiguous():
                raise ValueError(f"workspace must be contiguous, on {self.device}")
            work, n = workspace.data_ptr(), workspace.nbytes
        elif self.workspace_bytes:
            n = self.workspace_bytes
            workspace = torch.empty(n, dtype=torch.uint8, device=self.device)
            work = workspace.data_ptr()
        L.call_on(self.device, L.load().ffai_prefix_attn_fwd, *self._refs, q.data_ptr(),
                  _DT[self.q_dtype], self.heads_q, self.q_len, self._stride_array(q), self.scale,
                  out.data_ptr(), _DT[self.out_dtype], self._stride_array(out), work, n)
        return out

    __call__ = forward

    def step(self, q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor,
             out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """A decode step: append this step's K/V projections, (slots, q_len, heads * head_dim), to
        the own cache, then attend. The counterpart of kv_cache.self_attention_step, with each
        slot at its own length."""
        if k_new.dim() != 3 or k_new.shape[1] != self.q_len:
            raise ValueError(f"k_new and v_new must be (slots, {self.q_len}, heads * head_dim)")
        self.own.append(k_new, v_new)
        return self.forward(q, out=out)


def prefix_attention(q: torch.Tensor, prefix: KVCache, own: KVCache, *, scale: float = 1.0,
                     out_dtype: Optional[torch.dtype] = None,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One call without keeping a PrefixAttention."""
    if q.dim() != 4:
        raise ValueError("q must be (slots, heads_q, q_len, head_dim)")
    if out is not None and out_dtype is None:
        out_dtype = out.dtype
    return PrefixAttention(prefix, own, q.shape[1], q.shape[2], q_dtype=q.dtype,
                           out_dtype=out_dtype, scale=scale)(q, out=out)
