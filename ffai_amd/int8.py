"""Linear layers in 8-bit integers on torch device tensors, through include/ffai_int8.h: one scale
per row of activations and per output channel, exact integer sums, any number of rows.

Beside gemv.F16Gemv and gemv.Int8Vocab (a decode step's at most 16 rows): a prompt's tokens, a
batch of sequences, an encoder's frames. No counterpart in the reference.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from . import _lib as L
from .flash_attn import _DT

_PAD = 128  # quantized rows are padded with zeros to a multiple of this


class QuantizedRows(NamedTuple):
    """Rows as ffai_int8_quantize_rows leaves them: q (rows, dim rounded up to 128) int8, zeros past
    `dim`; scale (rows,) f32. Several layers over the same input can share one."""
    q: torch.Tensor
    scale: torch.Tensor
    dim: int


def _rows_view(x: torch.Tensor, dim: int) -> torch.Tensor:
    """x (..., dim) as (rows, dim): a view wherever one stride spans the rows."""
    shape = x.shape
    if len(shape) < 1 or shape[-1] != dim:
        raise ValueError(f"x must be (..., {dim}), not {tuple(shape)}")
    if x.dtype not in _DT:
        raise ValueError(f"x must be f32, f16 or bf16, not {x.dtype}")
    if len(shape) != 2:
        x = x.reshape(-1, dim)
    if not x.is_contiguous() and (x.stride(1) != 1 or (x.shape[0] > 1 and x.stride(0) < dim)):
        x = x.contiguous()
    return x


def quantize_rows(x: torch.Tensor) -> QuantizedRows:
    """x (rows, dim) f32, f16 or bf16 -> its rows in 8-bit integers and their scales."""
    if x.dim() != 2:
        raise ValueError("x must be (rows, dim)")
    rows, dim = x.shape
    x = _rows_view(x, dim)
    q = torch.empty(rows, (dim + _PAD - 1) // _PAD * _PAD, dtype=torch.int8, device=x.device)
    scale = torch.empty(rows, dtype=torch.float32, device=x.device)
    L.call_on(x.device, L.load().ffai_int8_quantize_rows, x.data_ptr(), _DT[x.dtype], rows, dim,
              x.stride(0), q.data_ptr(), q.shape[1], scale.data_ptr())
    return QuantizedRows(q, scale, dim)


class Int8Linear:
    """y = x W^T + b with W (out, in) in 8-bit integers, quantized on the device once."""

    def __init__(self, weight: torch.Tensor, bias: Optional[torch.Tensor] = None):
        if weight.dim() != 2:
            raise ValueError("weight must be (out, in)")
        qr = quantize_rows(weight)
        self._set(qr.q, qr.scale, bias, weight.shape[1])

    @classmethod
    def from_quantized(cls, qw: torch.Tensor, scale: torch.Tensor,
                       bias: Optional[torch.Tensor] = None) -> "Int8Linear":
        """Over weights that are quantized already: qw (out, in) int8, scale (out,) f32. Held as they
        are where their rows are aligned to 16 bytes, else copied once into rows that are."""
        if qw.dim() != 2 or qw.dtype != torch.int8:
            raise ValueError("qw must be (out, in) int8")
        if scale.dtype != torch.float32 or scale.shape != qw.shape[:1] or scale.device != qw.device:
            raise ValueError("scale must be f32 of one value per row of qw, on its device")
        in_dim = qw.shape[1]
        if qw.stride(1) != 1 or qw.stride(0) % 16 or qw.stride(0) < in_dim or qw.data_ptr() % 16:
            held = torch.zeros(qw.shape[0], (in_dim + 15) // 16 * 16, dtype=torch.int8,
                               device=qw.device)
            held[:, :in_dim] = qw
            qw = held
        self = cls.__new__(cls)
        self._set(qw, scale.contiguous(), bias, in_dim)
        return self

    def _set(self, qw, scale, bias, in_dim):
        if bias is not None:
            if bias.shape != scale.shape or bias.device != qw.device:
                raise ValueError("bias must hold one value per output, on the weights' device")
            bias = bias.float().contiguous()
        self.qw, self.scale, self.bias = qw, scale, bias
        self.out_dim, self.in_dim = qw.shape[0], in_dim
        self._w = (qw.data_ptr(), qw.stride(0), scale.data_ptr(),
                   None if bias is None else bias.data_ptr(), self.out_dim)
        self._sized = (0, 0)  # the last number of rows, and its workspace
        self._few = 0  # up to so many rows need no workspace
        while self._few < 64 and self.workspace_bytes(self._few + 1) == 0:
            self._few += 1

    def workspace_bytes(self, rows: int) -> int:
        n = ctypes.c_size_t(0)
        L.check(L.load().ffai_int8_linear_workspace_bytes(rows, self.in_dim, ctypes.byref(n)))
        return n.value

    def _out(self, shape, rows, dtype, out, device):
        if out is None:
            if dtype not in _DT:
                raise ValueError(f"out_dtype must be f32, f16 or bf16, not {dtype}")
            out = torch.empty(shape, dtype=dtype, device=device)
            return out, out.data_ptr(), self.out_dim
        if tuple(out.shape) != tuple(shape) or out.dtype not in _DT or out.device != device or \
                out.dtype != dtype:
            raise ValueError(f"out must be {tuple(shape)} {dtype} on {device}")
        o2 = out if out.dim() == 2 else out.view(rows, self.out_dim)
        if o2.stride(1) != 1:
            raise ValueError("out must be contiguous within a row")
        return out, o2.data_ptr(), o2.stride(0)

    def forward(self, x, out: Optional[torch.Tensor] = None,
                out_dtype: Optional[torch.dtype] = None,
                workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
        """x: (..., in) f32, f16 or bf16 -> (..., out) in x's type or `out_dtype`; or QuantizedRows
        -> (rows, out) f32 or `out_dtype`. `workspace` (workspace_bytes(rows), contents of no
        matter): memory that no call in flight on another stream uses."""
        if isinstance(x, QuantizedRows):
            return self._product(x, out, out_dtype)
        device = self.qw.device
        if x.device != device:
            raise ValueError(f"x must be on {device}, not {x.device}")
        dtype = out_dtype or (x.dtype if out is None else out.dtype)
        x2 = _rows_view(x, self.in_dim)
        rows = x2.shape[0]
        out, yp, ys = self._out((*x.shape[:-1], self.out_dim), rows, dtype, out, device)
        work, n = None, 0
        if workspace is not None:
            if workspace.device != device or not workspace.is_contiguous():
                raise ValueError(f"workspace must be contiguous, on {device}")
            work, n = workspace.data_ptr(), workspace.nbytes
        elif rows > self._few:
            sized = self._sized
            if sized[0] != rows:
                sized = self._sized = (rows, self.workspace_bytes(rows))
            n = sized[1]
            workspace = torch.empty(n, dtype=torch.uint8, device=device)
            work = workspace.data_ptr()
        L.call_on(device, L.load().ffai_int8_linear, x2.data_ptr(), _DT[x2.dtype], x2.stride(0), rows,
                  self.in_dim, *self._w, yp, _DT[dtype], ys, work, n)
        return out

    __call__ = forward

    def _product(self, x: QuantizedRows, out, out_dtype):
        device = self.qw.device
        if x.q.device != device or x.scale.device != device or x.dim != self.in_dim:
            raise ValueError(f"x must be rows of {self.in_dim} on {device}")
        if x.q.dtype != torch.int8 or x.q.dim() != 2 or x.q.stride(1) != 1 or \
                x.q.shape[1] < -(-x.dim // _PAD) * _PAD or x.scale.dtype != torch.float32 or \
                x.scale.shape != x.q.shape[:1] or not x.scale.is_contiguous():
            raise ValueError("x must be as quantize_rows returns it")
        rows = x.q.shape[0]
        dtype = out_dtype or (torch.float32 if out is None else out.dtype)
        out, yp, ys = self._out((rows, self.out_dim), rows, dtype, out, device)
        L.call_on(device, L.load().ffai_int8_product, x.q.data_ptr(), x.q.stride(0),
                  x.scale.data_ptr(), rows, self.in_dim, *self._w, yp, _DT[dtype], ys)
        return out


def plan_info(rows: int, in_dim: int, out_dim: int) -> dict:
    """The tile ffai_int8_product runs for these sizes."""
    info = (ctypes.c_int32 * 4)()
    L.check(L.load().ffai_int8_plan_info(rows, in_dim, out_dim, info))
    return dict(zip(("tile_rows", "tile_outputs", "waves", "workgroups"), info))
