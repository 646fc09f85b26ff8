"""Microscaled 4-bit floating point: quantisation, its inverse, and the linear
layer on the block-scaled tensor cores.

The format (OCP Microscaling, MXFP4) holds a matrix in 4-bit e2m1 values with
one power-of-two scale per 32 consecutive values of a row: 4.25 bits a value;
include/actcomp.h states the layout and the rounding.  The framework's integer
codes (``actcomp.encode``) compress what is saved; here the products themselves
run on the 4-bit operands (the linear layers of
low_rank_system_profile_backward.py:14-18, forward and both gradients):

  w = quantize(weight)                   # (N, K), once per weight
  w, wt = quantize_pair(weight)          # with the transpose for the backward pass
  y = linear(x, w)                       # x (..., K) -> (..., N)
  y, saved = linear_forward(x, w)        # saved: x in 4 bits, by columns
  dx, dw = linear_backward(dy, saved, wt)

A product contracts over the dimension its operands are blocked along, so a
gradient needs the other direction's blocks: wt is the quantised transpose, and
the weight gradient contracts dy and x over tokens, both quantised by columns.

Waits inside the product are bounded.  One that gives up leaves parts of the
result unwritten and is recorded in the device error word, which
``_lib.load().actcomp_last_device_error`` reads (ACT_E_TIMEOUT).  All functions
compute outside autograd: results carry no graph, whatever the inputs require.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib

_host = _lib.host


@dataclass
class Mx4:
    """A rows x cols matrix in the microscaled 4-bit format: codes (rows,
    ceil(cols / 32) * 16) uint8, scales uint8 in the tensor cores' order, and the
    dtype it was made from."""

    rows: int
    cols: int
    codes: torch.Tensor
    scales: torch.Tensor
    dtype: torch.dtype

    @property
    def shape(self) -> tuple[int, int]:
        return self.rows, self.cols

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()


def quantize(x: torch.Tensor, transpose: bool = False) -> Mx4:
    """x (float32, bfloat16 or float16; leading dimensions are joined) in 4 bits,
    blocks of 32 along the last dimension; with ``transpose`` the joined matrix's
    transpose, blocks along its rows.  A block that holds a NaN or an infinity
    becomes NaN."""
    rows, cols, c, s, ct, st = _host.quantize(x, not transpose, transpose)
    return Mx4(cols, rows, ct, st, x.dtype) if transpose else Mx4(rows, cols, c, s, x.dtype)


def quantize_pair(x: torch.Tensor) -> tuple[Mx4, Mx4]:
    """(quantize(x), quantize(x, transpose=True)) from one read of x."""
    rows, cols, c, s, ct, st = _host.quantize(x, True, True)
    return Mx4(rows, cols, c, s, x.dtype), Mx4(cols, rows, ct, st, x.dtype)


def dequantize(q: Mx4, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """The values of q, (rows, cols) of ``dtype`` (default: what q was made from)."""
    return _host.dequantize(q.rows, q.cols, q.codes, q.scales, dtype or q.dtype)


def matmul(a: Mx4, b: Mx4, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """a . b^T, (a.rows, b.rows), for operands blocked along the shared columns;
    float32 accumulation, rounded once to ``out_dtype`` (default: a's dtype)."""
    if a.cols != b.cols:
        raise ValueError(f"inner dimensions differ: {a.cols} vs {b.cols}")
    return _host.matmul(a.rows, b.rows, a.cols, a.codes, a.scales, b.codes, b.scales, out_dtype or a.dtype)


def linear(x: torch.Tensor, w: Mx4, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """x . w^T for x (..., K) and w (N, K) in 4 bits: x is quantised by rows on
    the way; (..., N) of ``out_dtype`` (default: x's).  One token, and up to four on
    a weight that is not large, take one kernel, the others quantisation and the
    tensor cores."""
    return _host.linear(x, w.rows, w.cols, w.codes, w.scales, out_dtype)


def linear_forward(x: torch.Tensor, w: Mx4, out_dtype: Optional[torch.dtype] = None) -> tuple[torch.Tensor, Mx4]:
    """(linear(x, w), saved): saved is x by columns in 4 bits, all that the
    weight gradient needs of it."""
    if x.shape[-1] != w.cols:
        raise ValueError(f"x has {x.shape[-1]} columns, the weight {w.cols}")
    if _host.one_kernel(x.numel() // w.cols, w.rows, w.cols):
        return linear(x, w, out_dtype), quantize(x, transpose=True)
    q, saved = quantize_pair(x)
    return matmul(q, w, out_dtype).view(x.shape[:-1] + (w.rows,)), saved


def linear_backward(dy: torch.Tensor, saved: Mx4, wt: Mx4,
                    out_dtype: Optional[torch.dtype] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(dx, dw) of :func:`linear_forward`: dx = dy . W with dy (..., N) by rows and
    wt = quantize(weight, transpose=True) (K, N); dw = dy^T . x (N, K), both by
    columns.  ``out_dtype`` defaults to dy's."""
    if dy.shape[-1] != wt.cols or saved.rows != wt.rows:
        raise ValueError(f"dy has {dy.shape[-1]} columns and the saved input {saved.rows} channels, "
                         f"the transposed weight is {wt.rows} x {wt.cols}")
    if dy.numel() // dy.shape[-1] != saved.cols:
        raise ValueError(f"dy has {dy.numel() // dy.shape[-1]} tokens, the saved input {saved.cols}")
    q, qt = quantize_pair(dy)
    dx = matmul(q, wt, out_dtype).view(dy.shape[:-1] + (wt.rows,))
    return dx, matmul(qt, saved, out_dtype)
