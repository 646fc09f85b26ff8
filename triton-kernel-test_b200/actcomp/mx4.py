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
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib
from .core import _launch, _need_cuda
from .norm import _DT, _dtype

_desc_args = _lib.packer(_lib.Mx4Desc).pack
_quant_fn, _dequant_fn = _lib.entry("actcomp_mx4_quantize"), _lib.entry("actcomp_mx4_dequantize")
_gemm_fn, _linear_fn = _lib.entry("actcomp_mx4_gemm"), _lib.entry("actcomp_mx4_linear")

#: x's values and scales in a few-token product, bytes of shared memory
_SMALL_BYTES = 160 * 1024

BLOCK = 32


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

    def desc(self) -> bytes:
        """The packed actcomp_mx4 structure."""
        return _desc_args(self.rows, self.cols, self.codes.data_ptr(), self.scales.data_ptr())


def _empty(x: torch.Tensor, rows: int, cols: int) -> Mx4:
    codes = x.new_empty((rows, (cols + 31) // 32 * 16), dtype=torch.uint8)
    scales = x.new_empty(((rows + 127) // 128 * ((cols + 127) // 128) * 512,), dtype=torch.uint8)
    return Mx4(rows, cols, codes, scales, x.dtype)


def _matrix(x: torch.Tensor) -> torch.Tensor:
    """x with its leading dimensions joined to rows and unit column stride."""
    if x.dim() < 1 or x.numel() == 0:
        raise ValueError(f"a non-empty tensor is expected, got shape {tuple(x.shape)}")
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    if x2.shape[1] > 1 and x2.stride(1) != 1 or (x2.shape[0] > 1 and x2.stride(0) < x2.shape[1]):
        x2 = x2.contiguous()
    return x2


def _quantize(x: torch.Tensor, by_rows: bool, by_cols: bool) -> tuple[Optional[Mx4], Optional[Mx4]]:
    _need_cuda(x)
    dt = _dtype(x)
    x2 = _matrix(x)
    rows, cols = x2.shape
    q = _empty(x, rows, cols) if by_rows else None
    qt = _empty(x, cols, rows) if by_cols else None
    _launch("actcomp_mx4_quantize", _quant_fn, x.device, x2.data_ptr(), rows, cols, max(x2.stride(0), cols), dt,
            q.desc() if by_rows else None, qt.desc() if by_cols else None)
    return q, qt


def quantize(x: torch.Tensor, transpose: bool = False) -> Mx4:
    """x (float32, bfloat16 or float16; leading dimensions are joined) in 4 bits,
    blocks of 32 along the last dimension; with ``transpose`` the joined matrix's
    transpose, blocks along its rows.  A block that holds a NaN or an infinity
    becomes NaN."""
    q, qt = _quantize(x, not transpose, transpose)
    return qt if transpose else q


def quantize_pair(x: torch.Tensor) -> tuple[Mx4, Mx4]:
    """(quantize(x), quantize(x, transpose=True)) from one read of x."""
    return _quantize(x, True, True)


def dequantize(q: Mx4, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """The values of q, (rows, cols) of ``dtype`` (default: what q was made from)."""
    dtype = dtype or q.dtype
    if dtype not in _DT:
        raise TypeError(f"float32, bfloat16 or float16 expected, got {dtype}")
    out = q.codes.new_empty((q.rows, q.cols), dtype=dtype)
    _launch("actcomp_mx4_dequantize", _dequant_fn, out.device, q.desc(), out.data_ptr(), q.cols, _DT[dtype])
    return out


def matmul(a: Mx4, b: Mx4, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """a . b^T, (a.rows, b.rows), for operands blocked along the shared columns;
    float32 accumulation, rounded once to ``out_dtype`` (default: a's dtype)."""
    dtype = out_dtype or a.dtype
    if dtype not in _DT:
        raise TypeError(f"float32, bfloat16 or float16 expected, got {dtype}")
    if a.cols != b.cols:
        raise ValueError(f"inner dimensions differ: {a.cols} vs {b.cols}")
    if a.device != b.device:
        raise ValueError(f"operands on {a.device} and {b.device}")
    out = a.codes.new_empty((a.rows, b.rows), dtype=dtype)
    _launch("actcomp_mx4_gemm", _gemm_fn, out.device, a.desc(), b.desc(), out.data_ptr(), b.rows, _DT[dtype])
    return out


def _few_tokens(x: torch.Tensor, w: Mx4, out_dtype: Optional[torch.dtype]) -> bool:
    tokens = x.numel() // w.cols
    return (0 < tokens <= _lib.MX4_LINEAR_TOKENS and tokens * ((w.cols + 31) // 32) * 36 <= _SMALL_BYTES
            and (out_dtype is None or out_dtype is x.dtype or out_dtype is torch.float32))


def _linear_few(x: torch.Tensor, w: Mx4, out_dtype: Optional[torch.dtype]) -> torch.Tensor:
    _need_cuda(x)
    dt = _dtype(x)
    if x.device != w.device:
        raise ValueError(f"operands on {x.device} and {w.device}")
    x2 = _matrix(x)
    dtype = out_dtype or x.dtype
    out = x.new_empty(x.shape[:-1] + (w.rows,), dtype=dtype)
    _launch("actcomp_mx4_linear", _linear_fn, x.device, x2.data_ptr(), x2.shape[0], w.cols, max(x2.stride(0), w.cols),
            dt, w.desc(), out.data_ptr(), w.rows, _DT[dtype])
    return out


def linear(x: torch.Tensor, w: Mx4, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """x . w^T for x (..., K) and w (N, K) in 4 bits: x is quantised by rows on
    the way; (..., N) of ``out_dtype`` (default: x's).  Up to four tokens take one
    kernel that reads the weight at memory speed, more the tensor cores."""
    if x.shape[-1] != w.cols:
        raise ValueError(f"x has {x.shape[-1]} columns, the weight {w.cols}")
    if _few_tokens(x, w, out_dtype):
        return _linear_few(x, w, out_dtype)
    return matmul(quantize(x), w, out_dtype).view(x.shape[:-1] + (w.rows,))


def linear_forward(x: torch.Tensor, w: Mx4, out_dtype: Optional[torch.dtype] = None) -> tuple[torch.Tensor, Mx4]:
    """(linear(x, w), saved): saved is x by columns in 4 bits, all that the
    weight gradient needs of it."""
    if x.shape[-1] != w.cols:
        raise ValueError(f"x has {x.shape[-1]} columns, the weight {w.cols}")
    if _few_tokens(x, w, out_dtype):
        return _linear_few(x, w, out_dtype), quantize(x, transpose=True)
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
    dx = matmul(q, wt, out_dtype or dy.dtype).view(dy.shape[:-1] + (wt.rows,))
    return dx, matmul(qt, saved, out_dtype or dy.dtype)
