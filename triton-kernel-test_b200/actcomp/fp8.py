"""8-bit floating point with a power-of-two scale per block of 128: quantisation, its
inverse, the linear layer on the block-scaled tensor cores, and the norm before it.

The scale of a block is the smallest power of two under which its largest magnitude
fits (include/actcomp.h states the format): floating-point codes lose nothing by it,
and the tensor cores apply it themselves.  Where :mod:`actcomp.mx4` holds 4.25 bits a
value, this holds 8.06 with four significand bits.  The linear layers of
low_rank_system_profile_backward.py:14-18, forward and both gradients:

  w = quantize_weight(weight)            # (N, K), once per weight; serves both directions
  y = linear(x, w)                       # x (..., K) -> (..., N)
  y, saved = linear_forward(x, w)        # saved: x in 8 bits, by columns
  dx, dw = linear_backward(dy, saved, w)

and the norm that gives a layer its input in 8 bits:

  q, h, rstd = add_rms_norm(x, residual, norm_weight)
  y = matmul(q, w)

A product contracts over the dimension its operands are blocked along.  Activations
and gradients have 1 x 128 blocks along their rows, for the weight gradient (which
contracts over tokens) down their columns; a weight has 128 x 128 tiles, which read
either way.  Codes stay in the matrix's own orientation.

Waits inside the product are bounded.  One that gives up leaves parts of the result
unwritten and is recorded in the device error word, which
``_lib.load().actcomp_last_device_error`` reads (ACT_E_TIMEOUT).  All functions
compute outside autograd: results carry no graph, whatever the inputs require.
"""
from __future__ import annotations

from dataclasses import dataclass, replace
from typing import Optional

import torch

from . import _lib

_host = _lib.host
#: code formats: largest value 448 with three mantissa bits, 57344 with two
FORMATS = ("e4m3", "e5m2")
_ROWS, _COLS, _TILES = 0, 1, 2


def _format(name: str) -> int:
    if name not in FORMATS:
        raise ValueError(f"format must be one of {FORMATS}, got {name!r}")
    return FORMATS.index(name)


@dataclass(slots=True)
class Fp8:
    """A rows x cols matrix in 8-bit floating point, a scale per 128 values of a row or
    (``tiles``) per 128 x 128.  ``transposed``: codes hold the transpose, cols x rows,
    each row padded to 16 bytes; scales are uint8 exponents in the tensor cores' order;
    dtype is what it was made from."""

    rows: int
    cols: int
    codes: torch.Tensor
    scales: torch.Tensor
    dtype: torch.dtype
    format: str = "e4m3"
    tiles: bool = False
    transposed: bool = False

    @property
    def shape(self) -> tuple[int, int]:
        return self.rows, self.cols

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()

    def t(self) -> "Fp8":
        """The transpose, over the same buffers; its blocks have to read either way."""
        if not self.tiles:
            raise ValueError("blocks of 1 x 128 do not read as blocks of the transpose")
        return replace(self, rows=self.cols, cols=self.rows, transposed=not self.transposed)


def _stored(q: Fp8) -> tuple:
    """(rows, cols, codes, scales, format, block, transposed) of what the buffers hold."""
    rows, cols = (q.cols, q.rows) if q.transposed else (q.rows, q.cols)
    block = _TILES if q.tiles else _COLS if q.transposed else _ROWS
    return rows, cols, q.codes, q.scales, _format(q.format), block, q.transposed


def quantize(x: torch.Tensor, transpose: bool = False, format: str = "e4m3") -> Fp8:
    """x (float32, bfloat16 or float16; leading dimensions are joined) in 8 bits, blocks
    of 128 along the last dimension; with ``transpose`` the joined matrix's transpose,
    blocks along its rows.  A block that holds a NaN or an infinity becomes NaN."""
    rows, cols, c, s, ct, st = _host.fp8_quantize(x, not transpose, transpose, False, _format(format))
    if transpose:
        return Fp8(cols, rows, ct, st, x.dtype, format, transposed=True)
    return Fp8(rows, cols, c, s, x.dtype, format)


def quantize_pair(x: torch.Tensor, format: str = "e4m3") -> tuple[Fp8, Fp8]:
    """(quantize(x), quantize(x, transpose=True)) from one read of x."""
    rows, cols, c, s, ct, st = _host.fp8_quantize(x, True, True, False, _format(format))
    return Fp8(rows, cols, c, s, x.dtype, format), Fp8(cols, rows, ct, st, x.dtype, format, transposed=True)


def quantize_weight(x: torch.Tensor, format: str = "e4m3") -> Fp8:
    """x in 8 bits with a scale per 128 x 128: products read it, and its :meth:`Fp8.t`,
    from the same buffers."""
    rows, cols, c, s, _, _ = _host.fp8_quantize(x, False, False, True, _format(format))
    return Fp8(rows, cols, c, s, x.dtype, format, tiles=True)


def dequantize(q: Fp8, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """The values of q, (rows, cols) of ``dtype`` (default: what q was made from); for a
    matrix that is held transposed the transposed view of its values as they lie."""
    rows, cols, codes, scales, fmt, block, transposed = _stored(q)
    v = _host.fp8_dequantize(rows, cols, codes, scales, fmt, block, dtype or q.dtype)
    return v.t() if transposed else v


def matmul(a: Fp8, b: Fp8, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """a . b^T, (a.rows, b.rows), for operands blocked along the shared columns;
    float32 accumulation, rounded once to ``out_dtype`` (default: a's dtype)."""
    if a.cols != b.cols:
        raise ValueError(f"inner dimensions differ: {a.cols} vs {b.cols}")
    return _host.fp8_matmul(_stored(a), _stored(b), out_dtype or a.dtype)


def linear(x: torch.Tensor, w: Fp8, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """x . w^T for x (..., K) and w (N, K) in 8 bits: x is quantised by rows on the way;
    (..., N) of ``out_dtype`` (default: x's)."""
    return _host.fp8_linear(x, _stored(w), out_dtype)


def linear_forward(x: torch.Tensor, w: Fp8, out_dtype: Optional[torch.dtype] = None) -> tuple[torch.Tensor, Fp8]:
    """(linear(x, w), saved): saved is x by columns in 8 bits, all that the weight
    gradient needs of it."""
    if x.shape[-1] != w.cols:
        raise ValueError(f"x has {x.shape[-1]} columns, the weight {w.cols}")
    q, saved = quantize_pair(x)
    return matmul(q, w, out_dtype).view(x.shape[:-1] + (w.rows,)), saved


def linear_backward(dy: torch.Tensor, saved: Fp8, w: Fp8, out_dtype: Optional[torch.dtype] = None,
                    grad_format: str = "e4m3") -> tuple[torch.Tensor, torch.Tensor]:
    """(dx, dw) of :func:`linear_forward`: dx = dy . W with dy (..., N) by rows and the
    weight's tiles; dw = dy^T . x (N, K), both by columns.  ``out_dtype`` defaults to
    dy's; ``grad_format`` is what dy is held in."""
    if not w.tiles:
        raise ValueError("the input gradient needs the weight by tiles (quantize_weight)")
    if dy.shape[-1] != w.rows or saved.rows != w.cols:
        raise ValueError(f"dy has {dy.shape[-1]} columns and the saved input {saved.rows} channels, "
                         f"the weight is {w.rows} x {w.cols}")
    if dy.numel() // dy.shape[-1] != saved.cols:
        raise ValueError(f"dy has {dy.numel() // dy.shape[-1]} tokens, the saved input {saved.cols}")
    q, qt = quantize_pair(dy, grad_format)
    dx = matmul(q, w.t(), out_dtype).view(dy.shape[:-1] + (w.cols,))
    return dx, matmul(qt, saved, out_dtype)


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: float = 1e-5) -> tuple[Fp8, torch.Tensor]:
    """(q, rstd): :func:`actcomp.norm.rms_norm` with its output by rows in 8 bits (e4m3),
    rounded from the float32 result; leading dimensions are joined in q."""
    rows, cols, codes, scales, _, rstd = _host.rms_norm_fp8(x, None, weight, eps)
    return Fp8(rows, cols, codes, scales, x.dtype), rstd


def add_rms_norm(x: torch.Tensor, residual: torch.Tensor, weight: Optional[torch.Tensor] = None,
                 eps: float = 1e-5) -> tuple[Fp8, torch.Tensor, torch.Tensor]:
    """(q, h, rstd) of h = x + residual: :func:`actcomp.norm.add_rms_norm` with y in 8
    bits, as :func:`rms_norm`."""
    rows, cols, codes, scales, h, rstd = _host.rms_norm_fp8(x, residual, weight, eps)
    return Fp8(rows, cols, codes, scales, x.dtype), h, rstd
