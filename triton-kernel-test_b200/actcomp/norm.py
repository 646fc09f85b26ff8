"""Dropout without a stored mask, layer norm with its backward pass, and both
across a residual branch.

The reference's step (low_rank_system_profile_backward.py) has only the linear
layers; these are what a training step runs between them.  What they save for
the backward pass is a seed and two float32 per row:

  y                    = dropout(x, p, seed)
  dx                   = dropout_backward(dy, p, seed)
  y, mean, rstd        = layer_norm(x, weight, bias)
  dx, dw, db           = layer_norm_backward(dy, x, weight, mean, rstd)
  y, h, mean, rstd     = dropout_add_layer_norm(x, residual, weight, bias, p, seed)
  dx, dresidual, dw, db = dropout_add_layer_norm_backward(dy, h, weight, mean, rstd, p, seed, dh=dh)

Activations are float32, bfloat16 or float16 of any leading shape, normalised
over the last dimension; weight and bias have their dtype or float32.  A row is
one index of the leading dimensions, and a mask depends on (seed, row_offset +
row, column) alone: a rank that holds rows from ``row_offset`` on draws its part
of the whole batch's mask.  ``seed`` is an int in [0, 2^64) or a one-element
int64 CUDA tensor that the kernel reads (so that a captured graph can draw new
masks); ``p`` is held to 16 bits (``round(p * 65536) / 65536``) and the scale
uses the held value."""
from __future__ import annotations

from typing import Optional, Union

import torch

from . import _lib
from .core import _launch, _need_cuda, _ptr

_DT = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
Seed = Union[int, torch.Tensor]

_drop_fn, _drop_args = _lib.entry("actcomp_dropout"), _lib.packer(_lib.DropArgs).pack
_ln_fn, _ln_args = _lib.entry("actcomp_layer_norm"), _lib.packer(_lib.LnArgs).pack
_bwd_fn, _bwd_args = _lib.entry("actcomp_layer_norm_bwd"), _lib.packer(_lib.LnBwdArgs).pack
_bwd_workspace = _lib.entry("actcomp_layer_norm_bwd_workspace")


def _like(x: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor of x's shape (a third of torch.empty's host time)."""
    return torch.empty_like(x, memory_format=torch.contiguous_format)


def _dtype(x: torch.Tensor) -> int:
    dt = _DT.get(x.dtype)
    if dt is None:
        raise TypeError(f"float32, bfloat16 or float16 expected, got {x.dtype}")
    return dt


def _rows2d(x: torch.Tensor, cols: int) -> tuple[torch.Tensor, int]:
    """x as rows of ``cols`` with unit column stride, and its row stride; copied
    only if the leading dimensions have no common stride."""
    if x.is_contiguous():
        return x, cols
    if x.dim() == 1:
        return x.contiguous(), cols
    try:
        x2 = x.view(-1, cols) if x.dim() != 2 else x
    except RuntimeError:
        x2 = x.contiguous().view(-1, cols)
    if x2.stride(1) != 1 and cols != 1 or (x2.shape[0] > 1 and x2.stride(0) < cols):
        x2 = x2.contiguous()
    return x2, max(x2.stride(0), cols)


def _geometry(x: torch.Tensor) -> tuple[int, int]:
    if x.dim() == 0:
        raise ValueError("a tensor of at least one dimension is expected")
    cols = x.shape[-1]
    return (x.numel() // cols if cols else 0), cols


def _same(x: torch.Tensor, **others: Optional[torch.Tensor]) -> None:
    for name, t in others.items():
        if t is None:
            continue
        if t.shape != x.shape or t.dtype != x.dtype or t.device != x.device:
            raise ValueError(f"{name} must have the shape, dtype and device of the activation "
                             f"({tuple(x.shape)} {x.dtype}), got {tuple(t.shape)} {t.dtype} on {t.device}")


def _affine(x: torch.Tensor, cols: int, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor] = None) -> int:
    """Checks weight and bias; returns their dtype code."""
    wdt = None
    for t in (weight, bias):
        if t is None:
            continue
        if t.dim() != 1 or t.numel() != cols or t.device != x.device:
            raise ValueError(f"weight and bias must be vectors of {cols} values on {x.device}")
        if t.dtype != x.dtype and t.dtype != torch.float32:
            raise TypeError(f"weight and bias must be {x.dtype} or float32, got {t.dtype}")
        if wdt is not None and t.dtype != wdt:
            raise TypeError("weight and bias must have one dtype")
        wdt = t.dtype
    return _DT[x.dtype if wdt is None else wdt]


def _vec(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return t if t is None or t.is_contiguous() else t.contiguous()


def _stats(rows: int, x: torch.Tensor, **stats: torch.Tensor) -> list:
    out = []
    for name, t in stats.items():
        if t.dtype != torch.float32 or t.numel() != rows or t.device != x.device:
            raise ValueError(f"{name} must hold {rows} float32 values on {x.device}")
        out.append(t if t.is_contiguous() else t.contiguous())
    return out


def _draw(x: torch.Tensor, p: float, seed: Seed, row_offset: int) -> tuple:
    """(seed, seed_ptr, row_offset) after their checks."""
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout probability must be in [0, 1], got {p}")
    if not 0 <= row_offset < 1 << 63:
        raise ValueError("row_offset must be a non-negative 64-bit integer")
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1 or seed.device != x.device:
            raise ValueError("a seed tensor holds one int64 on the activation's device")
        return 0, seed.data_ptr(), row_offset
    if not 0 <= seed < 1 << 64:
        raise ValueError("seed must be in [0, 2^64)")
    return seed, 0, row_offset


def dropout(x: torch.Tensor, p: float, seed: Seed, row_offset: int = 0,
            out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Each value kept with probability 1 - p and scaled by 1 / (1 - p), else 0.
    ``out`` (contiguous, like x; may be x itself) receives the result."""
    _need_cuda(x)
    dt = _dtype(x)
    rows, cols = _geometry(x)
    seed, seed_ptr, row_offset = _draw(x, p, seed, row_offset)
    if out is None:
        out = _like(x)
    else:
        _same(x, out=out)
        if not out.is_contiguous():
            raise ValueError("out must be contiguous")
    x2, ldx = _rows2d(x, cols)
    _launch("actcomp_dropout", _drop_fn, x.device,
            _drop_args(rows, cols, x2.data_ptr(), ldx, out.data_ptr(), cols, dt, 0, p, seed, seed_ptr, row_offset))
    return out


def dropout_backward(dy: torch.Tensor, p: float, seed: Seed, row_offset: int = 0,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The gradient of :func:`dropout`: dy under the mask of the same arguments."""
    return dropout(dy, p, seed, row_offset, out)


def _forward(x, res, weight, bias, eps, p, draw):
    dt = _dtype(x)
    rows, cols = _geometry(x)
    wdt = _affine(x, cols, weight, bias)
    if cols == 0:
        raise ValueError("layer norm over an empty last dimension")
    if not eps >= 0.0:
        raise ValueError("eps must not be negative")
    x2, ldx = _rows2d(x, cols)
    r2, ldr = _rows2d(res, cols) if res is not None else (None, 0)
    weight, bias = _vec(weight), _vec(bias)
    y = _like(x)
    h = _like(x) if res is not None else None
    mean = x.new_empty(x.shape[:-1], dtype=torch.float32)
    rstd = torch.empty_like(mean)
    _launch("actcomp_layer_norm", _ln_fn, x.device,
            _ln_args(rows, cols, x2.data_ptr(), ldx, _ptr(r2), ldr, _ptr(weight), _ptr(bias), y.data_ptr(), cols,
                     _ptr(h), cols, mean.data_ptr(), rstd.data_ptr(), dt, wdt, eps, 0, p, *draw))
    return y, h, mean, rstd


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, mean, rstd): each row of the last dimension normalised, scaled and
    shifted; mean and 1 / sqrt(var + eps) (float32, the leading shape) are what
    the backward pass needs beside x."""
    _need_cuda(x, weight, bias)
    y, _, mean, rstd = _forward(x, None, weight, bias, eps, 0.0, (0, 0, 0))
    return y, mean, rstd


def dropout_add_layer_norm(x: torch.Tensor, residual: torch.Tensor, weight: Optional[torch.Tensor],
                           bias: Optional[torch.Tensor], p: float, seed: Seed, row_offset: int = 0,
                           eps: float = 1e-5) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, h, mean, rstd) with h = residual + dropout(x) and y = layer_norm(h),
    in one pass; y normalises the float32 sum, h is its rounding to the dtype."""
    _need_cuda(x, residual, weight, bias)
    _same(x, residual=residual)
    return _forward(x, residual, weight, bias, eps, p, _draw(x, p, seed, row_offset))


def _backward(dy, x, weight, mean, rstd, p, draw, dh, fused, bias_grad):
    dt = _dtype(x)
    rows, cols = _geometry(x)
    wdt = _affine(x, cols, weight)
    if cols == 0:
        raise ValueError("layer norm over an empty last dimension")
    mean, rstd = _stats(rows, x, mean=mean, rstd=rstd)
    dy2, lddy = _rows2d(dy, cols)
    x2, ldx = _rows2d(x, cols)
    dh2, lddh = _rows2d(dh, cols) if dh is not None else (None, 0)
    weight = _vec(weight)
    dx = _like(x)
    dr = _like(x) if fused else None
    dw = torch.empty_like(weight) if weight is not None else None
    db = None
    if bias_grad:
        db = torch.empty_like(weight) if weight is not None else x.new_empty((cols,))
    need = _bwd_workspace(rows, cols)
    ws = x.new_empty((max(need, 1),), dtype=torch.uint8)
    _launch("actcomp_layer_norm_bwd", _bwd_fn, x.device,
            _bwd_args(rows, cols, dy2.data_ptr(), lddy, x2.data_ptr(), ldx, _ptr(dh2), lddh, _ptr(weight),
                      mean.data_ptr(), rstd.data_ptr(), dx.data_ptr(), cols, _ptr(dr), cols, _ptr(dw), _ptr(db), dt,
                      wdt, p, *draw),
            ws.data_ptr(), need)
    return dx, dr, dw, db


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, weight: Optional[torch.Tensor], mean: torch.Tensor,
                        rstd: torch.Tensor, bias_grad: bool = True):
    """(dx, dweight, dbias) of :func:`layer_norm` (dweight None without a
    weight, dbias None with bias_grad=False).  The sums over rows run in a fixed
    order: the same inputs give the same bits."""
    _need_cuda(dy, x, weight, mean, rstd)
    _same(x, dy=dy)
    dx, _, dw, db = _backward(dy, x, weight, mean, rstd, 0.0, (0, 0, 0), None, False, bias_grad)
    return dx, dw, db


def dropout_add_layer_norm_backward(dy: torch.Tensor, h: torch.Tensor, weight: Optional[torch.Tensor],
                                    mean: torch.Tensor, rstd: torch.Tensor, p: float, seed: Seed,
                                    row_offset: int = 0, dh: Optional[torch.Tensor] = None, bias_grad: bool = True):
    """(dx, dresidual, dweight, dbias) of :func:`dropout_add_layer_norm` from
    the gradient of y and, if h is used further on, dh, the gradient h gets there."""
    _need_cuda(dy, h, weight, mean, rstd, dh)
    _same(h, dy=dy, dh=dh)
    return _backward(dy, h, weight, mean, rstd, p, _draw(h, p, seed, row_offset), dh, True, bias_grad)
