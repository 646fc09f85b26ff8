"""Dropout without a stored mask, layer norm with its backward pass, both across a
residual branch, and root-mean-square norm.

The reference's step (low_rank_system_profile_backward.py) has only the linear
layers; these are what a training step runs between them.  What they save for
the backward pass is a seed and two float32 per row:

  y                    = dropout(x, p, seed)
  dx                   = dropout_backward(dy, p, seed)
  y, mean, rstd        = layer_norm(x, weight, bias)
  dx, dw, db           = layer_norm_backward(dy, x, weight, mean, rstd)
  y, h, mean, rstd     = dropout_add_layer_norm(x, residual, weight, bias, p, seed)
  dx, dresidual, dw, db = dropout_add_layer_norm_backward(dy, h, weight, mean, rstd, p, seed, dh=dh)
  y, rstd              = rms_norm(x, weight)
  y, h, rstd           = add_rms_norm(x, residual, weight)
  dx, dw               = rms_norm_backward(dy, x or h, weight, rstd, dh=dh)

(:func:`actcomp.fp8.rms_norm` and :func:`actcomp.fp8.add_rms_norm` give y in 8 bits.)

Activations are float32, bfloat16 or float16 of any leading shape, normalised
over the last dimension; weight and bias have their dtype or float32.  A row is
one index of the leading dimensions, and a mask depends on (seed, row_offset +
row, column) alone: a rank that holds rows from ``row_offset`` on draws its part
of the whole batch's mask.  ``seed`` is an int in [0, 2^64) or a one-element
int64 CUDA tensor that the kernel reads (so that a captured graph can draw new
masks); ``p`` is held to 16 bits (``round(p * 65536) / 65536``) and the scale
uses the held value.

Waits inside the norms' kernels are bounded.  One that gives up leaves NaN in
the rows that its part of the device had and in the weight gradients, and is
recorded in the device error word, which
``_lib.load().actcomp_last_device_error`` reads (ACT_E_TIMEOUT).

All functions compute outside autograd: results carry no graph, whatever the inputs
require."""
from __future__ import annotations

from typing import Optional, Union

import torch

from . import _lib

_host = _lib.host
Seed = Union[int, torch.Tensor]


def dropout(x: torch.Tensor, p: float, seed: Seed, row_offset: int = 0,
            out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Each value kept with probability 1 - p and scaled by 1 / (1 - p), else 0.
    ``out`` (contiguous, like x; may be x itself) receives the result; where it lies
    over other parts of x, x is copied first."""
    return _host.dropout(x, p, seed, row_offset, out)


def dropout_backward(dy: torch.Tensor, p: float, seed: Seed, row_offset: int = 0,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The gradient of :func:`dropout`: dy under the mask of the same arguments."""
    return _host.dropout(dy, p, seed, row_offset, out)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, mean, rstd): each row of the last dimension normalised, scaled and
    shifted; mean and 1 / sqrt(var + eps) (float32, the leading shape) are what
    the backward pass needs beside x."""
    return _host.layer_norm(x, weight, bias, eps)


def dropout_add_layer_norm(x: torch.Tensor, residual: torch.Tensor, weight: Optional[torch.Tensor],
                           bias: Optional[torch.Tensor], p: float, seed: Seed, row_offset: int = 0,
                           eps: float = 1e-5) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, h, mean, rstd) with h = residual + dropout(x) and y = layer_norm(h),
    in one pass; y normalises the float32 sum, h is its rounding to the dtype."""
    return _host.branch(x, residual, weight, bias, p, seed, row_offset, eps)


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, weight: Optional[torch.Tensor], mean: torch.Tensor,
                        rstd: torch.Tensor, bias_grad: bool = True, bias_dtype: Optional[torch.dtype] = None):
    """(dx, dweight, dbias) of :func:`layer_norm` (dweight None without a
    weight, dbias None with bias_grad=False), the two sums in the weight's dtype;
    without a weight dbias is in ``bias_dtype`` (the bias's: the activation's, which
    is the default, or float32).  They run over the rows in a fixed order: the same
    inputs give the same bits."""
    return _host.layer_norm_backward(dy, x, weight, mean, rstd, bias_grad, bias_dtype)


def dropout_add_layer_norm_backward(dy: torch.Tensor, h: torch.Tensor, weight: Optional[torch.Tensor],
                                    mean: torch.Tensor, rstd: torch.Tensor, p: float, seed: Seed,
                                    row_offset: int = 0, dh: Optional[torch.Tensor] = None, bias_grad: bool = True,
                                    bias_dtype: Optional[torch.dtype] = None):
    """(dx, dresidual, dweight, dbias) of :func:`dropout_add_layer_norm` from
    the gradient of y and, if h is used further on, dh, the gradient h gets there.
    ``bias_grad`` and ``bias_dtype`` as in :func:`layer_norm_backward`."""
    return _host.branch_backward(dy, h, weight, mean, rstd, p, seed, row_offset, dh, bias_grad, bias_dtype)


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None,
             eps: float = 1e-5) -> tuple[torch.Tensor, torch.Tensor]:
    """(y, rstd): each row of the last dimension over the root of its mean square, times
    weight; rstd = 1 / sqrt(mean of squares + eps) (float32, the leading shape) is what
    the backward pass needs beside x."""
    return _host.rms_norm(x, weight, eps)


def add_rms_norm(x: torch.Tensor, residual: torch.Tensor, weight: Optional[torch.Tensor] = None,
                 eps: float = 1e-5) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, h, rstd) with h = x + residual and y = rms_norm(h), in one pass; y normalises
    the float32 sum, h is its rounding to the dtype."""
    return _host.add_rms_norm(x, residual, weight, eps)


def rms_norm_backward(dy: torch.Tensor, x: torch.Tensor, weight: Optional[torch.Tensor], rstd: torch.Tensor,
                      dh: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(dx, dweight) of :func:`rms_norm`, or with x = h of :func:`add_rms_norm`, whose x
    and residual both have the gradient dx; dh is the gradient that h gets where it is
    used further on.  dweight (None without a weight) has the weight's dtype; its sum
    runs over the rows in a fixed order: the same inputs give the same bits."""
    return _host.rms_norm_backward(dy, x, weight, rstd, dh)
