"""torch custom ops (namespace ``actcomp``) over the C ABI.

Each op is functional (returns new tensors), has a fake implementation for
meta/abstract tracing, and launches on the current CUDA stream.  The
reference-named functions in :mod:`actcomp.reference_api` call these ops.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import core, fp8, loss, mx4, norm, refcompat

_U8, _F32, _BF = torch.uint8, torch.float32, torch.bfloat16


def _empty(shape, dtype, like):
    return torch.empty(shape, dtype=dtype, device=like.device)


# ---------------------------------------------------------------- reference-compatible
@torch.library.custom_op("actcomp::rc_encode", mutates_args=())
def rc_encode(l: torch.Tensor, r: torch.Tensor, x: torch.Tensor, s: torch.Tensor, bits: int, outlier: float,
              flags: int) -> tuple[torch.Tensor, torch.Tensor]:
    return refcompat.encode(l, r, x, s, bits, outlier, flags)


@rc_encode.register_fake
def _(l, r, x, s, bits, outlier, flags):
    B, M, N = x.shape
    return _empty((B, M, N), _BF, x), _empty((B, M, N * bits // 8), _U8, x)


@torch.library.custom_op("actcomp::rc_decode", mutates_args=())
def rc_decode(l: torch.Tensor, r: torch.Tensor, q: torch.Tensor, o: Optional[torch.Tensor], s: torch.Tensor,
              bits: int, flags: int, op: int, y: Optional[torch.Tensor]) -> torch.Tensor:
    return refcompat.decode(l, r, q, o, s, bits, flags, op, y)


@rc_decode.register_fake
def _(l, r, q, o, s, bits, flags, op, y):
    B, M, W = q.shape
    return _empty((B, M, W * 8 // bits), _BF, q)


@torch.library.custom_op("actcomp::lowrank_add", mutates_args=())
def lowrank_add(l: torch.Tensor, r: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
    return refcompat.lowrank_add(l, r, x)


@lowrank_add.register_fake
def _(l, r, x):
    return _empty(x.shape, _BF, x)


# ---------------------------------------------------------------- channel-group format
def _basis(basis_t, basis, basis_tile=None):
    if basis is None or basis.numel() == 0:
        return None
    return core.Basis(basis_t, basis, basis_tile)


@torch.library.custom_op("actcomp::cg_encode", mutates_args=())
def cg_encode(x: torch.Tensor, basis_t: Optional[torch.Tensor], basis: Optional[torch.Tensor],
              basis_tile: Optional[torch.Tensor], outlier_idx: Optional[torch.Tensor], bits: int, group: int,
              wht: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    c = core.encode(x, _basis(basis_t, basis, basis_tile), outlier_idx, bits=bits, group=group, wht=wht)
    e = x.new_empty((0,))
    return (c.codes, c.scales, c.lowrank if c.rank else e.to(_F32), c.outliers if c.n_outlier else e)


@cg_encode.register_fake
def _(x, basis_t, basis, basis_tile, outlier_idx, bits, group, wht):
    T = x.numel() // x.shape[-1]
    H = x.shape[-1]
    r = 0 if basis is None else basis.shape[-1]
    k = 0 if outlier_idx is None else outlier_idx.shape[-1]
    return (_empty((T, H * bits // 8), _U8, x), _empty((T, H // group), _F32, x),
            _empty((T, r) if r else (0,), _F32, x), _empty((T, k) if k else (0,), _BF, x))


def _compressed(shape, codes, scales, lowrank, outliers, outlier_idx, basis_t, basis, basis_tile, bits, group, wht):
    batch = shape[0] if len(shape) == 3 else 1
    T, H = shape[-2], shape[-1]
    b = _basis(basis_t, basis, basis_tile)
    k = 0 if outlier_idx is None else outlier_idx.shape[-1]
    return core.Compressed(T, H, bits, group, wht, batch, codes, scales, lowrank if b else None,
                           outliers if k else None, outlier_idx.reshape(batch, -1) if k else None, b)


@torch.library.custom_op("actcomp::cg_consume", mutates_args=())
def cg_consume(shape: list[int], codes: torch.Tensor, scales: torch.Tensor, lowrank: torch.Tensor,
               outliers: torch.Tensor, outlier_idx: Optional[torch.Tensor], basis_t: Optional[torch.Tensor],
               basis: Optional[torch.Tensor], basis_tile: Optional[torch.Tensor], bits: int, group: int, wht: bool,
               op: int, y: Optional[torch.Tensor]) -> torch.Tensor:
    c = _compressed(shape, codes, scales, lowrank, outliers, outlier_idx, basis_t, basis, basis_tile, bits, group,
                    wht)
    if op == 0:
        return core.decode(c).reshape(shape)
    return core._consume(c, op, y.reshape(shape)).reshape(shape)


@cg_consume.register_fake
def _(shape, codes, scales, lowrank, outliers, outlier_idx, basis_t, basis, basis_tile, bits, group, wht, op, y):
    return _empty(tuple(shape), _BF, codes)


@torch.library.custom_op("actcomp::gemm", mutates_args=())
def gemm(a: torch.Tensor, b: torch.Tensor, out_dtype: torch.dtype, activation: str) -> torch.Tensor:
    return core.gemm(a, b, out_dtype, activation)


@torch.library.custom_op("actcomp::gemm_two", mutates_args=())
def gemm_two(a: torch.Tensor, b: torch.Tensor, a2: torch.Tensor, b2: torch.Tensor, out_dtype: torch.dtype) -> torch.Tensor:
    """a @ b + a2 @ b2 (2-D) in one float32 accumulator."""
    return core.gemm(a, b, out_dtype, "", a2, b2)


@gemm_two.register_fake
def _(a, b, a2, b2, out_dtype):
    return a.new_empty((a.shape[0], b.shape[1]), dtype=out_dtype)


@gemm.register_fake
def _(a, b, out_dtype, activation):
    if a.dim() == 3 or b.dim() == 3:
        batch = max(a.shape[0] if a.dim() == 3 else 1, b.shape[0] if b.dim() == 3 else 1)
        return a.new_empty((batch, a.shape[-2], b.shape[-1]), dtype=out_dtype)
    return a.new_empty((a.shape[0], b.shape[1]), dtype=out_dtype)


# ---------------------------------------------------------------- residual branch
@torch.library.custom_op("actcomp::dropout", mutates_args=())
def dropout(x: torch.Tensor, p: float, seed: torch.Tensor, row_offset: int) -> torch.Tensor:
    """norm.dropout with the seed as a one-element int64 tensor (its backward is itself, on the gradient)."""
    return norm.dropout(x, p, seed, row_offset)


@dropout.register_fake
def _(x, p, seed, row_offset):
    return _empty(x.shape, x.dtype, x)


@torch.library.custom_op("actcomp::layer_norm", mutates_args=())
def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor],
               eps: float) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return norm.layer_norm(x, weight, bias, eps)


@layer_norm.register_fake
def _(x, weight, bias, eps):
    return _empty(x.shape, x.dtype, x), _empty(x.shape[:-1], _F32, x), _empty(x.shape[:-1], _F32, x)


def _weight_grads(x, weight, bias_dtype):
    """Fake dweight and dbias; dweight is empty without a weight (a custom op returns no None)."""
    dt = weight.dtype if weight is not None else bias_dtype or x.dtype
    return _empty(x.shape[-1:] if weight is not None else (0,), dt, x), _empty(x.shape[-1:], dt, x)


@torch.library.custom_op("actcomp::layer_norm_backward", mutates_args=())
def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, weight: Optional[torch.Tensor], mean: torch.Tensor,
                        rstd: torch.Tensor, bias_dtype: Optional[torch.dtype] = None) -> tuple[torch.Tensor,
                                                                                               torch.Tensor,
                                                                                               torch.Tensor]:
    """norm.layer_norm_backward; without a weight its gradient is an empty tensor."""
    dx, dw, db = norm.layer_norm_backward(dy, x, weight, mean, rstd, True, bias_dtype)
    return dx, db.new_empty(0) if dw is None else dw, db


@layer_norm_backward.register_fake
def _(dy, x, weight, mean, rstd, bias_dtype=None):
    return (_empty(x.shape, x.dtype, x),) + _weight_grads(x, weight, bias_dtype)


@torch.library.custom_op("actcomp::dropout_add_layer_norm", mutates_args=())
def dropout_add_layer_norm(x: torch.Tensor, residual: torch.Tensor, weight: Optional[torch.Tensor],
                           bias: Optional[torch.Tensor], p: float, seed: torch.Tensor, row_offset: int,
                           eps: float) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    return norm.dropout_add_layer_norm(x, residual, weight, bias, p, seed, row_offset, eps)


@dropout_add_layer_norm.register_fake
def _(x, residual, weight, bias, p, seed, row_offset, eps):
    return (_empty(x.shape, x.dtype, x), _empty(x.shape, x.dtype, x), _empty(x.shape[:-1], _F32, x),
            _empty(x.shape[:-1], _F32, x))


@torch.library.custom_op("actcomp::dropout_add_layer_norm_backward", mutates_args=())
def dropout_add_layer_norm_backward(dy: torch.Tensor, h: torch.Tensor, weight: Optional[torch.Tensor],
                                    mean: torch.Tensor, rstd: torch.Tensor, p: float, seed: torch.Tensor,
                                    row_offset: int, dh: Optional[torch.Tensor],
                                    bias_dtype: Optional[torch.dtype] = None) -> tuple[torch.Tensor, torch.Tensor,
                                                                                       torch.Tensor, torch.Tensor]:
    """norm.dropout_add_layer_norm_backward; without a weight its gradient is an empty tensor."""
    dx, dr, dw, db = norm.dropout_add_layer_norm_backward(dy, h, weight, mean, rstd, p, seed, row_offset, dh, True,
                                                          bias_dtype)
    return dx, dr, db.new_empty(0) if dw is None else dw, db


@dropout_add_layer_norm_backward.register_fake
def _(dy, h, weight, mean, rstd, p, seed, row_offset, dh, bias_dtype=None):
    return (_empty(h.shape, h.dtype, h), _empty(h.shape, h.dtype, h)) + _weight_grads(h, weight, bias_dtype)


@torch.library.custom_op("actcomp::rms_norm", mutates_args=())
def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor], eps: float) -> tuple[torch.Tensor, torch.Tensor]:
    return norm.rms_norm(x, weight, eps)


@rms_norm.register_fake
def _(x, weight, eps):
    return _empty(x.shape, x.dtype, x), _empty(x.shape[:-1], _F32, x)


@torch.library.custom_op("actcomp::add_rms_norm", mutates_args=())
def add_rms_norm(x: torch.Tensor, residual: torch.Tensor, weight: Optional[torch.Tensor],
                 eps: float) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return norm.add_rms_norm(x, residual, weight, eps)


@add_rms_norm.register_fake
def _(x, residual, weight, eps):
    return _empty(x.shape, x.dtype, x), _empty(x.shape, x.dtype, x), _empty(x.shape[:-1], _F32, x)


@torch.library.custom_op("actcomp::rms_norm_backward", mutates_args=())
def rms_norm_backward(dy: torch.Tensor, x: torch.Tensor, weight: Optional[torch.Tensor], rstd: torch.Tensor,
                      dh: Optional[torch.Tensor]) -> tuple[torch.Tensor, torch.Tensor]:
    """norm.rms_norm_backward; without a weight its gradient is an empty tensor."""
    dx, dw = norm.rms_norm_backward(dy, x, weight, rstd, dh)
    return dx, dx.new_empty(0) if dw is None else dw


@rms_norm_backward.register_fake
def _(dy, x, weight, rstd, dh):
    dw = x.new_empty(0) if weight is None else _empty(weight.shape, weight.dtype, x)
    return _empty(x.shape, x.dtype, x), dw


# ---------------------------------------------------------------- microscaled 4-bit
def _mx4_shapes(rows, cols):
    return (rows, (cols + 31) // 32 * 16), ((rows + 127) // 128 * ((cols + 127) // 128) * 512,)


@torch.library.custom_op("actcomp::mx4_quantize", mutates_args=())
def mx4_quantize(x: torch.Tensor, transpose: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of mx4.quantize."""
    q = mx4.quantize(x, transpose)
    return q.codes, q.scales


@mx4_quantize.register_fake
def _(x, transpose):
    rows, cols = x.numel() // x.shape[-1], x.shape[-1]
    c, s = _mx4_shapes(cols, rows) if transpose else _mx4_shapes(rows, cols)
    return _empty(c, _U8, x), _empty(s, _U8, x)


@torch.library.custom_op("actcomp::mx4_linear", mutates_args=())
def mx4_linear(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, out_dtype: torch.dtype) -> torch.Tensor:
    """mx4.linear with the weight's buffers (codes: (N, K / 2 rounded up to blocks))."""
    return mx4.linear(x, mx4.Mx4(codes.shape[0], x.shape[-1], codes, scales, x.dtype), out_dtype)


@mx4_linear.register_fake
def _(x, codes, scales, out_dtype):
    return _empty(x.shape[:-1] + (codes.shape[0],), out_dtype, x)


# ---------------------------------------------------------------- 8-bit floating point
def _fp8_shapes(rows, cols, tiles):
    blocks = (rows + 127) // 128 * ((cols + 127) // 128)
    return (rows, (cols + 15) // 16 * 16), (blocks if tiles else blocks * 128,)


@torch.library.custom_op("actcomp::fp8_quantize", mutates_args=())
def fp8_quantize(x: torch.Tensor, transpose: bool, tiles: bool, format: str) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of fp8.quantize, or with tiles of fp8.quantize_weight."""
    q = fp8.quantize_weight(x, format) if tiles else fp8.quantize(x, transpose, format)
    return q.codes, q.scales


@fp8_quantize.register_fake
def _(x, transpose, tiles, format):
    c, s = _fp8_shapes(x.numel() // x.shape[-1], x.shape[-1], tiles)
    return _empty(c, _U8, x), _empty(s, _U8, x)


@torch.library.custom_op("actcomp::fp8_linear", mutates_args=())
def fp8_linear(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, format: str,
               out_dtype: torch.dtype) -> torch.Tensor:
    """fp8.linear with the buffers of a weight by tiles (codes: (N, K rounded up to 16))."""
    w = fp8.Fp8(codes.shape[0], x.shape[-1], codes, scales, x.dtype, format, tiles=True)
    return fp8.linear(x, w, out_dtype)


@fp8_linear.register_fake
def _(x, codes, scales, format, out_dtype):
    return _empty(x.shape[:-1] + (codes.shape[0],), out_dtype, x)


# ---------------------------------------------------------------- cross entropy of a linear layer
@torch.library.custom_op("actcomp::linear_cross_entropy", mutates_args=())
def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor,
                         ignore_index: int) -> tuple[torch.Tensor, torch.Tensor]:
    return loss.linear_cross_entropy(x, weight, target, ignore_index)


@linear_cross_entropy.register_fake
def _(x, weight, target, ignore_index):
    return _empty(target.shape, _F32, x), _empty(target.shape, _F32, x)


@torch.library.custom_op("actcomp::linear_cross_entropy_backward", mutates_args=())
def linear_cross_entropy_backward(dloss: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor,
                                  lse: torch.Tensor, dlse: Optional[torch.Tensor], ignore_index: int,
                                  vocab_piece: int) -> tuple[torch.Tensor, torch.Tensor]:
    return loss.linear_cross_entropy_backward(dloss, x, weight, target, lse, dlse, ignore_index,
                                              vocab_piece=vocab_piece)


@linear_cross_entropy_backward.register_fake
def _(dloss, x, weight, target, lse, dlse, ignore_index, vocab_piece):
    return _empty(x.shape, x.dtype, x), _empty(weight.shape, weight.dtype, x)
