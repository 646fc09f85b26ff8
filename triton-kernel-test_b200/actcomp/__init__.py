"""actcomp -- B200-native (sm_100a) activation compression.

Compute runs only in libactcomp.so (hand-written CUDA for sm_100a, C ABI in
include/actcomp.h); this package allocates tensors, builds descriptors and
launches through ctypes on the current CUDA stream.

Main entry points:
  Basis, Compressed, encode, decode, mul, silu_backward, gelu_backward,
  softmax_backward, weight_grad, select_outlier_channels   (channel-group format)
  refcompat.encode / refcompat.decode                       (the reference's format)
  reference_api.*                                           (the reference's function names)
  offload.Offloader                                         (pinned-host offload on a side stream)
  nf4.dequantize_4bit                                       (NF4 base weight -> bf16)
  dropout, layer_norm, dropout_add_layer_norm, *_backward   (residual branch: no stored mask)
  rms_norm, add_rms_norm, rms_norm_backward                 (root-mean-square norm)
  mx4.quantize / matmul / linear / linear_backward          (microscaled 4-bit floating point)
  fp8.quantize / matmul / linear / linear_backward, norms   (8-bit floating point, a scale per 128)
  linear_cross_entropy, linear_cross_entropy_backward       (loss over a vocabulary: no stored logits)
  dist.shard_rows / dist.reduce_error_stats                 (token sharding, error-stat all-reduce)
"""
from . import _lib
from .core import (Basis, Compressed, copy_into, decode, encode, error_stats, gelu_backward, gemm, mul,
                   select_outlier_channels, silu_backward, softmax_backward, weight_grad)

from . import dist, fp8, loss, mx4, nf4, offload
from .loss import linear_cross_entropy, linear_cross_entropy_backward
from .norm import (add_rms_norm, dropout, dropout_add_layer_norm, dropout_add_layer_norm_backward, dropout_backward,
                   layer_norm, layer_norm_backward, rms_norm, rms_norm_backward)
from .offload import HostActivation, Offloader

_lib.load()  # fail loudly at import if the CUDA library is missing

__all__ = ["Basis", "Compressed", "encode", "decode", "mul", "silu_backward", "gelu_backward", "softmax_backward",
           "weight_grad", "select_outlier_channels", "gemm", "error_stats", "copy_into", "Offloader",
           "HostActivation", "dist", "mx4", "nf4", "offload", "dropout", "dropout_backward", "layer_norm",
           "layer_norm_backward", "dropout_add_layer_norm", "dropout_add_layer_norm_backward", "rms_norm", "add_rms_norm",
           "rms_norm_backward", "fp8", "loss", "linear_cross_entropy", "linear_cross_entropy_backward"]
