"""Softmax cross entropy of a linear layer over a large vocabulary, whose logits are
never in memory.

The logits of a training step are its largest activation (tokens x vocabulary); where
the rest of the package compresses what is saved, this saves four bytes a token:

  loss, lse = linear_cross_entropy(x, weight, target)        # x (..., H), weight (V, H)
  dx, dw    = linear_cross_entropy_backward(dloss, x, weight, target, lse)

with z = x . weight^T, lse = log sum_v exp z_v and loss = lse - z[target], all float32 per
token (the caller reduces; dloss, the gradient of each loss, carries its weights).  Both
results have a gradient: dlse, where lse is used too (a penalty on the normaliser).
Targets equal to ``ignore_index`` have loss 0 and no gradient through it; other targets
outside the vocabulary give NaN.

The products run on bf16 or fp16 operands with float32 accumulation.  The backward pass
computes the logits again, a piece of the vocabulary at a time, and keeps the piece's
gradient in x's dtype, scaled so that fp16 holds it (workspace: by default 1 GiB, or
4096 columns where those are more; ``vocab_piece`` chooses); a copy of x and, with
several pieces, dx in float32 come on top.  Tokens without a gradient add nothing,
whatever their rows of x hold.

Waits inside the products are bounded.  One that gives up leaves NaN in the losses it
had, or parts of the gradients unwritten, and is recorded in the device error word, which
``_lib.load().actcomp_last_device_error`` reads (ACT_E_TIMEOUT).  All functions
compute outside autograd: results carry no graph, whatever the inputs require.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib

_host = _lib.host


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor,
                         ignore_index: int = -100) -> tuple[torch.Tensor, torch.Tensor]:
    """(loss, lse), float32 in target's shape, for x (..., H) and weight (V, H) of one
    dtype (bfloat16 or float16) and int64 targets (...)."""
    return _host.xent(x, weight, target, ignore_index)


def linear_cross_entropy_backward(dloss: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor,
                                  lse: torch.Tensor, dlse: Optional[torch.Tensor] = None, ignore_index: int = -100,
                                  x_grad: bool = True, weight_grad: bool = True,
                                  vocab_piece: int = 0) -> tuple[Optional[torch.Tensor], Optional[torch.Tensor]]:
    """(dx, dweight) in x's dtype from the float32 gradients of loss and lse (one value
    a token); what is not asked for is None.  ``vocab_piece``: columns of the vocabulary
    at a time, in whole tiles of 256 (0: see above)."""
    return _host.xent_backward(dloss, x, weight, target, lse, dlse, ignore_index, x_grad, weight_grad, vocab_piece)
