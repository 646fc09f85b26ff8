"""One training step of a feed-forward block and the loss at a model's end, with little
saved state.

    z, h = add_rms_norm(x, residual)        4 bytes a row saved, and h
    u = z W1^T, v = silu(u) W2^T            8-bit floating point, inputs saved in 8 bits
    t, g = add_rms_norm(v, h)
    loss = mean cross entropy of t W^T      logits not kept: 4 bytes a token

and its backward pass, then the same step by autograd in float32 torch.

    python triton-kernel-test_b200/examples/language_step.py
"""
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))

import actcomp  # noqa: E402
from actcomp import fp8  # noqa: E402
from actcomp.reference_api import triton_silu_backward  # noqa: E402

NAMES = ("x", "residual", "norm1", "w1", "w2", "norm2", "head")


def step(x, residual, norm1, w1, w2, norm2, head, target):
    """(loss, gradients in NAMES' order)."""
    q1, q2 = fp8.quantize_weight(w1), fp8.quantize_weight(w2)
    z, h, rstd1 = actcomp.add_rms_norm(x, residual, norm1)
    u, saved1 = fp8.linear_forward(z, q1)
    v, saved2 = fp8.linear_forward(torch.nn.functional.silu(u), q2)
    t, g, rstd2 = actcomp.add_rms_norm(v, h, norm2)
    loss, lse = actcomp.linear_cross_entropy(t, head, target)
    live = (target != -100).sum()
    dloss = torch.ones_like(loss) / live
    # backward; h is used twice, g once
    dt, dhead = actcomp.linear_cross_entropy_backward(dloss, t, head, target, lse)
    dg, dnorm2 = actcomp.rms_norm_backward(dt, g, norm2, rstd2)
    da, dw2 = fp8.linear_backward(dg, saved2, q2)
    du = triton_silu_backward(u[None], da[None])[0]
    dz, dw1 = fp8.linear_backward(du, saved1, q1)
    dh, dnorm1 = actcomp.rms_norm_backward(dz, h, norm1, rstd1, dh=dg)
    return loss.sum() / live, (dh, dh, dnorm1, dw1, dw2, dnorm2, dhead)


def serve(x, residual, norm1, q1):
    """The first projection of single tokens being served: the norm gives it its input in 8 bits."""
    q, h, _ = fp8.add_rms_norm(x, residual, norm1)
    return fp8.matmul(q, q1), h


def plain_step(x, residual, norm1, w1, w2, norm2, head, target):
    """The same step by autograd in float32."""
    p = [v.detach().float().requires_grad_() for v in (x, residual, norm1, w1, w2, norm2, head)]
    rms = lambda v, w: v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-5) * w  # noqa: E731
    h = p[0] + p[1]
    v = torch.nn.functional.silu(rms(h, p[2]) @ p[3].t()) @ p[4].t()
    loss = torch.nn.functional.cross_entropy(rms(v + h, p[5]) @ p[6].t(), target)
    loss.backward()
    return loss.detach(), [v.grad for v in p]


def inputs(tokens=512, channels=512, hidden=1408, vocab=5003, device="cuda"):
    g = torch.Generator(device=device).manual_seed(0)
    rand = lambda *s: torch.randn(*s, generator=g, device=device)  # noqa: E731
    target = torch.randint(0, vocab, (tokens,), generator=g, device=device)
    target[::7] = -100
    t = [rand(tokens, channels), rand(tokens, channels), 1 + 0.1 * rand(channels), rand(hidden, channels) / channels ** 0.5,
         rand(channels, hidden) / hidden ** 0.5, 1 + 0.1 * rand(channels), rand(vocab, channels) / channels ** 0.5]
    return [v.to(torch.bfloat16) for v in t] + [target]


def main():
    args = inputs()
    loss, grads = step(*args)
    ref, ref_grads = plain_step(*args)
    err = lambda a, b: float((a.float() - b).norm() / b.norm())  # noqa: E731
    return {"loss": err(loss, ref), **{"d" + n: err(a, b) for n, a, b in zip(NAMES, grads, ref_grads)}}


if __name__ == "__main__":
    print({k: round(v, 5) for k, v in main().items()})
