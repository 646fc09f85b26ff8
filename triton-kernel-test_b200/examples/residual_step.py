"""One training step of a residual branch with little saved state.

    h = residual + dropout(f)          mask from a seed, nothing stored
    z = layer_norm(h)                  8 bytes a row stored
    y = z W^T                          both operands in 4-bit floating point
    loss = sum(y * target)

and its backward pass, then the same step in plain float32 torch.  Saved for the
backward pass: the seed, h (here compressed by actcomp.encode as well), two
float32 per row, and z by columns in 4 bits.

    python triton-kernel-test_b200/examples/residual_step.py
"""
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))

import actcomp  # noqa: E402
from actcomp import mx4  # noqa: E402


def step(f, residual, weight, bias, w, target, p, seed, compress=False):
    """(y, gradients of f, residual, weight, bias, w) and the bytes saved."""
    wq, wt = mx4.quantize_pair(w)  # a frozen weight's pair is kept from step to step
    z, h, mean, rstd = actcomp.dropout_add_layer_norm(f, residual, weight, bias, p, seed)
    y, saved = mx4.linear_forward(z, wq)
    kept = actcomp.encode(h, actcomp.Basis.fit(h, 16), None, bits=8, group=64) if compress else h
    del z, h
    nbytes = saved.nbytes() + 8 * mean.numel() + 8
    nbytes += kept.nbytes() if compress else kept.numel() * kept.element_size()
    # backward: target is the gradient of y
    dz, dw = mx4.linear_backward(target, saved, wt)
    h = actcomp.decode(kept) if compress else kept
    df, dres, dweight, dbias = actcomp.dropout_add_layer_norm_backward(dz, h, weight, mean, rstd, p, seed)
    return y, (df, dres, dweight, dbias, dw), nbytes


def plain_step(f, residual, weight, bias, w, target, keep, scale):
    """The same step by autograd in float32, with the mask given."""
    t = [v.detach().float().requires_grad_() for v in (f, residual, weight, bias, w)]
    h = t[1] + torch.where(keep, t[0] * scale, 0.0)
    z = torch.nn.functional.layer_norm(h, h.shape[-1:], t[2], t[3], 1e-5)
    y = z @ t[4].t()
    y.backward(target.float())
    return y.detach(), [v.grad for v in t]


def main(tokens=2048, channels=1024, out=1536, p=0.1, device="cuda"):
    g = torch.Generator(device=device).manual_seed(0)
    rand = lambda *s: torch.randn(*s, generator=g, device=device).to(torch.bfloat16)  # noqa: E731
    f, residual, target = rand(tokens, channels), rand(tokens, channels), rand(tokens, out) * 0.01
    weight, bias = 1 + 0.1 * rand(channels), 0.1 * rand(channels)
    w = rand(out, channels) / channels ** 0.5
    seed = 1234
    keep = actcomp.dropout(torch.ones_like(f), p, seed) != 0
    held = round(p * 65536) / 65536
    ref, ref_grads = plain_step(f, residual, weight, bias, w, target, keep, 1 / (1 - held))
    err = lambda a, b: float((a.float() - b).norm() / b.norm())  # noqa: E731
    report = {}
    for compress in (False, True):
        y, grads, nbytes = step(f, residual, weight, bias, w, target, p, seed, compress)
        report[compress] = {"bytes": nbytes, "y": err(y, ref)}
        for name, a, b in zip(("f", "residual", "weight", "bias", "w"), grads, ref_grads):
            report[compress]["d" + name] = err(a, b)
    return report


if __name__ == "__main__":
    for compress, r in main().items():
        print("h compressed" if compress else "h kept in bf16", {k: round(v, 4) for k, v in r.items()})
