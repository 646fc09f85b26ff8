"""Child process of tests/test_first_calls.py: every call here is the first of
its kernel in this process, so that no larger call before it has raised the
kernel's shared-memory limit.  argv[1] names the group; prints one line per
failed call."""
import os
import sys

import torch

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, os.path.join(os.path.dirname(HERE), "triton-kernel-test_b200"))
sys.path.insert(0, HERE)


def linear():
    """K at both ends and in the middle of the range where x and the staging
    buffers together are just under 48 KB, for one to four tokens."""
    from actcomp import mx4
    from test_mx4 import U, data, values

    for tokens, ks in ((1, (7169, 7200, 7264)), (2, (3521, 3584, 3616)), (3, (2305, 2368, 2400)),
                       (4, (1697, 1760, 1792))):
        for dtype, out, k in zip((torch.bfloat16, torch.float16, torch.float32),
                                 (torch.bfloat16, torch.float32, torch.float32), ks):
            n = 136
            w = mx4.quantize(data(n, k, torch.bfloat16, n).cuda())
            x = data(tokens, k, dtype, k)
            q, v = values(mx4.quantize(x.cuda())).cuda(), values(w).cuda()
            ref, mag = q @ v.t(), q.abs() @ v.abs().t()
            for xs in (torch.nn.functional.pad(x, (0, -k % 8)).cuda()[:, :k],  # 16-byte rows and others
                       torch.nn.functional.pad(x, (1, 8)).cuda()[:, 1:1 + k]):
                def call():
                    got = mx4.linear(xs, w, out).double()
                    assert ((got - ref).abs() <= U[out] * ref.abs() + k * 2.0 ** -23 * mag * (1 + U[out]) + 1e-7).all()
                yield f"linear {tokens} x {k} {dtype}", call


def norm():
    """Row lengths whose ring is just under 48 KB."""
    import test_norm_ops as T

    for dtype in T.DTYPES:
        for cols in ((3050,) if dtype == torch.float32 else (6104, 6100)):
            yield f"forward {cols} {dtype}", lambda: T.test_layer_norm_forward(dtype, 3, cols)
        if dtype == torch.float32:
            continue
        for cols in (3048, 3045):
            yield f"branch forward {cols} {dtype}", lambda: T.test_branch_forward(dtype, 3, cols)
            yield f"backward {cols} {dtype}", lambda: T.check_backward(dtype, 5, cols, wide=False, fused=False)


def main(group):
    failed = 0
    for name, call in {"linear": linear, "norm": norm}[group]():
        try:
            call()
        except Exception as e:
            failed += 1
            print(f"{name}: {type(e).__name__}: {e}", flush=True)
    torch.cuda.synchronize()
    return failed


if __name__ == "__main__":
    sys.exit(1 if main(sys.argv[1]) else 0)
