"""Child process of tests/test_bounds_ops.py: the dropout, layer norm and 4-bit
operators on ragged shapes through the library named by ACTCOMP_LIBRARY; saves
every output and the device error word to the .npz path given as argv[1]."""
import ctypes
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "triton-kernel-test_b200"))


def main(out_path):
    import actcomp
    from actcomp import _lib, mx4

    lib = _lib.load()
    s = torch.cuda.current_stream().cuda_stream
    assert lib.actcomp_clear_device_error(s) == _lib.ACT_OK
    res = {}

    def keep(name, *tensors):
        for i, t in enumerate(tensors):
            if t is not None:
                res[f"{name}.{i}"] = t.contiguous().view(torch.uint8).cpu().numpy()

    g = torch.Generator(device="cuda").manual_seed(5)
    rand = lambda r, c, dt: torch.randn(r, c, generator=g, device="cuda").to(dt)  # noqa: E731
    for dt in (torch.bfloat16, torch.float16, torch.float32):
        for r, c in ((1, 1), (5, 7), (300, 33), (70, 515), (9, 1000), (40, 4097), (17, 5120), (9, 9216), (3, 16384),
                     (3, 20001)):
            x, dy = rand(r, c, dt), rand(r, c, dt)
            w, b = rand(1, c, dt)[0], rand(1, c, dt)[0]
            name = f"{dt} {r}x{c}"
            keep("dropout " + name, actcomp.dropout(x, 0.2, 7, 3))
            y, mean, rstd = actcomp.layer_norm(x, w, b)
            keep("forward " + name, y, mean, rstd, *actcomp.dropout_add_layer_norm(x, dy, w, b, 0.2, 7))
            keep("backward " + name, *actcomp.layer_norm_backward(dy, x, w, mean, rstd),
                 *actcomp.dropout_add_layer_norm_backward(dy, x, w, mean, rstd, 0.2, 7, dh=x))
            for q in (mx4.quantize(x), mx4.quantize(x, transpose=True), *mx4.quantize_pair(x)):
                keep(f"mx4 {name} {len(res)}", q.codes, q.scales, mx4.dequantize(q), mx4.dequantize(q, torch.float32))
        for m, n, k in ((1, 1, 1), (3, 300, 97), (4, 129, 2080), (5, 33, 64), (130, 257, 289), (700, 1001, 160)):
            x, wq = rand(m, k, dt), mx4.quantize(rand(n, k, torch.bfloat16))
            keep(f"linear {dt} {m}x{n}x{k}", mx4.linear(x, wq), mx4.linear(x, wq, torch.float32))
    word = ctypes.c_uint32(0)
    res["status"] = np.array([lib.actcomp_last_device_error(s, ctypes.byref(word))])
    res["word"] = np.array([word.value])
    np.savez(out_path, **res)


if __name__ == "__main__":
    main(sys.argv[1])
