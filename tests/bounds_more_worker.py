"""Child process of tests/test_bounds_more.py: the root-mean-square norm, the 8-bit
operators and the cross entropy on ragged shapes through the library named by
ACTCOMP_LIBRARY; saves every output and the device error word to the .npz path given
as argv[1]."""
import ctypes
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "triton-kernel-test_b200"))


def main(out_path):
    import actcomp
    from actcomp import _lib, fp8

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
            x, dy, w = rand(r, c, dt), rand(r, c, dt), rand(1, c, dt)[0]
            name = f"{dt} {r}x{c}"
            y, rstd = actcomp.rms_norm(x, w)
            keep("forward " + name, y, rstd, *actcomp.add_rms_norm(x, dy, w))
            q, h, rs = fp8.add_rms_norm(x, dy, w)
            keep("8-bit norm " + name, fp8.dequantize(q), h, rs, fp8.dequantize(fp8.rms_norm(x, w)[0], torch.float32))
            keep("backward " + name, *actcomp.rms_norm_backward(dy, x, w, rstd),
                 *actcomp.rms_norm_backward(dy, x, w, rstd, dh=y))
            for f in fp8.FORMATS:
                for q in (fp8.quantize(x, format=f), fp8.quantize(x, True, f), fp8.quantize_weight(x, f),
                          *fp8.quantize_pair(x, f)):
                    keep(f"fp8 {name} {len(res)}", fp8.dequantize(q), fp8.dequantize(q, torch.float32))
        for m, n, k in ((1, 1, 1), (3, 300, 97), (16, 129, 2080), (100, 33, 64), (130, 257, 289), (700, 1001, 160)):
            x, wq, dy = rand(m, k, dt), fp8.quantize_weight(rand(n, k, torch.bfloat16)), rand(m, n, dt)
            y, saved = fp8.linear_forward(x, wq)
            keep(f"linear {dt} {m}x{n}x{k}", y, fp8.linear(x, wq, torch.float32), *fp8.linear_backward(dy, saved, wq))
    for dt in (torch.bfloat16, torch.float16):
        for t, h, v, piece in ((1, 1, 1, 0), (5, 33, 300, 256), (130, 100, 1001, 512), (300, 257, 5000, 0),
                               (40, 64, 9001, 2048)):
            x, w = rand(t, h, dt), rand(v, h, dt)
            target = torch.randint(0, v, (t,), generator=g, device="cuda")
            target[::3] = -100
            loss, lse = actcomp.linear_cross_entropy(x, w, target)
            keep(f"xent {dt} {t}x{h}x{v}", loss, lse, *actcomp.linear_cross_entropy_backward(
                lse, x, w, target, lse, dlse=loss, vocab_piece=piece))
    word = ctypes.c_uint32(0)
    res["status"] = np.array([lib.actcomp_last_device_error(s, ctypes.byref(word))])
    res["word"] = np.array([word.value])
    np.savez(out_path, **res)


if __name__ == "__main__":
    main(sys.argv[1])
