"""Two host threads that call one kernel with different amounts of shared memory:
neither may have its launch refused because of the other's.  (Calls by ctypes,
which gives the interpreter lock away; each thread has its own stream.)"""
import ctypes
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu
CALLS = 20000


def run(*calls):
    bad, start = [], threading.Barrier(len(calls))

    def work(call):
        start.wait()
        for _ in range(CALLS):
            st = call()
            if st:
                bad.append(st)
                return

    threads = [threading.Thread(target=work, args=(c,)) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not bad, bad


def test_layer_norm_of_two_row_lengths():
    from actcomp import _lib

    lib, keep = _lib.load(), []

    def call(cols):
        x, y = torch.randn(2, cols, device="cuda").bfloat16(), torch.empty(2, cols, device="cuda", dtype=torch.bfloat16)
        st, s = torch.empty(2, 2, device="cuda"), torch.cuda.Stream()
        a = _lib.LnArgs(rows=2, cols=cols, x=x.data_ptr(), ldx=cols, y=y.data_ptr(), ldy=cols, mean=st[0].data_ptr(),
                        rstd=st[1].data_ptr(), dtype=1, wdtype=1, eps=1e-5)
        keep.append((x, y, st, s, a))
        return lambda: lib.actcomp_layer_norm(ctypes.byref(a), s.cuda_stream)

    calls = call(8192), call(6400)
    torch.cuda.synchronize()
    run(*calls)
    for x, y, *_ in keep:
        want = torch.nn.functional.layer_norm(x.double(), x.shape[1:])
        assert ((y.double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-4).all()


def test_linear_of_two_widths():
    from actcomp import _lib, mx4

    lib, keep = _lib.load(), []

    def call(k):
        x, w = torch.randn(1, k, device="cuda").bfloat16(), mx4.quantize(torch.randn(8, k, device="cuda"))
        out, s = torch.empty(1, 8, device="cuda", dtype=torch.bfloat16), torch.cuda.Stream()
        d = _lib.Mx4Desc(8, k, w.codes.data_ptr(), w.scales.data_ptr())
        keep.append((x, w, out, s, d))
        return lambda: lib.actcomp_mx4_linear(x.data_ptr(), 1, k, k, 1, ctypes.byref(d), out.data_ptr(), 8, 1,
                                              s.cuda_stream)

    calls = call(16384), call(8000)
    torch.cuda.synchronize()
    run(*calls)
    for x, w, out, *_ in keep:
        assert torch.equal(out, mx4.linear(x, w))
