"""The 4-bit product through the C entry point into rows that are longer than the
result: what lies behind the result's columns and rows keeps what it held, also where
the columns end inside 16 bytes."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n,ld,code,dtype", [(70, 90, 128, 1, torch.bfloat16), (5, 33, 40, 2, torch.float16),
                                               (300, 257, 264, 1, torch.bfloat16), (9, 30, 32, 0, torch.float32),
                                               (6, 64, 72, 1, torch.bfloat16)])
def test_columns_behind_the_result(m, n, ld, code, dtype):
    from actcomp import _lib, mx4

    lib, g = _lib.load(), torch.Generator(device="cuda").manual_seed(1)
    a, b = (mx4.quantize(torch.randn(r, 200, generator=g, device="cuda")) for r in (m, n))
    out = torch.full((m + 2, ld), 7.0, dtype=dtype, device="cuda")
    da, db = (_lib.Mx4Desc(q.rows, q.cols, q.codes.data_ptr(), q.scales.data_ptr()) for q in (a, b))
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.actcomp_mx4_gemm(ctypes.byref(da), ctypes.byref(db), out.data_ptr(), ld, code, stream) == _lib.ACT_OK
    torch.cuda.synchronize()
    assert (out[m:] == 7).all() and (out[:, n:] == 7).all()
    assert torch.equal(out[:m, :n], mx4.matmul(a, b, dtype))
