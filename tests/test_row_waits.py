"""A wait of the layer norm kernels that gives up: the results are NaN, never made
of what a slot held before, and the device error word says so.  The copies are
simply not issued; nothing faults or hangs."""
import ctypes

import pytest
import torch


def test_validation_without_gpu():
    from actcomp import _lib

    f = _lib.load().actcomp_selftest_row_waits
    P = 1 << 20  # aligned, never dereferenced
    for bad in ((None, 4, 4, 64, P), (P, 4, 4, 64, None), (P, 0, 0, 64, P), (P, 1025, 4, 64, P), (P, 4, 5, 64, P),
                (P, 4, -1, 64, P), (P, 4, 4, 0, P), (P, 4, 4, (1 << 24) + 1, P)):
        assert f(*bad, None) == _lib.ACT_E_INVALID, bad
    assert f(P + 4, 4, 4, 64, P, None) == _lib.ACT_E_ALIGN


@pytest.mark.gpu
@pytest.mark.parametrize("rows,brought", [(1, 1), (9, 9), (1, 0), (9, 0), (9, 1), (9, 2), (9, 4), (9, 5), (8, 7)])
def test_rows_that_never_come_are_nan(rows, brought):
    from actcomp import _lib

    lib, word = _lib.load(), ctypes.c_uint32(0)
    s = torch.cuda.current_stream().cuda_stream
    assert lib.actcomp_clear_device_error(s) == _lib.ACT_OK
    x = torch.randint(-8, 9, (rows, 128), generator=torch.Generator().manual_seed(rows)).float().cuda()
    out = torch.full((rows,), -1.0, device="cuda")
    assert lib.actcomp_selftest_row_waits(x.data_ptr(), rows, brought, 4096, out.data_ptr(), s) == _lib.ACT_OK
    st = lib.actcomp_last_device_error(s, ctypes.byref(word))
    assert st == (_lib.ACT_OK if brought == rows else _lib.ACT_E_TIMEOUT)
    if brought == rows:
        assert torch.equal(out, x.sum(1))  # small whole numbers: exact
    else:
        assert out.isnan().all()
    assert lib.actcomp_clear_device_error(s) == _lib.ACT_OK
    assert lib.actcomp_last_device_error(s, ctypes.byref(word)) == _lib.ACT_OK
