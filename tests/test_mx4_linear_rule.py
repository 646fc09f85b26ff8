"""Which form a linear layer on few tokens takes, and that both agree."""
import pytest
import torch


def test_rule():
    from actcomp import _lib

    one = _lib.host.one_kernel
    assert all(one(1, n, k) for n, k in ((1, 1), (16384, 16384), (40000, 20000)))
    assert one(4, 4096, 4096) and one(2, 8192, 8192) and not one(3, 8192, 8192)
    assert not one(4, 11008, 4096) and not one(2, 16384, 16384) and not one(5, 1, 1)
    assert not one(4, 8, 1 << 20) and not one(1, 8, 1 << 20)  # x outgrows shared memory
    assert not one(2, (1 << 31) - 256, 1 << 14)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 2, 3, 4, 5])
def test_both_forms_on_a_large_weight(tokens):
    """Each result within K 2^-23 sum|terms| of the exact product, rounded once."""
    from actcomp import mx4
    from test_mx4 import U, data, values

    n, k = 9001, 8200
    w, x = mx4.quantize(data(n, k, torch.bfloat16, 1).cuda()), data(tokens, k, torch.bfloat16, 2).cuda()
    a, b = values(mx4.quantize(x)).cuda(), mx4.dequantize(w, torch.float32).double()
    ref, mag = a @ b.t(), a.abs() @ b.abs().t()
    y, saved = mx4.linear_forward(x, w)
    assert torch.equal(y, mx4.linear(x, w))
    for got in (y, mx4.matmul(mx4.quantize(x), w)):
        u = U[torch.bfloat16]
        assert ((got.double() - ref).abs() <= u * ref.abs() + k * 2.0 ** -23 * mag * (1 + u)).all()
    assert torch.equal(saved.codes, mx4.quantize(x, transpose=True).codes)
