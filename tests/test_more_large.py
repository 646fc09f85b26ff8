"""Sizes at which the CTA pairs of the 8-bit product and of the cross entropy's products
take several tiles each (both accumulators, their shared columns, scale sets and ring
stages used again), with contractions from one stage to many, and at which the few-row
product's contraction is cut over a cluster.  Tolerances as in test_fp8 and test_xent."""
import pytest
import torch

from test_fp8 import U, data, values
from test_xent import check_backward, check_forward, make

pytestmark = pytest.mark.gpu


def close(got, va, vb, k, dtype):
    ref, mag = va @ vb.t(), va.abs() @ vb.abs().t()
    ref = torch.where(ref.to(dtype).isinf(), ref.to(dtype).double(), ref)
    bad = (got.double() != ref) & ~((got.double() - ref).abs() <= U[dtype] * ref.abs() + k * 2.0 ** -23 * mag * (1 + U[dtype]) + 1e-7)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist())


@pytest.mark.parametrize("m,n,k,dtype", [(5000, 5000, 100, torch.bfloat16), (4100, 5100, 1160, torch.float32),
                                         (2817, 7000, 896, torch.float16), (300, 40000, 640, torch.bfloat16)])
def test_product_over_several_turns(m, n, k, dtype):
    from actcomp import fp8

    x, y = data(m, k, torch.bfloat16, 1).cuda(), data(n, k, torch.bfloat16, 2).cuda()
    xt, yt = x.t().contiguous(), y.t().contiguous()
    for a, b in ((fp8.quantize(x), fp8.quantize_weight(y)), (fp8.quantize(xt, transpose=True), fp8.quantize(yt, transpose=True)),
                 (fp8.quantize(x), fp8.quantize_weight(yt).t())):
        close(fp8.matmul(a, b, dtype), values(a).cuda(), values(b).cuda(), k, dtype)


@pytest.mark.parametrize("m", [1, 16, 17, 48, 49, 97, 128])
@pytest.mark.parametrize("n,k", [(11008, 4096), (4096, 11008), (1000, 128), (129, 4100), (20000, 384), (128, 16384)])
def test_few_rows(m, n, k):
    from actcomp import fp8

    x, y = data(m, k, torch.bfloat16, m).cuda(), data(n, k, torch.bfloat16, 2).cuda()
    a, w, wt = fp8.quantize(x), fp8.quantize_weight(y), fp8.quantize_weight(y.t().contiguous()).t()
    va, vw = values(a).cuda(), values(w).cuda()
    close(fp8.matmul(a, w), va, vw, k, torch.bfloat16)
    close(fp8.matmul(a, wt, torch.float32), va, values(wt).cuda(), k, torch.float32)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,channels,vocab,piece", [(3000, 72, 20000, 0), (1500, 520, 9001, 4096), (300, 1160, 30001, 0),
                                                         (5000, 2056, 3000, 1024)])
def test_cross_entropy_over_several_turns(dtype, tokens, channels, vocab, piece):
    import actcomp

    x, w, t = make(tokens, channels, vocab, dtype, 3)
    loss, lse = actcomp.linear_cross_entropy(x.cuda(), w.cuda(), t.cuda())
    check_forward(x, w, t, loss, lse)
    d = (torch.rand(tokens, generator=torch.Generator().manual_seed(1)) / tokens).cuda()
    dx, dw = actcomp.linear_cross_entropy_backward(d, x.cuda(), w.cuda(), t.cuda(), lse, dlse=d * 0.1, vocab_piece=piece)
    check_backward(x, w, t, d, d * 0.1, lse, dx, dw)
