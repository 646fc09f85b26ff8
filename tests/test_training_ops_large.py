"""Sizes at which a CTA of the dropout, 4-bit quantisation and 4-bit product
kernels takes several turns of its loop: more segments than the grid has warps,
more row groups than CTAs, several output tiles per CTA pair (both accumulators,
their shared columns and both column orders).

Tolerances as in test_mx4 (a product is within K 2^-23 sum|terms|, rounded once)
and exact elsewhere."""
import numpy as np
import pytest
import torch

from test_norm_ops import held_scale, keep_mask

pytestmark = pytest.mark.gpu
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def rounded(x):
    """The values that x (float64, blocks of 32 along its rows) has in the 4-bit format."""
    rows, cols = x.shape
    b = torch.nn.functional.pad(x, (0, -cols % 32)).reshape(rows, -1, 32)
    amax = b.abs().amax(-1, keepdim=True)
    e = torch.where(amax > 0, torch.frexp(amax).exponent - 3, -127).clamp_min(-127)  # floor(log2) - 2
    a = torch.ldexp(b.abs(), -e).clamp_max(6.0)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).double()
    q = torch.ldexp((a / step).round() * step, e)  # round: ties to even, as the mantissa's last bit
    return torch.copysign(q, b).reshape(rows, -1)[:, :cols]


def data(rows, cols, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, cols, generator=g, device="cuda")
    return (x * torch.exp2(torch.randint(-6, 7, (rows, 1), generator=g, device="cuda").float())).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(3000, 4096), (3001, 4001), (700001, 17), (30, 500003)])
def test_dropout_over_several_turns(dtype, rows, cols):
    import actcomp

    x = data(rows, cols, dtype, rows)
    keep = keep_mask(rows, cols, 0.3, 99, 12).cuda()
    y = actcomp.dropout(x, 0.3, 99, 12)
    want = torch.where(keep, x.double() * held_scale(0.3), 0.0)
    assert torch.equal(y != 0, keep & (want.to(dtype) != 0))
    # one product with a scale rounded to float32, one rounding; the smallest subnormal steps of fp16
    assert ((y.double() - want).abs() <= (U[dtype] + 2.0 ** -23) * want.abs() + 6e-8 * (dtype == torch.float16)).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(80003, 40), (20011, 1003), (20000, 1024)])
def test_quantise_over_several_turns(dtype, rows, cols):
    from actcomp import mx4

    x = data(rows, cols, dtype, cols)
    want = rounded(x.double())
    q = mx4.quantize(x)
    for out in DTYPES:
        assert torch.equal(mx4.dequantize(q, out), want.to(out)), out
    pair = mx4.quantize_pair(x)
    assert torch.equal(pair[0].codes, q.codes) and torch.equal(pair[0].scales, q.scales)
    want_t = rounded(x.double().t().contiguous()).float()
    assert torch.equal(mx4.dequantize(pair[1], torch.float32), want_t)
    assert torch.equal(mx4.dequantize(mx4.quantize(x, transpose=True), torch.float32), want_t)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", [(2048, 9216, 256), (2100, 9001, 289), (4600, 4100, 1024), (257, 40000, 96),
                                   (40000, 300, 1500)])
def test_products_of_several_tiles_per_pair(dtype, M, N, K):
    from actcomp import mx4

    a, b = mx4.quantize(data(M, K, torch.float32, M)), mx4.quantize(data(N, K, torch.float32, N))
    got = mx4.matmul(a, b, dtype)
    va, vb = mx4.dequantize(a, torch.float32).double(), mx4.dequantize(b, torch.float32).double()
    assert torch.equal(va, rounded(data(M, K, torch.float32, M).double()))
    ref, mag = va @ vb.t(), va.abs() @ vb.abs().t()
    slack = K * 2.0 ** -23 * mag * (1 + U[dtype]) + 1e-7 * (dtype == torch.float16)
    ok = (got.double() - ref).abs() <= U[dtype] * ref.abs() + slack
    if dtype == torch.float16:
        ok |= got.isinf() & (torch.sign(got) == torch.sign(ref)) & (ref.abs() + slack >= 65520)
    assert ok.all(), int((~ok).sum())


def test_step_of_several_tiles_per_pair():
    """Forward and both gradients at sizes that give every product more tiles than pairs."""
    from actcomp import mx4

    t, k, n = 4111, 2500, 4200
    x, w, dy = (data(*s, torch.bfloat16, i) for i, s in enumerate(((t, k), (n, k), (t, n))))
    wq, wt = mx4.quantize_pair(w)
    y, saved = mx4.linear_forward(x, wq)
    dx, dw = mx4.linear_backward(dy, saved, wt)
    r = lambda v: rounded(v.double())  # noqa: E731
    rt = lambda v: rounded(v.double().t().contiguous())  # noqa: E731
    for got, a, b in ((y, r(x), r(w)), (dx, r(dy), rt(w)), (dw, rt(dy), rt(x))):
        ref, mag = a @ b.t(), a.abs() @ b.abs().t()
        assert got.shape == ref.shape
        assert ((got.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + a.shape[1] * 2.0 ** -22 * mag).all()


def test_rounding_restatement():
    """The vectorised form above against the definition, value by value."""
    from test_mx4 import GRID, encode64

    x = torch.randn(6, 70, generator=torch.Generator().manual_seed(0)).double()
    x[0, :8] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0])
    codes, scale = encode64(x.numpy())
    v = np.where(codes & 8, -1.0, 1.0) * GRID[codes & 7] * np.repeat(2.0 ** (scale - 127.0), 32, 1)
    assert np.array_equal(rounded(x).numpy(), v[:, :70])
