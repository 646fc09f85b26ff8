"""Microscaled 4-bit floating point: the format against a plain restatement, bit
for bit; the products against float64 products of the values that the operands
stand for.

Tolerance of a product: the operands' products are exact in float32, a sum of K
terms in any order with each addition rounded or truncated is within K 2^-23
sum|terms|, and the result is rounded once to the output type."""
import ctypes

import numpy as np
import pytest
import torch

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


# ---------------------------------------------------------------- plain form
def encode64(v):
    """(codes 0..15, scale bytes) of a float64 matrix by the definition."""
    rows, cols = v.shape
    nb = -(-cols // 32)
    p = np.zeros((rows, nb * 32))
    p[:, :cols] = v
    p = p.reshape(rows, nb, 32)
    amax = np.abs(p).max(-1)
    scale = np.zeros((rows, nb), np.int64)
    codes = np.zeros(p.shape, np.int64)
    for r in range(rows):
        for b in range(nb):
            if not np.isfinite(amax[r, b]):
                scale[r, b] = 255
                continue
            e = -127 if amax[r, b] == 0 else max(int(np.floor(np.log2(amax[r, b]))) - 2, -127)
            scale[r, b] = e + 127
            for j, x in enumerate(p[r, b] / 2.0 ** e):
                d = np.abs(GRID - min(abs(x), 6.0))
                near = np.flatnonzero(d == d.min())
                k = near[0] if len(near) == 1 else near[near % 2 == 0][0]  # a tie: the even mantissa
                codes[r, b, j] = k + (8 if np.signbit(x) else 0)
    return codes.reshape(rows, -1), scale


def unpack(q):
    """(codes 0..15, scale bytes) as the buffers hold them, and the padding's scale bytes."""
    c = q.codes.cpu().numpy()
    codes = np.stack([c & 15, c >> 4], -1).reshape(q.rows, -1)
    nb, nka = -(-q.cols // 32), -(-q.cols // 128)
    s = q.scales.cpu().numpy()
    r, b = np.meshgrid(np.arange(-(-q.rows // 128) * 128), np.arange(nka * 4), indexing="ij")
    full = s[((r // 128) * nka + b // 4) * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + b % 4]
    pad = full.copy()
    pad[: q.rows, :nb] = 0
    return codes, full[: q.rows, :nb].astype(np.int64), pad


def values(q):
    codes, scale, _ = unpack(q)
    v = np.where(codes & 8, -1.0, 1.0) * GRID[codes & 7]
    s = np.where(scale == 255, np.nan, 2.0 ** (scale - 127.0))
    return torch.from_numpy((v * np.repeat(s, 32, 1))[:, : q.cols])


def data(rows, cols, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * torch.exp2(torch.randint(-6, 7, (rows, 1), generator=g).float())
    x[torch.rand(rows, cols, generator=g) < 0.1] = 0
    return x.to(dtype)


def check_codes(q, v):
    codes, scale, pad = unpack(q)
    want, ws = encode64(v.double().cpu().numpy())
    assert np.array_equal(scale, ws)
    fine = np.repeat(ws != 255, 32, 1)
    assert np.array_equal(codes[fine], want[fine])
    assert not pad.any()


# ---------------------------------------------------------------- CPU
def test_sizes_and_validation_without_gpu():
    from actcomp import _lib

    lib = _lib.load()
    assert lib.actcomp_mx4_code_bytes(3, 33) == 3 * 32 and lib.actcomp_mx4_scale_bytes(129, 129) == 4 * 512
    assert lib.actcomp_mx4_code_bytes(0, 5) == 0 and lib.actcomp_mx4_scale_bytes(5, -1) == 0
    P = 1 << 20
    d = lambda r=64, c=96, codes=P, scales=P: ctypes.byref(_lib.Mx4Desc(r, c, codes, scales))  # noqa: E731
    quant = lambda q, qt, x=P, ld=96, dt=1: lib.actcomp_mx4_quantize(x, 64, 96, ld, dt, q, qt, None)  # noqa: E731
    assert quant(None, None) == _lib.ACT_E_INVALID
    assert quant(d(), None, x=None) == _lib.ACT_E_INVALID and quant(d(), None, ld=95) == _lib.ACT_E_INVALID
    assert quant(d(96, 64), None) == _lib.ACT_E_INVALID and quant(None, d()) == _lib.ACT_E_INVALID
    assert quant(d(), None, dt=3) == _lib.ACT_E_INVALID
    assert quant(d(codes=P + 8), None) == _lib.ACT_E_ALIGN and quant(d(), None, x=P + 1) == _lib.ACT_E_ALIGN
    assert quant(d(scales=None), None) == _lib.ACT_E_INVALID
    gemm = lambda a, b, ld=64, dt=1, c=P: lib.actcomp_mx4_gemm(a, b, c, ld, dt, None)  # noqa: E731
    assert gemm(d(), d(64, 128)) == _lib.ACT_E_INVALID and gemm(d(), d(), ld=63) == _lib.ACT_E_INVALID
    assert gemm(d(), d(), dt=5) == _lib.ACT_E_INVALID and gemm(d(), d(), c=P + 1) == _lib.ACT_E_ALIGN
    assert gemm(d(), d(0, 96)) == _lib.ACT_E_INVALID
    lin = lambda t=1, k=96, ld=96, x=P, w=None, o=1: lib.actcomp_mx4_linear(  # noqa: E731
        x, t, k, ld, 1, w or d(), P, 64, o, None)
    assert lin(0) == _lib.ACT_E_INVALID and lin(k=64) == _lib.ACT_E_INVALID and lin(ld=8) == _lib.ACT_E_INVALID
    assert lin(o=2) == _lib.ACT_E_INVALID and lin(x=P + 1) == _lib.ACT_E_ALIGN
    assert lin(_lib.MX4_LINEAR_TOKENS + 1) == _lib.ACT_E_UNSUPPORTED
    assert lin(4, 1 << 20, 1 << 20, w=d(64, 1 << 20)) == _lib.ACT_E_UNSUPPORTED  # x outgrows shared memory
    assert lib.actcomp_mx4_dequantize(d(), P, 95, 1, None) == _lib.ACT_E_INVALID
    assert lib.actcomp_mx4_dequantize(d(1 << 31), P, 96, 1, None) == _lib.ACT_E_UNSUPPORTED


def test_cpu_tensors_are_refused():
    from actcomp import mx4

    with pytest.raises(ValueError):
        mx4.quantize(torch.zeros(4, 32))


# ---------------------------------------------------------------- quantisation
SHAPES = [(1, 1), (1, 31), (3, 32), (2, 33), (130, 40), (5, 256), (33, 257), (70, 300), (129, 129), (40, 1000)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quantise_both_ways(dtype, rows, cols):
    from actcomp import mx4

    x = data(rows, cols, dtype, rows + cols)
    q, qt = mx4.quantize(x.cuda()), mx4.quantize(x.cuda(), transpose=True)
    check_codes(q, x)
    check_codes(qt, x.t())
    for a, b in zip(mx4.quantize_pair(x.cuda()), (q, qt)):
        assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
    for t in (q, qt):
        for out in DTYPES:
            assert torch.equal(mx4.dequantize(t, out).double().cpu(), values(t).to(out).double())


@pytest.mark.gpu
def test_quantise_special_values():
    """Ties, saturation, signs, zero and subnormal blocks, the largest values, NaN and infinity."""
    from actcomp import mx4

    mids = (GRID[:-1] + GRID[1:]) / 2
    row = np.concatenate([mids, -mids, [6.5, 7.0, 7.9, -7.99, 4.0, 5.0, -5.0, 0.0, 0.25, -0.25, 3.5, -3.5, 1.25, 1.75,
                                        0.75, 2.5, 4.5, 5.5]]).astype(np.float32)
    v = np.zeros((16, 64), np.float32)
    for i, s in enumerate([1.0, 2.0 ** 60, 2.0 ** -100, 2.0 ** -125, 2.0 ** -126, 2.0 ** -130, 2.0 ** 125]):
        v[i, :32] = row * np.float32(s)
    v[7, 3] = np.float32(1e-45)                      # one subnormal value
    v[8, 0] = np.finfo(np.float32).max
    v[9, 5], v[10, 40], v[11, 33] = np.nan, np.inf, -np.inf
    x = torch.from_numpy(v)
    q = mx4.quantize(x.cuda())
    check_codes(q, x)
    y = mx4.dequantize(q).cpu()
    assert torch.equal(y.nan_to_num(0.0), values(q).float().nan_to_num(0.0))
    nan = torch.zeros(16, 64, dtype=torch.bool)
    nan[9, :32] = nan[10, 32:] = nan[11, 32:] = True
    assert torch.equal(y.isnan(), nan)
    qt = mx4.quantize(x.t().contiguous().cuda(), transpose=True)
    assert torch.equal(qt.codes, q.codes) and torch.equal(qt.scales, q.scales)
    for dt in (torch.bfloat16, torch.float16):
        z = torch.tensor([[1e-8, 6e-8, 0, 65504.0 if dt == torch.float16 else 3e38] * 8]).to(dt)
        check_codes(mx4.quantize(z.cuda()), z)
        z[0, 4] = float("nan")
        assert mx4.dequantize(mx4.quantize(z.cuda())).isnan().all()


@pytest.mark.gpu
def test_quantise_strides_and_streams():
    from actcomp import mx4

    wide = data(200, 640, torch.bfloat16, 3).cuda()
    for v in (wide[:, 64:320], wide[:, 3:200], wide[::3], wide.t(), wide[5:6, :77], wide.view(4, 50, 640)):
        want = v.reshape(-1, v.shape[-1]).contiguous()
        for t in (False, True):
            a, b = mx4.quantize(v, transpose=t), mx4.quantize(want, transpose=t)
            assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
    q = mx4.quantize(wide)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = mx4.linear(wide, q)
    side.synchronize()
    assert torch.equal(y, mx4.linear(wide, q))


# ---------------------------------------------------------------- products
def check_product(a, b, dt):
    from actcomp import mx4

    got = mx4.matmul(a, b, dt)
    va, vb = values(a).cuda(), values(b).cuda()
    ref, mag = va @ vb.t(), va.abs() @ vb.abs().t()
    assert got.shape == ref.shape and got.dtype == dt
    slack = a.cols * 2.0 ** -23 * mag * (1 + U[dt]) + 1e-7 * (dt == torch.float16)
    ok = (got.double() - ref).abs() <= U[dt] * ref.abs() + slack
    if dt == torch.float16:  # its range ends: values that round past 65504 are infinite
        past = got.isinf() & (torch.sign(got) == torch.sign(ref)) & (ref.abs() + slack >= 65520)
        ok = ok | past
    assert ok.all(), int((~ok).sum())


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 300, 64), (2, 33, 96), (16, 256, 128), (17, 129, 160), (64, 520, 256),
                                   (128, 256, 256), (129, 257, 289), (200, 128, 512), (257, 513, 1000), (31, 700, 4096),
                                   (300, 1, 288), (1, 4096, 2048), (8, 1000, 2080), (520, 384, 1312)])
def test_products(M, N, K):
    from actcomp import mx4

    a, b = mx4.quantize(data(M, K, torch.float32, M + K).cuda()), mx4.quantize(data(N, K, torch.float32, N).cuda())
    for dt in DTYPES:
        if dt != torch.float16 or K < 1000:
            check_product(a, b, dt)


@pytest.mark.gpu
def test_product_small_values_are_exact():
    """Small whole numbers: every partial sum is a whole number below 2^24, so the result is exact."""
    from actcomp import mx4

    g = torch.Generator().manual_seed(0)
    pick = torch.tensor([0.0, 1.0, 2.0, 3.0, 4.0, 6.0, -1.0, -2.0, -3.0, -6.0])
    a, b = (pick[torch.randint(0, 10, s, generator=g)].cuda() for s in ((300, 512), (700, 512)))
    a[:, ::32], b[:, ::32] = 4.0, 6.0
    got = mx4.matmul(mx4.quantize(a), mx4.quantize(b), torch.float32)
    assert torch.equal(got.double(), a.double() @ b.double().t())


@pytest.mark.gpu
def test_product_carries_nan_blocks():
    from actcomp import mx4

    x, w = data(5, 256, torch.bfloat16, 1).cuda(), data(40, 256, torch.bfloat16, 2).cuda()
    x[2, 100] = float("nan")
    w[7, 3] = float("inf")
    y = mx4.linear(x, mx4.quantize(w))
    bad = torch.zeros(5, 40, dtype=torch.bool, device="cuda")
    bad[2], bad[:, 7] = True, True
    assert torch.equal(y.isnan(), bad)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,k,n", [(1, 96, 40), (33, 200, 136), (256, 512, 384), (1000, 129, 257)])
def test_linear_step(tokens, k, n):
    """Forward and both gradients against float64 products of the quantised operands."""
    from actcomp import mx4

    x, w, dy = (data(*s, torch.bfloat16, i).cuda() for i, s in enumerate(((tokens, k), (n, k), (tokens, n))))
    wq, wt = mx4.quantize_pair(w)
    y, saved = mx4.linear_forward(x, wq)
    dx, dw = mx4.linear_backward(dy, saved, wt)
    assert torch.equal(y, mx4.linear(x, wq))
    val = lambda t, turn=False: values(mx4.quantize(t, transpose=turn)).cuda()  # noqa: E731
    for got, a, b in ((y, val(x), val(w)), (dx, val(dy), val(w, True)), (dw, val(dy, True), val(x, True))):
        ref, mag = a @ b.t(), a.abs() @ b.abs().t()
        assert got.shape == ref.shape
        assert not ((got.double() - ref).abs() > 2.0 ** -8 * ref.abs() + a.shape[1] * 2.0 ** -22 * mag).any()
    assert mx4.linear(x.view(1, tokens, k), wq).shape == (1, tokens, n)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("n,k", [(1, 1), (40, 96), (129, 1000), (300, 33), (64, 16384), (1000, 2080), (4096, 4096)])
def test_few_tokens(tokens, n, k):
    """The few-token kernel (and, at five tokens, the tensor cores) on the same operands."""
    from actcomp import mx4

    w = mx4.quantize(data(n, k, torch.bfloat16, n).cuda())
    for dt in DTYPES:
        x = data(tokens, k, dt, k)
        for xs in (x.cuda(), torch.nn.functional.pad(x, (3, 6)).cuda()[:, 3:3 + k]):
            q = values(mx4.quantize(x.cuda())).cuda()
            for out in {dt, torch.float32}:
                got = mx4.linear(xs, w, out)
                ref, mag = q @ values(w).cuda().t(), q.abs() @ values(w).abs().cuda().t()
                assert got.shape == ref.shape and got.dtype == out
                ok = (got.double() - ref).abs() <= U[out] * ref.abs() + k * 2.0 ** -23 * mag * (1 + U[out]) + 1e-7
                if out == torch.float16:
                    ok |= got.isinf() & (torch.sign(got) == torch.sign(ref)) & (ref.abs() + k * 2.0 ** -23 * mag >= 65520)
                assert ok.all(), (dt, out, int((~ok).sum()))


@pytest.mark.gpu
def test_few_tokens_extreme_scales():
    """Block scales near both ends of float32's range: products that are in range come out exactly."""
    from actcomp import mx4

    x, w = torch.zeros(2, 64), torch.zeros(3, 64)
    x[0, 0], x[1, 32] = 6 * 2.0 ** 124, 1.5 * 2.0 ** -127
    w[0, 0], w[1, 32], w[2, 0] = 1.5 * 2.0 ** -120, 3 * 2.0 ** 120, 4 * 2.0 ** -126
    want = x.double() @ w.double().t()
    assert torch.equal(mx4.linear(x.cuda(), mx4.quantize(w.cuda())).double().cpu(), want)
    x[0, 1] = float("inf")
    y = mx4.linear(x.cuda(), mx4.quantize(w.cuda())).cpu()
    assert y[0].isnan().all() and torch.equal(y[1].double(), want[1])


@pytest.mark.gpu
def test_refusals():
    from actcomp import mx4

    x = torch.randn(4, 64, device="cuda")
    q, q2 = mx4.quantize(x), mx4.quantize(x[:, :32])
    for bad in (lambda: mx4.matmul(q, q2), lambda: mx4.linear(x, q2), lambda: mx4.quantize(x[:0]),
                lambda: mx4.linear_forward(x, q2), lambda: mx4.linear_backward(x, q, q),
                lambda: mx4.linear_backward(x[:3], mx4.quantize(x, transpose=True), mx4.quantize(x, transpose=True))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: mx4.quantize(x.double()), lambda: mx4.dequantize(q, torch.int8),
                lambda: mx4.matmul(q, q, torch.float64)):
        with pytest.raises(TypeError):
            bad()
