"""8-bit floating point with a scale per block of 128: the format against a plain
restatement, bit for bit; the products against float64 products of the values that the
operands stand for.

Tolerance of a product: the operands' products are exact in float32, a sum of K terms in
any order with each addition rounded or truncated is within K 2^-23 sum|terms|, and the
result is rounded once to the output type."""
import ctypes

import pytest
import torch

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
# mantissa bits, exponent bias, largest value's exponent
FORMATS = {"e4m3": (3, 7, 8), "e5m2": (2, 15, 15)}


# ---------------------------------------------------------------- plain form
def code_values(fmt):
    """Value of each of the 256 codes, from the encoding's definition."""
    bits, bias, _ = FORMATS[fmt]
    c = torch.arange(256)
    e, m = (c & 127) >> bits, (c & ((1 << bits) - 1)).double()
    v = torch.where(e == 0, m * 2.0 ** (1 - bias - bits), (1 + m / 2 ** bits) * torch.exp2((e - bias).double()))
    if fmt == "e4m3":
        v[(c & 127) == 127] = float("nan")
    else:
        v[(c & 127) == 124], v[(c & 127) > 124] = float("inf"), float("nan")
    return torch.where(c >= 128, -v, v)


def blocks_amax(v, br, bc):
    rows, cols = v.shape
    p = torch.nn.functional.pad(v.abs(), (0, -cols % bc, 0, -rows % br))
    return p.view(p.shape[0] // br, br, p.shape[1] // bc, bc).amax((1, 3))


def encode64(v, br, bc, fmt):
    """(value of each code, scale byte of each block) of a float64 matrix by the definition."""
    bits, bias, top = FORMATS[fmt]
    amax = blocks_amax(v, br, bc)
    m, e = torch.frexp(amax)
    e = e.long() - 1 - top + (2 * m > 1.75)  # both formats' largest value is 1.75 2^top
    byte = torch.where(amax > 0, e, -127).clamp_min(-127) + 127
    byte = torch.where(torch.isfinite(amax), byte, 255)
    f = torch.exp2(byte.double() - 127).repeat_interleave(br, 0).repeat_interleave(bc, 1)[: v.shape[0], : v.shape[1]]
    a = v / f
    grid = torch.exp2((torch.frexp(a.abs()).exponent.double() - 1).clamp_min(1 - bias) - bits)
    return torch.round(a / grid) * grid, byte


def stored(q):
    """(codes without padding, scale bytes per block) as the buffers hold them."""
    rows, cols = (q.cols, q.rows) if q.transposed else (q.rows, q.cols)
    codes, s = q.codes.cpu()[:, :cols].long(), q.scales.cpu().long()
    assert q.codes.shape == (rows, -(-cols // 16) * 16)
    rb, cb = -(-rows // 128), -(-cols // 128)
    if q.tiles:
        return codes, s.view(rb, cb)
    lines, groups, n = (cols, cb, rb) if q.transposed else (rows, rb, cb)
    b = s.view(n, groups, 32, 4).permute(0, 1, 3, 2).reshape(n, groups * 128)[:, :lines]
    return codes, b if q.transposed else b.t()


def block_of(q):
    return (128, 128) if q.tiles else (128, 1) if q.transposed else (1, 128)


def values(q):
    """What q stands for, (rows, cols), float64."""
    codes, byte = stored(q)
    br, bc = block_of(q)
    f = torch.exp2(byte.double() - 127)
    f[byte == 255] = float("nan")
    v = code_values(q.format)[codes] * f.repeat_interleave(br, 0).repeat_interleave(bc, 1)[: codes.shape[0], : codes.shape[1]]
    return v.t() if q.transposed else v


def data(rows, cols, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * torch.exp2(torch.randint(-6, 7, (rows, 1), generator=g).float())
    x[torch.rand(rows, cols, generator=g) < 0.1] = 0
    return x.to(dtype)


def check_codes(q, v):
    """q's buffers against the definition for the stored matrix v."""
    codes, byte = stored(q)
    want, wb = encode64(v.double(), *block_of(q), q.format)
    assert torch.equal(byte, wb)
    br, bc = block_of(q)
    fine = (wb != 255).repeat_interleave(br, 0).repeat_interleave(bc, 1)[: v.shape[0], : v.shape[1]]
    got = code_values(q.format)[codes]
    assert torch.equal(got[fine], want[fine])
    assert torch.equal((codes >= 128)[fine], torch.signbit(v.cpu())[fine])


# ---------------------------------------------------------------- CPU
def test_sizes_and_validation_without_gpu():
    from actcomp import _lib

    lib = _lib.load()
    assert lib.actcomp_fp8_scale_bytes(129, 257, 0) == 2 * 3 * 128 and lib.actcomp_fp8_scale_bytes(129, 257, 2) == 6
    assert lib.actcomp_fp8_scale_bytes(0, 5, 0) == 0 and lib.actcomp_fp8_scale_bytes(5, 5, 3) == 0
    P, I, A, N = 1 << 20, _lib.ACT_E_INVALID, _lib.ACT_E_ALIGN, _lib.ACT_E_UNSUPPORTED
    d = lambda r=64, c=96, ld=96, codes=P, scales=P, fmt=0, block=0, tr=None: ctypes.byref(  # noqa: E731
        _lib.Fp8Desc(r, c, ld, codes, scales, fmt, block, (block == 1) if tr is None else tr, 0))
    quant = lambda q, qt, x=P, ld=96, dt=1: lib.actcomp_fp8_quantize(x, 64, 96, ld, dt, q, qt, None)  # noqa: E731
    assert quant(None, None) == I and quant(d(), None, x=None) == I and quant(d(), None, ld=95) == I
    assert quant(d(96, 64), None) == I and quant(d(block=1), None) == I and quant(None, d()) == I
    assert quant(d(block=2), d(block=1)) == I and quant(d(), d(block=1, fmt=1)) == I
    assert quant(d(fmt=2), None) == I and quant(d(block=3), None) == I and quant(d(tr=1), None) == I
    assert quant(None, d(block=1, tr=0)) == I and quant(d(), None, dt=3) == I and quant(d(ld=80), None) == I
    assert quant(d(codes=P + 8), None) == A and quant(d(ld=104), None) == A and quant(d(), None, x=P + 1) == A
    gemm = lambda a, b, ld=64, dt=1, c=P: lib.actcomp_fp8_gemm(a, b, c, ld, dt, None)  # noqa: E731
    assert gemm(d(), d(64, 128, 128)) == I and gemm(d(), d(), ld=63) == I and gemm(d(), d(), dt=5) == I
    assert gemm(d(), d(), c=P + 1) == A and gemm(d(0), d()) == I and gemm(d(), d(block=1)) == I
    assert lib.actcomp_fp8_dequantize(d(), P, 95, 1, None) == I
    assert lib.actcomp_fp8_dequantize(d(1 << 31), P, 96, 1, None) == N


def test_calls_are_refused():
    from actcomp import fp8

    with pytest.raises(ValueError, match="CUDA"):
        fp8.quantize(torch.zeros(4, 32))
    with pytest.raises(ValueError, match="format"):
        fp8.quantize(torch.zeros(4, 32), format="e3m4")
    e = torch.empty(0, dtype=torch.uint8)
    with pytest.raises(ValueError, match="transpose"):
        fp8.Fp8(4, 4, e, e, torch.float32).t()
    with pytest.raises(ValueError, match="inner"):
        fp8.matmul(fp8.Fp8(4, 4, e, e, torch.float32), fp8.Fp8(4, 5, e, e, torch.float32))


def test_code_values_of_the_plain_form():
    """The restatement's tables against torch's types."""
    for fmt, t in (("e4m3", torch.float8_e4m3fn), ("e5m2", torch.float8_e5m2)):
        want = torch.arange(256, dtype=torch.uint8).view(t).double()
        got = code_values(fmt)
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got[~got.isnan()], want[~want.isnan()])


# ---------------------------------------------------------------- quantisation
SHAPES = [(1, 1), (1, 127), (3, 128), (2, 129), (130, 40), (128, 256), (33, 257), (300, 70), (129, 129), (40, 1000),
          (257, 384)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", list(FORMATS))
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quantise(dtype, fmt, rows, cols):
    from actcomp import fp8

    x = data(rows, cols, dtype, rows + cols)
    xc = x.cuda()
    q, qt, w = fp8.quantize(xc, format=fmt), fp8.quantize(xc, transpose=True, format=fmt), fp8.quantize_weight(xc, fmt)
    assert q.shape == w.shape == (rows, cols) and qt.shape == w.t().shape == (cols, rows)
    for t in (q, qt, w):
        check_codes(t, x)
    for a, b in zip(fp8.quantize_pair(xc, format=fmt), (q, qt)):
        assert torch.equal(a.codes[:, :cols], b.codes[:, :cols])
        assert all(torch.equal(u, v) for u, v in zip(stored(a), stored(b)))
    for t in (q, qt, w, w.t()):
        for out in DTYPES:
            got = fp8.dequantize(t, out)
            assert got.shape == t.shape and torch.equal(got.double().cpu(), values(t).to(out).double())
    padded = torch.nn.functional.pad(xc, (1, 2))[:, 1:1 + cols]  # rows that are not 16-byte aligned
    for a, b in ((fp8.quantize(padded, format=fmt), q), (fp8.quantize_weight(padded, fmt), w)):
        assert all(torch.equal(u, v) for u, v in zip(stored(a), stored(b)))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", list(FORMATS))
def test_quantise_special_values(fmt):
    """Ties, the largest magnitude at its scale's border, signs, zero and subnormal
    blocks, the largest float32, NaN and infinity."""
    from actcomp import fp8

    top = 2.0 ** FORMATS[fmt][2]
    grid = code_values(fmt)[:128]
    grid = grid[torch.isfinite(grid)]
    mids = torch.cat([(grid[:-1] + grid[1:]) / 2, grid])
    v = torch.zeros(24, 384)
    for i, s in enumerate((1.0, 2.0 ** 60, 2.0 ** -90, 2.0 ** -116)):
        v[i, : mids.numel()] = (mids * s).float()
        v[i, 1:mids.numel():3] *= -1
    up = torch.nextafter(torch.tensor(1.75 * top), torch.tensor(1e9)).item()
    for i, a in enumerate((1.75 * top, up, top, 1.0, 1.75, 1e-45, 2.0 ** -126, 3.4e38, 2.0 ** -119 * 1.75)):
        v[6 + i, 0], v[6 + i, 130] = a, -a / 3
    v[16, 3], v[17, 140], v[18, 5], v[19, 300] = float("nan"), float("inf"), -0.0, float("-inf")
    x = v.cuda()
    for q in (fp8.quantize(x, format=fmt), fp8.quantize(x, transpose=True, format=fmt), fp8.quantize_weight(x, fmt)):
        check_codes(q, v)
        d = fp8.dequantize(q, torch.float32)
        want = values(q).float()  # the largest block's value may round past float32: infinity
        same = (d.cpu() == want) | (d.cpu().isnan() & want.isnan())
        assert same.all(), same.logical_not().nonzero()[:4].tolist()


# ---------------------------------------------------------------- products
def product_close(got, a, b, dtype):
    va, vb = values(a).cuda(), values(b).cuda()
    ref, mag = va @ vb.t(), va.abs() @ vb.abs().t()
    assert got.shape == ref.shape and got.dtype == dtype
    ref = torch.where(ref.to(dtype).isinf(), ref.to(dtype).double(), ref)  # past the output type: infinity
    bad = (got.double() != ref) & ~((got.double() - ref).abs() <= U[dtype] * ref.abs() + a.cols * 2.0 ** -23 * mag * (1 + U[dtype]) + 1e-7)
    assert not bad.any(), (int(bad.sum()), float((got.double() - ref).abs().max()), bad.nonzero()[:4].tolist())


SIZES = [(1, 1, 1), (3, 5, 128), (130, 33, 129), (256, 256, 256), (257, 300, 1000), (100, 700, 97), (16, 1024, 2048),
         (513, 129, 640), (8, 11008, 130), (1000, 511, 384)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", SIZES)
def test_product_of_every_block_form(m, n, k):
    from actcomp import fp8

    x, y = data(m, k, torch.bfloat16, 1).cuda(), data(n, k, torch.bfloat16, 2).cuda()

    def forms(v):
        t = v.t().contiguous()
        return [fp8.quantize(v), fp8.quantize(t, transpose=True), fp8.quantize_weight(v), fp8.quantize_weight(t).t()]

    for a in forms(x):
        for b in forms(y):
            product_close(fp8.matmul(a, b), a, b, torch.bfloat16)
    for out in DTYPES:
        a, b = fp8.quantize(x), fp8.quantize_weight(y)
        product_close(fp8.matmul(a, b, out), a, b, out)


@pytest.mark.gpu
@pytest.mark.parametrize("fa,fb", [("e5m2", "e4m3"), ("e4m3", "e5m2"), ("e5m2", "e5m2")])
def test_product_of_formats(fa, fb):
    from actcomp import fp8

    for m, n, k in ((5, 300, 520), (300, 260, 520)):
        a, b = fp8.quantize(data(m, k, torch.float16, 3).cuda(), format=fa), fp8.quantize_weight(
            data(n, k, torch.float16, 4).cuda(), fb)
        product_close(fp8.matmul(a, b, torch.float32), a, b, torch.float32)
        at = fp8.quantize(data(k, m, torch.float32, 5).cuda(), transpose=True, format=fa)
        product_close(fp8.matmul(at, b, torch.float32), at, b, torch.float32)


@pytest.mark.gpu
def test_product_nan_stays_in_its_row_and_column():
    from actcomp import fp8

    x, y = data(300, 400, torch.bfloat16, 1).cuda(), data(500, 400, torch.bfloat16, 2).cuda()
    x[7, 390], y[260, 3] = float("nan"), float("inf")
    for a, rows in ((fp8.quantize(x), 300), (fp8.quantize(x[5:8]), 3)):
        c = fp8.matmul(a, fp8.quantize(y))
        bad = torch.zeros(rows, 500, dtype=torch.bool, device="cuda")
        bad[7 if rows == 300 else 2], bad[:, 260] = True, True
        assert torch.equal(c.isnan(), bad)


@pytest.mark.gpu
def test_product_leaves_what_lies_behind():
    """Rows and columns past the result keep what they held."""
    from actcomp import _lib, fp8

    lib = _lib.load()
    for m, n, ld, dt, tdt in ((70, 90, 128, 1, torch.bfloat16), (3, 300, 301, 0, torch.float32), (260, 270, 272, 2, torch.float16)):
        a, b = fp8.quantize(data(m, 200, torch.bfloat16, 1).cuda()), fp8.quantize_weight(data(n, 200, torch.bfloat16, 2).cuda())
        out = torch.full((m + 3, ld), 7.0, dtype=tdt, device="cuda")
        da, db = (_lib.Fp8Desc(q.rows, q.cols, q.codes.size(1), q.codes.data_ptr(), q.scales.data_ptr(), 0,
                               2 if q.tiles else 0, 0, 0) for q in (a, b))
        s = torch.cuda.current_stream().cuda_stream
        assert lib.actcomp_fp8_gemm(ctypes.byref(da), ctypes.byref(db), out.data_ptr(), ld, dt, s) == _lib.ACT_OK
        torch.cuda.synchronize()
        assert (out[m:] == 7).all() and (out[:, n:] == 7).all()
        product_close(out[:m, :n].contiguous(), a, b, tdt)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,k,n", [(1, 64, 40), (2, 1000, 300), (8, 4096, 1024), (9, 130, 257), (300, 520, 260)])
def test_linear_layer(dtype, tokens, k, n):
    from actcomp import fp8

    x, dy = data(tokens, k, dtype, 1).cuda(), data(tokens, n, dtype, 2).cuda()
    w = fp8.quantize_weight(data(n, k, torch.bfloat16, 3).cuda())
    q, qt = fp8.quantize_pair(x)
    product_close(fp8.linear(x, w), q, w, dtype)
    product_close(fp8.linear(x, w, torch.float32), q, w, torch.float32)
    y, saved = fp8.linear_forward(x.view(1, tokens, k), w)
    assert y.shape == (1, tokens, n) and torch.equal(y[0], fp8.matmul(q, w, dtype))
    assert all(torch.equal(u, v) for u, v in zip(stored(saved), stored(qt)))
    dx, dw = fp8.linear_backward(dy.view(1, tokens, n), saved, w)
    g, gt = fp8.quantize_pair(dy)
    assert dx.shape == (1, tokens, k)
    product_close(dx[0], g, w.t(), dtype)
    product_close(dw, gt, saved, dtype)
    g, gt = fp8.quantize_pair(dy, "e5m2")
    dx, dw = fp8.linear_backward(dy, saved, w, torch.float32, grad_format="e5m2")
    product_close(dx, g, w.t(), torch.float32)
    product_close(dw, gt, saved, torch.float32)


@pytest.mark.gpu
def test_linear_layer_refusals():
    from actcomp import fp8

    x, w = data(4, 256, torch.bfloat16, 1).cuda(), fp8.quantize_weight(data(300, 256, torch.bfloat16, 2).cuda())
    y, saved = fp8.linear_forward(x, w)
    for bad in (lambda: fp8.linear(x[:, :128], w), lambda: fp8.linear(x[:0], w), lambda: fp8.linear_forward(x[:, :128], w),
                lambda: fp8.linear_backward(y[:, :200], saved, w), lambda: fp8.linear_backward(y[:2], saved, w),
                lambda: fp8.linear_backward(y, saved, fp8.quantize(data(300, 256, torch.bfloat16, 2).cuda())),
                lambda: fp8.quantize(x[:0]), lambda: fp8.matmul(w, fp8.quantize(x[:, :128])),
                lambda: fp8.matmul(fp8.Fp8(8, 256, w.codes, w.scales, x.dtype), w)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        fp8.quantize(x.double())
    with pytest.raises(TypeError):
        fp8.matmul(w, w, torch.int32)


# ---------------------------------------------------------------- streams and graphs
@pytest.mark.gpu
def test_other_stream_and_graph():
    from actcomp import fp8

    x, wt = data(48, 640, torch.bfloat16, 1).cuda(), data(384, 640, torch.bfloat16, 2).cuda()

    def step():
        w = fp8.quantize_weight(wt)
        y, saved = fp8.linear_forward(x, w)
        return (y, fp8.linear(x[:1], w)) + fp8.linear_backward(y, saved, w)

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    first = x.clone()
    for v in (data(48, 640, torch.bfloat16, 9).cuda(), first):
        x.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
