"""Root-mean-square norm (with the residual's addition, with an 8-bit output) and its
backward pass against plain float64 implementations.

Tolerances.  U is the output type's unit roundoff (one rounding of the exact result).
Float32 arithmetic before it: a row's sum and the few products after it are bounded by
ROW = 64 units of 2^-24 of the row's largest intermediate (a lane adds at most 32 terms
in turn, then trees of 5 and at most 16); a sum over rows is within its length more.
An 8-bit output is the quantisation of a value that near the exact one: between those of
the two ends of that interval (rounding is monotonic)."""
import ctypes

import pytest
import torch

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
E, ROW = 2.0 ** -24, 64
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
SHAPES = [(1, 1), (3, 7), (130, 33), (9, 256), (5, 515), (70, 1000), (17, 1032), (40, 4097), (33, 4096), (9, 5120),
          (5, 9216), (3, 16384), (3, 16390), (3, 20000)]


def data(rows, cols, dtype, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, cols, generator=g) * spread + 0.3 * torch.randn(rows, 1, generator=g)).to(dtype)


def rms64(h, w, eps):
    rstd = (h.square().mean(-1) + eps).rsqrt()
    return h * rstd[..., None] * (1 if w is None else w), rstd


def rms_bwd64(dy, x, w, rstd, dh):
    """dx, the terms of dw, and a bound of dx's intermediates."""
    g = dy if w is None else dy * w
    xh = x * rstd[:, None]
    dx = rstd[:, None] * (g - xh * (g * xh).mean(1, keepdim=True)) + (0 if dh is None else dh)
    mag = rstd.abs()[:, None] * (g.abs() + xh.abs() * (g * xh).abs().mean(1, keepdim=True))
    return dx, dy * xh, mag + (0 if dh is None else dh.abs())


def close(got, ref, u, slack):
    got, ref = got.double().cpu(), ref.double().cpu()
    bad = ~((got - ref).abs() <= u * ref.abs() + slack + 1e-7 * (u > 2 ** -24) + 1e-37)
    assert not bad.any(), (int(bad.sum()), float((got - ref).abs().max()))


# ---------------------------------------------------------------- CPU
def test_formula_against_differences():
    g = torch.Generator().manual_seed(1)
    x, w, dy, dh = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((3, 11), (11,), (3, 11), (3, 11)))
    f = lambda x, w: (rms64(x, w, 1e-3)[0] * dy).sum() + (x * dh).sum()  # noqa: E731
    dx, terms, _ = rms_bwd64(dy, x, w, rms64(x, w, 1e-3)[1], dh)
    for t, grad in ((x, dx), (w, terms.sum(0))):
        for i in range(t.numel()):
            step = torch.zeros(t.numel(), dtype=torch.float64)
            step[i] = 1e-5
            a, b = t + step.view(t.shape), t - step.view(t.shape)
            num = (f(a, w) - f(b, w)) / 2e-5 if t is x else (f(x, a) - f(x, b)) / 2e-5
            assert abs(float(num - grad.flatten()[i])) < 1e-8


def test_entry_points_validate_without_gpu():
    from actcomp import _lib

    lib = _lib.load()
    P = 1 << 20  # aligned, never dereferenced
    base = dict(rows=4, cols=16, x=P, ldx=16, y=P, ldy=16, rstd=P, dtype=1, wdtype=1, eps=1e-5)
    f = lambda **k: lib.actcomp_rms_norm(ctypes.byref(_lib.RmsArgs(**{**base, **k})), None)  # noqa: E731
    assert lib.actcomp_rms_norm(None, None) == _lib.ACT_E_INVALID
    assert f(rows=0) == _lib.ACT_OK
    for bad in (dict(cols=0), dict(wdtype=2), dict(dtype=3), dict(eps=-1.0), dict(eps=float("nan")), dict(rstd=None),
                dict(ldy=15), dict(y=None), dict(res=P, ldr=16, ldh=16), dict(res=P, h=P, ldr=8, ldh=16),
                dict(codes=P, scales=P, ldc=16), dict(y=None, codes=P, ldc=16), dict(y=None, codes=P, scales=P, ldc=0)):
        assert f(**bad) == _lib.ACT_E_INVALID, bad
    assert f(rstd=P + 2) == _lib.ACT_E_ALIGN and f(x=P + 1) == _lib.ACT_E_ALIGN
    assert f(y=None, codes=P, scales=P, ldc=24) == _lib.ACT_E_ALIGN
    assert f(y=None, codes=P + 8, scales=P, ldc=16) == _lib.ACT_E_ALIGN
    assert f(cols=1 << 31, ldx=1 << 31, ldy=1 << 31) == _lib.ACT_E_UNSUPPORTED
    need = lib.actcomp_rms_norm_bwd_workspace(4, 16)
    assert need > 0 and lib.actcomp_rms_norm_bwd_workspace(0, 16) == 0
    bw = dict(rows=4, cols=16, dy=P, lddy=16, x=P, ldx=16, rstd=P, dx=P, lddx=16, dtype=1, wdtype=0)
    back = lambda ws=P, n=need, **k: lib.actcomp_rms_norm_bwd(  # noqa: E731
        ctypes.byref(_lib.RmsBwdArgs(**{**bw, **k})), ws, n, None)
    for bad in (dict(cols=0), dict(dy=None), dict(rstd=None), dict(dh=P, lddh=8), dict(lddx=8), dict(wdtype=2)):
        assert back(**bad) == _lib.ACT_E_INVALID, bad
    assert back(dweight=P + 2) == _lib.ACT_E_ALIGN
    assert back(n=need - 1) == _lib.ACT_E_WORKSPACE and back(ws=None) == _lib.ACT_E_WORKSPACE


def test_calls_are_refused():
    import actcomp

    x = torch.zeros(2, 8)
    for call in (lambda: actcomp.rms_norm(x), lambda: actcomp.add_rms_norm(x, x),
                 lambda: actcomp.rms_norm_backward(x, x, None, torch.zeros(2)), lambda: actcomp.fp8.rms_norm(x)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


# ---------------------------------------------------------------- forward
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_forward(dtype, rows, cols):
    import actcomp

    x, r = data(rows, cols, dtype, rows), data(rows, cols, dtype, cols, 3.0)
    for wt in {None, dtype, torch.float32}:
        w = None if wt is None else data(1, cols, wt, 7)[0]
        wd, wc = (None, None) if w is None else (w.double(), w.cuda())
        y, rstd = actcomp.rms_norm(x.cuda(), wc, 1e-5)
        ref, s = rms64(x.double(), wd, 1e-5)
        close(y, ref, U[dtype], ROW * E * ref.abs())
        close(rstd, s, 0, ROW * E * s)
        y, h, rstd = actcomp.add_rms_norm(x.cuda(), r.cuda(), wc, 1e-5)
        sum64 = x.double() + r.double()
        ref, s = rms64(sum64, wd, 1e-5)
        close(y, ref, U[dtype], ROW * E * ref.abs())
        close(h, sum64, U[dtype], E * sum64.abs())
        close(rstd, s, 0, ROW * E * s)


def scale_of(amax):
    """Scale byte of a block from its largest magnitude (float64), e4m3."""
    m, e = torch.frexp(amax)
    e = e.long() - 1 - 8 + (2 * m > 1.75)
    return torch.where(amax > 0, e, -127).clamp_min(-127) + 127


def e4m3(v):
    grid = torch.exp2((torch.frexp(v.abs()).exponent.double() - 1).clamp_min(-6) - 3)
    return (torch.round(v / grid) * grid).clamp(-448, 448)


def line_scales(q):
    """Scale bytes of a matrix by rows, as (rows, blocks)."""
    lines = q.rows
    groups = -(-lines // 128)
    s = q.scales.cpu().view(-1, groups, 32, 4).permute(0, 1, 3, 2).reshape(-1, groups * 128)
    return s[:, :lines].t().long()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("add", [False, True])
def test_8bit_output(dtype, rows, cols, add):
    from actcomp import fp8

    x, r, w = data(rows, cols, dtype, 3), data(rows, cols, dtype, 4, 2.0), data(1, cols, dtype, 5)[0]
    if add:
        q, h, rstd = fp8.add_rms_norm(x.cuda(), r.cuda(), w.cuda())
        sum64 = x.double() + r.double()
        close(h, sum64, U[dtype], E * sum64.abs())
    else:
        q, rstd = fp8.rms_norm(x.cuda(), w.cuda())
        sum64 = x.double()
    ref, s = rms64(sum64, w.double(), 1e-5)
    close(rstd, s, 0, ROW * E * s)
    assert (q.rows, q.cols, q.format, q.transposed, q.tiles) == (rows, cols, "e4m3", False, False)
    nb = -(-cols // 128)
    slack = ROW * E * ref.abs()
    amax = torch.nn.functional.pad(ref.abs(), (0, nb * 128 - cols)).view(rows, nb, 128).amax(-1)
    sc = line_scales(q)
    assert ((sc >= scale_of(amax * (1 - ROW * E))) & (sc <= scale_of(amax * (1 + ROW * E)))).all()
    f = torch.exp2(sc.double() - 127).repeat_interleave(128, 1)[:, :cols]
    got = fp8.dequantize(q, torch.float32).double().cpu()
    lo, hi = e4m3((ref - slack) / f) * f, e4m3((ref + slack) / f) * f
    assert ((got >= lo) & (got <= hi)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_8bit_output_special_rows(dtype):
    """Zero rows, rows with a NaN or an infinity, and tiny ones."""
    from actcomp import fp8

    x = data(300, 400, dtype, 9)
    x[3] = 0
    x[5, 17], x[140, 300], x[299] = float("nan"), float("inf"), x[299] * 2 ** -14
    q, rstd = fp8.rms_norm(x.cuda(), None, 0.0 if dtype != torch.float16 else 1e-12)
    v = fp8.dequantize(q, torch.float32).cpu()
    assert v[5].isnan().all() and v[140, 256:384].isnan().all()
    ok = torch.ones(300, dtype=torch.bool)
    ok[[3, 5, 140]] = False
    assert torch.isfinite(v[ok]).all()
    ref, _ = rms64(x.double()[ok], None, 0.0 if dtype != torch.float16 else 1e-12)
    assert ((v[ok] - ref).abs() <= 2.0 ** -4 * ref.abs() * 1.001 + 2.0 ** -10 * ref.abs().amax(1, keepdim=True)).all()


@pytest.mark.gpu
def test_forward_shapes_strides_and_empty():
    import actcomp
    from actcomp import fp8

    x = data(60, 80, torch.bfloat16, 1).cuda()
    w = data(1, 48, torch.bfloat16, 2)[0].cuda()
    ref, s = actcomp.rms_norm(x[:, 8:56].contiguous(), w)
    for v in (x[:, 8:56], torch.nn.functional.pad(x, (1, 0))[:, 9:57], x[:, 8:56].view(4, 15, 48)):
        y, rstd = actcomp.rms_norm(v, w)
        assert y.shape == v.shape and rstd.shape == v.shape[:-1]
        assert (y.reshape(60, 48).float() - ref.float()).abs().max() <= 2.0 ** -6 * ref.float().abs().max()
        q, rstd = fp8.rms_norm(v, w)
        assert q.shape == (60, 48) and rstd.shape == v.shape[:-1]
    y, rstd = actcomp.rms_norm(x[:1, 8:56].expand(5, 48), w)
    assert torch.equal(y, ref[:1].expand(5, 48))
    y, h, rstd = actcomp.add_rms_norm(x.t()[:40], x.t()[:40], None)
    assert torch.equal(h, (2 * x.t()[:40].float()).bfloat16())
    y, rstd = actcomp.rms_norm(x[:0], None)
    assert y.shape == (0, 80) and rstd.shape == (0,)
    dx, dw = actcomp.rms_norm_backward(y, y, x[0], rstd)
    assert dx.shape == (0, 80) and not dw.any()
    with pytest.raises(ValueError):
        fp8.rms_norm(x[:0])
    for bad in (lambda: actcomp.rms_norm(x, w), lambda: actcomp.add_rms_norm(x, x[:30]), lambda: actcomp.rms_norm(x[:, :0]),
                lambda: actcomp.rms_norm(x, None, -1.0), lambda: actcomp.rms_norm_backward(x, x, None, s[:3]),
                lambda: actcomp.rms_norm_backward(x, x, None, s, dh=x.float())):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        actcomp.rms_norm(x, x[0].half())
    with pytest.raises(TypeError):
        actcomp.rms_norm(x.double())


# ---------------------------------------------------------------- backward
def check_backward(dtype, rows, cols, wt, add):
    import actcomp

    x, dy, dh = data(rows, cols, dtype, 1), data(rows, cols, dtype, 2), data(rows, cols, dtype, 3) if add else None
    w = None if wt is None else data(1, cols, wt, 7)[0]
    rstd = (x.float().square().mean(1) + 1e-5).rsqrt()
    dx, dw = actcomp.rms_norm_backward(dy.cuda(), x.cuda(), None if w is None else w.cuda(), rstd.cuda(),
                                       None if dh is None else dh.cuda())
    ref, terms, mag = rms_bwd64(dy.double(), x.double(), None if w is None else w.double(), rstd.double(),
                                None if dh is None else dh.double())
    close(dx, ref, U[dtype], ROW * E * mag)
    if w is None:
        assert dw is None
    else:
        assert dw.dtype == w.dtype
        close(dw, terms.sum(0), U[w.dtype], (ROW + rows) * E * terms.abs().sum(0))
        again = actcomp.rms_norm_backward(dy.cuda(), x.cuda(), w.cuda(), rstd.cuda(), None if dh is None else dh.cuda())
        assert torch.equal(again[0], dx) and torch.equal(again[1], dw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", SHAPES + [(1000, 64), (700, 600), (2000, 2048), (5, 13952), (4, 13960), (6, 9304)])
def test_backward(dtype, rows, cols):
    for wt in {None, dtype, torch.float32}:
        for add in (False, True):
            check_backward(dtype, rows, cols, wt, add)


@pytest.mark.gpu
def test_many_rows_in_turn():
    """More rows than resident CTAs take at once: slots are filled again."""
    for dtype in (torch.bfloat16, torch.float32):
        for rows, cols in ((20000, 128), (9000, 520), (3001, 4096), (1500, 8192), (1200, 9216)):
            check_backward(dtype, rows, cols, dtype, True)
            test_forward(dtype, rows, cols)


# ---------------------------------------------------------------- streams and graphs
@pytest.mark.gpu
def test_other_stream_and_graph():
    import actcomp
    from actcomp import fp8

    x, r, w = (data(*s, torch.bfloat16, i).cuda() for i, s in enumerate(((64, 2048), (64, 2048), (1, 2048))))
    w = w[0]

    def step():
        y, h, rstd = actcomp.add_rms_norm(x, r, w)
        q, _, _ = fp8.add_rms_norm(x, r, w)
        return (y, h, rstd, fp8.dequantize(q)) + actcomp.rms_norm_backward(y, h, w, rstd, dh=h)

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
    for v in (data(64, 2048, torch.bfloat16, 50).cuda(), first):
        x.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
