"""Dropout without a stored mask, layer norm with its backward pass, and both
across a residual branch, against plain float64 implementations.

Tolerances.  u is the output type's unit roundoff (2^-24, 2^-8, 2^-11 for
float32, bf16, fp16): one rounding of the exact result.  Float32 arithmetic
before it: a sum of n terms in any order is within n 2^-24 sum|terms|; a row's
statistics and the few products after them are bounded by ROW = 64 units of
2^-24 of the row's largest intermediate (lanes add at most 32 terms in turn,
then trees of 5 and at most 16)."""
import ctypes
import os
import subprocess
import tempfile

import numpy as np
import pytest
import torch

from conftest import ROOT

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
E = 2.0 ** -24
ROW = 64
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
M32 = 0xFFFFFFFF


# ---------------------------------------------------------------- plain forms
def philox(ctr, key):
    """Philox4x32-10 on numpy uint64 arrays that hold 32-bit words."""
    c = [np.asarray(v, np.uint64) for v in ctr]
    k = [int(v) for v in key]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & np.uint64(M32),
             (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & np.uint64(M32)]
        k = [(k[0] + 0x9E3779B9) & M32, (k[1] + 0xBB67AE85) & M32]
    return c


def keep_mask(rows, cols, p, seed, row_offset=0):
    r = np.arange(rows, dtype=np.uint64)[:, None] + np.uint64(row_offset)
    blk = np.arange((cols + 7) // 8, dtype=np.uint64)[None, :]
    z = np.zeros((rows, blk.shape[1]), np.uint64)
    w = philox([z + blk, z, (r & np.uint64(M32)) + z, (r >> np.uint64(32)) + z], [seed & M32, seed >> 32])
    halves = np.stack([w[j // 2] >> np.uint64(16 * (j % 2)) & np.uint64(0xFFFF) for j in range(8)], -1)
    return torch.from_numpy(halves.reshape(rows, -1)[:, :cols] >= round(p * 65536))


def held_scale(p):
    t = round(p * 65536)
    return 65536.0 / (65536 - t) if t < 65536 else 0.0


def ln64(x, w, b, eps):
    mean = x.mean(-1)
    xc = x - mean[..., None]
    rstd = (xc.square().mean(-1) + eps).rsqrt()
    xh = xc * rstd[..., None]
    return xh * (1 if w is None else w) + (0 if b is None else b), mean, rstd


def ln_bwd64(dy, x, w, mean, rstd):
    xh = (x - mean[:, None]) * rstd[:, None]
    g = dy if w is None else dy * w
    dx = rstd[:, None] * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    return dx, (dy * xh), xh


def close(got, ref, u, slack):
    """|got - ref| <= u |ref| + slack, with the type's smallest subnormal allowed for."""
    got, ref = got.double().cpu(), ref.double().cpu()
    slack = torch.as_tensor(slack, dtype=torch.float64).cpu()
    bad = (got - ref).abs() > u * ref.abs() + slack + 1e-7 * (u > 2 ** -24)
    assert not bad.any(), (int(bad.sum()), float((got - ref).abs().max()))


def data(rows, cols, dtype, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * spread + 0.5 * torch.randn(rows, 1, generator=g)
    return x.to(dtype)


# ---------------------------------------------------------------- CPU
def test_philox_known_answers():
    """The generator's published test vectors."""
    pi = [0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], [0xA4093822, 0x299F31D0]
    for (c, k), want in (
            (([0] * 4, [0] * 2), [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]),
            (([M32] * 4, [M32] * 2), [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]),
            (pi, [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1])):
        assert [int(v) for v in philox(c, k)] == want


def test_struct_layouts_match_the_header():
    from actcomp import _lib

    structs = {"actcomp_drop_args": _lib.DropArgs, "actcomp_ln_args": _lib.LnArgs,
               "actcomp_ln_bwd_args": _lib.LnBwdArgs, "actcomp_mx4": _lib.Mx4Desc}
    lines = ['#include <stdio.h>', '#include <stddef.h>',
             f'#include "{os.path.join(ROOT, "include", "actcomp.h")}"', "int main(void){"]
    for c, py in structs.items():
        lines.append(f'printf("{c} %zu\\n", sizeof({c}));')
        lines += [f'printf("{c}.{f} %zu\\n", offsetof({c}, {f}));' for f, _ in py._fields_]
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "p.c"), os.path.join(d, "p")
        open(src, "w").write("\n".join(lines) + "return 0;}")
        subprocess.run(["gcc", "-std=c11", src, "-o", exe], check=True)
        got = dict(ln.split() for ln in subprocess.check_output([exe], text=True).splitlines())
    for c, py in structs.items():
        assert int(got[c]) == ctypes.sizeof(py), c
        for f, _ in py._fields_:
            assert int(got[f"{c}.{f}"]) == getattr(py, f).offset, f"{c}.{f}"


def test_entry_points_validate_without_gpu():
    from actcomp import _lib

    lib = _lib.load()
    P = 1 << 20  # aligned, never dereferenced
    drop = lambda **k: lib.actcomp_dropout(ctypes.byref(_lib.DropArgs(  # noqa: E731
        **{**dict(rows=4, cols=16, x=P, ldx=16, y=P, ldy=16, dtype=1, p=0.1), **k})), None)
    assert lib.actcomp_dropout(None, None) == _lib.ACT_E_INVALID
    assert drop(rows=0) == _lib.ACT_OK and drop(cols=0) == _lib.ACT_OK  # nothing to do
    for bad in (dict(p=-0.1), dict(p=1.5), dict(p=float("nan")), dict(dtype=3), dict(ldx=8), dict(x=None),
                dict(rows=-1)):
        assert drop(**bad) == _lib.ACT_E_INVALID, bad
    assert drop(x=P + 1) == _lib.ACT_E_ALIGN and drop(seed_ptr=P + 4) == _lib.ACT_E_ALIGN
    base = dict(rows=4, cols=16, x=P, ldx=16, y=P, ldy=16, mean=P, rstd=P, dtype=1, wdtype=1, eps=1e-5)
    ln = lambda **k: lib.actcomp_layer_norm(ctypes.byref(_lib.LnArgs(**{**base, **k})), None)  # noqa: E731
    assert ln(rows=0) == _lib.ACT_OK
    for bad in (dict(cols=0), dict(wdtype=2), dict(eps=-1.0), dict(mean=None), dict(ldy=15),
                dict(res=P, ldr=16, ldh=16), dict(res=P, h=P, ldr=16, ldh=16, p=2.0)):
        assert ln(**bad) == _lib.ACT_E_INVALID, bad
    assert ln(rstd=P + 2) == _lib.ACT_E_ALIGN
    bw = dict(rows=4, cols=16, dy=P, lddy=16, x=P, ldx=16, mean=P, rstd=P, dx=P, lddx=16, dtype=1, wdtype=0)
    need = lib.actcomp_layer_norm_bwd_workspace(4, 16)
    back = lambda ws=P, wsb=need, **k: lib.actcomp_layer_norm_bwd(  # noqa: E731
        ctypes.byref(_lib.LnBwdArgs(**{**bw, **k})), ws, wsb, None)
    assert need > 0 and lib.actcomp_layer_norm_bwd_workspace(0, 16) == 0
    assert back(rows=0) == _lib.ACT_OK
    assert back(ws=None) == _lib.ACT_E_WORKSPACE and back(wsb=need - 1) == _lib.ACT_E_WORKSPACE
    for bad in (dict(dy=None), dict(dh=P, lddh=16), dict(dr=P, lddr=4), dict(dtype=-1)):
        assert back(**bad) == _lib.ACT_E_INVALID, bad


def test_cpu_tensors_are_refused():
    import actcomp

    x = torch.zeros(2, 8)
    with pytest.raises(ValueError):
        actcomp.dropout(x, 0.1, 0)
    with pytest.raises(ValueError):
        actcomp.layer_norm(x)


# ---------------------------------------------------------------- dropout
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 8), (64, 257), (33, 1024), (2, 5000), (700, 24)])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 1.0])
def test_dropout_matches_the_generator(dtype, rows, cols, p):
    import actcomp

    x = data(rows, cols, dtype, rows + cols).cuda()
    seed, off = 0x9ABCDEF012345678, (1 << 33) + 5
    y = actcomp.dropout(x, p, seed, off)
    keep = keep_mask(rows, cols, p, seed, off).cuda()
    assert torch.equal(y != 0, keep & (x != 0))
    close(y, torch.where(keep, x.double() * held_scale(p), 0.0), U[dtype] + 2 * E, 0.0)
    assert torch.equal(actcomp.dropout_backward(x, p, seed, off), y)


@pytest.mark.gpu
def test_dropout_strides_shards_streams_and_seed_tensors():
    import actcomp

    wide = data(96, 512, torch.bfloat16, 1).cuda()
    whole = actcomp.dropout(wide[:, :200], 0.3, 7)
    assert torch.equal(whole, actcomp.dropout(wide[:, :200].contiguous(), 0.3, 7))
    assert torch.equal(actcomp.dropout(wide[:, 3:203], 0.3, 7), actcomp.dropout(wide[:, 3:203].contiguous(), 0.3, 7))
    assert torch.equal(actcomp.dropout(wide.t(), 0.3, 7), actcomp.dropout(wide.t().contiguous(), 0.3, 7))
    assert torch.equal(actcomp.dropout(wide[::2], 0.3, 7), actcomp.dropout(wide[::2].contiguous(), 0.3, 7))
    # a shard draws its part of the whole's mask, and leading dimensions are rows
    assert torch.equal(actcomp.dropout(wide[40:, :200], 0.3, 7, row_offset=40), whole[40:])
    assert torch.equal(actcomp.dropout(wide.view(4, 24, 512), 0.3, 7).view(96, 512), actcomp.dropout(wide, 0.3, 7))
    st = torch.tensor([7], dtype=torch.int64, device="cuda")
    assert torch.equal(actcomp.dropout(wide[:, :200], 0.3, st), whole)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = actcomp.dropout(wide[:, :200], 0.3, 7)
    side.synchronize()
    assert torch.equal(y, whole)
    z = wide.clone()
    assert actcomp.dropout(z, 0.3, 7, out=z) is z and torch.equal(z, actcomp.dropout(wide, 0.3, 7))
    assert not torch.equal(actcomp.dropout(wide, 0.3, 8), z)
    assert actcomp.dropout(wide[:0], 0.3, 7).shape == (0, 512)
    # dropped values are 0 whatever they held
    bad = torch.full((4, 64), float("nan"), device="cuda")
    keep = keep_mask(4, 64, 0.5, 3).cuda()
    y = actcomp.dropout(bad, 0.5, 3)
    assert torch.equal(y.isnan(), keep) and bool((y[~keep] == 0).all())


@pytest.mark.gpu
def test_dropout_keeps_the_stated_share():
    """2^22 values at p = 0.1: the kept share is binomial, six standard deviations."""
    import actcomp

    n = 1 << 22
    y = actcomp.dropout(torch.ones(1024, n // 1024, device="cuda"), 0.1, 12345)
    q = 1 - round(0.1 * 65536) / 65536
    kept = float((y != 0).double().sum())
    assert abs(kept - n * q) < 6 * (n * q * (1 - q)) ** 0.5


# ---------------------------------------------------------------- layer norm forward
SHAPES = [(1, 1), (3, 5), (9, 64), (4, 257), (2, 1000), (5, 1024), (3, 2048), (7, 4096), (2, 4100), (300, 1032),
          (3, 11008), (2, 16384), (2, 16385), (3, 20000), (1300, 4096), (900, 4095), (600, 16383), (4000, 130)]


def bound_rows(x, rstd):
    """Largest normalised magnitude of each row, at least 1."""
    return ((x.abs().amax(-1) * 2) * rstd).clamp_min(1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_layer_norm_forward(dtype, rows, cols):
    import actcomp

    x = data(rows, cols, dtype, rows * cols, 2.0)
    wide = (rows + cols) % 2 == 1
    wt = torch.float32 if wide else dtype
    g = torch.Generator().manual_seed(5)
    w, b = torch.randn(cols, generator=g).to(wt), torch.randn(cols, generator=g).to(wt)
    y, mean, rstd = actcomp.layer_norm(x.cuda(), w.cuda(), b.cuda(), 1e-5)
    ry, rm, rr = ln64(x.double(), w.double(), b.double(), 1e-5)
    assert y.dtype == dtype and mean.dtype == rstd.dtype == torch.float32
    mag = x.double().abs().amax(-1)
    close(mean, rm, E, ROW * E * mag)
    # d rstd / rstd = d var / (2 (var + eps)); var's error: ROW units of (2 mag)^2
    close(rstd, rr, 8 * E, ROW * E * rr ** 3 * (2 * mag) ** 2)
    k = bound_rows(x.double(), rr)
    slack = (ROW * E * k * (1 + k * k))[:, None] * w.double().abs() + 4 * E * b.double().abs()
    close(y, ry, U[dtype] + 2 * E, slack)
    if cols > 4:  # without weight and bias
        y, _, _ = actcomp.layer_norm(x.cuda())
        close(y, ln64(x.double(), None, None, 1e-5)[0], U[dtype] + 2 * E, (ROW * E * k * (1 + k * k))[:, None])


@pytest.mark.gpu
def test_layer_norm_constant_and_nonfinite_rows():
    import actcomp

    x = torch.full((4, 4096), 3.0, device="cuda")
    x[1] = torch.randn(4096, device="cuda")
    x[2, 17] = float("inf")
    x[3, 99] = float("nan")
    y, mean, rstd = actcomp.layer_norm(x, None, torch.full((4096,), 0.25, device="cuda"))
    assert bool((y[0] == 0.25).all()) and float(mean[0]) == 3.0  # no variance: the bias alone
    assert torch.isfinite(y[1]).all() and y[2].isnan().any() and y[3].isnan().all()
    # a large mean does not cancel: values 4096 + {0, 1}
    z = 4096 + (torch.arange(2048, device="cuda") % 2).float().repeat(2, 1)
    y, mean, rstd = actcomp.layer_norm(z)
    assert torch.allclose(mean.double(), torch.full((2,), 4096.5, dtype=torch.float64, device="cuda"), atol=1e-3)
    assert torch.allclose(rstd.double(), torch.full((2,), 1 / (0.25 + 1e-5) ** 0.5, dtype=torch.float64,
                                                    device="cuda"), rtol=1e-6)


@pytest.mark.gpu
def test_layer_norm_strides_and_empty():
    import actcomp

    wide = data(64, 4096, torch.bfloat16, 3).cuda()
    w = data(1, 2048, torch.bfloat16, 4).cuda()[0]
    for v in (wide[:, 1024:3072], wide[:, 3:2051], wide[::3, :2048]):
        a, c = actcomp.layer_norm(v, w), actcomp.layer_norm(v.contiguous(), w)
        for s, t in zip(a, c):
            close(s, t, 2 * U[s.dtype], 64 * E)  # another access path may sum in another order
    y, mean, rstd = actcomp.layer_norm(wide.view(4, 16, 4096))
    assert y.shape == (4, 16, 4096) and mean.shape == rstd.shape == (4, 16)
    y, mean, _ = actcomp.layer_norm(wide[:0])
    assert y.shape == (0, 4096) and mean.shape == (0,)
    dx, dw, db = actcomp.layer_norm_backward(wide[:0], wide[:0], data(1, 4096, torch.bfloat16, 5).cuda()[0], mean, mean)
    assert dx.shape == (0, 4096) and not dw.any() and not db.any()


# ---------------------------------------------------------------- layer norm backward
def check_backward(dtype, rows, cols, wide, fused, p=0.25, with_dh=True, view=None):
    import actcomp

    x = data(rows, cols, dtype, 3 * rows + cols, 2.0)
    dy = data(rows, cols, dtype, 5 * rows + cols)
    dh = data(rows, cols, dtype, 7 * rows + cols) if with_dh else None
    w = torch.randn(cols, generator=torch.Generator().manual_seed(9)).to(torch.float32 if wide else dtype)
    _, m, r = ln64(x.double(), None, None, 1e-5)
    mean, rstd = m.float(), r.float()
    put = (lambda t: t.cuda()) if view is None else (lambda t: view(t.cuda()))
    if fused:
        dx, dr, dw, db = actcomp.dropout_add_layer_norm_backward(
            put(dy), put(x), w.cuda(), mean.cuda(), rstd.cuda(), p, 77, 11, dh=None if dh is None else put(dh))
    else:
        dr, dw, db = actcomp.layer_norm_backward(put(dy), put(x), w.cuda(), mean.cuda(), rstd.cuda())
    rx, terms, xh = ln_bwd64(dy.double(), x.double(), w.double(), mean.double(), rstd.double())
    if fused and dh is not None:
        rx = rx + dh.double()
    g = (dy.double() * w.double()).abs().amax(1)
    k = xh.abs().amax(1)
    slack = (ROW * E * (rstd.double() * g * (1 + k * k) * 4) + 4 * E * (4.0 if dh is not None else 0.0))[:, None]
    close(dr, rx, U[dtype] + 2 * E, slack)
    wu = U[w.dtype]
    n = (rows + 64) * E
    # a term's own error: dy xh with xh within a few units of (|x| + |mean|) rstd
    own = (dy.double().abs() * ((x.double().abs() + mean.double().abs()[:, None]) * rstd.double()[:, None])).sum(0)
    close(dw, terms.sum(0), wu, n * terms.abs().sum(0) + 4 * E * own)
    close(db, dy.double().sum(0), wu, n * dy.double().abs().sum(0))
    if fused:
        keep = keep_mask(rows, cols, p, 77, 11)
        close(dx, torch.where(keep, rx * held_scale(p), 0.0), U[dtype] + 4 * E, slack * held_scale(p))
        assert torch.equal(dx.cpu() != 0, keep & (dx.cpu() != 0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", SHAPES + [(1500, 40), (777, 1001), (1200, 2056), (400, 11008), (330, 13002),
                                                  (320, 16384)])
def test_layer_norm_backward(dtype, rows, cols):
    check_backward(dtype, rows, cols, wide=(rows + cols) % 2 == 0, fused=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 5), (9, 64), (300, 1032), (2, 1001), (7, 4096), (3, 11008),
                                       (2, 16385), (3, 20000), (520, 5120), (320, 9001), (310, 9600),
                                       (320, 16384), (3000, 33), (1300, 515)])
def test_branch_backward(dtype, rows, cols):
    check_backward(dtype, rows, cols, wide=rows % 2 == 0, fused=True, with_dh=cols != 64)


@pytest.mark.gpu
def test_backward_strided_inputs():
    pad = lambda off: (lambda t: torch.nn.functional.pad(t, (off, 8 - off))[:, off:off + t.shape[1]])  # noqa: E731
    check_backward(torch.bfloat16, 37, 2048, True, True, view=pad(0))
    check_backward(torch.bfloat16, 37, 2048, True, True, view=pad(3))


@pytest.mark.gpu
def test_backward_without_weight_and_repeatable():
    import actcomp

    x, dy = data(3000, 512, torch.bfloat16, 1).cuda(), data(3000, 512, torch.bfloat16, 2).cuda()
    w = torch.ones(512, dtype=torch.bfloat16, device="cuda")
    _, mean, rstd = actcomp.layer_norm(x)
    dx, dw, db = actcomp.layer_norm_backward(dy, x, None, mean, rstd)
    dx1, dw1, db1 = actcomp.layer_norm_backward(dy, x, w, mean, rstd)
    assert dw is None and torch.equal(dx, dx1) and torch.equal(db, db1)
    assert actcomp.layer_norm_backward(dy, x, w, mean, rstd, bias_grad=False)[2] is None
    for _ in range(3):  # fixed order of the sums
        again = actcomp.layer_norm_backward(dy, x, w, mean, rstd)
        assert all(torch.equal(s, t) for s, t in zip(again, (dx1, dw1, db1)))


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [24, 1100])
def test_gradients_against_differences(cols):
    """d sum(dy * y) / d(input, weight, bias) of the whole branch by central
    differences in float64 at a sample of places: step 1e-4, truncation about
    1e-8 of the third derivative, float64 rounding 1e-12 / 1e-4."""
    import actcomp

    rows, p, seed = 4, 0.3, 99
    x, res, dy, dh = (data(rows, cols, torch.float32, s).double() for s in (1, 2, 3, 4))
    w, b = data(1, cols, torch.float32, 5)[0].double(), data(1, cols, torch.float32, 6)[0].double()
    keep = keep_mask(rows, cols, p, seed)

    def loss(x, res, w, b):
        h = res + torch.where(keep, x * held_scale(p), 0.0)
        return (ln64(h, w, b, 1e-5)[0] * dy).sum() + (h * dh).sum()

    f = lambda t: t.float().cuda()  # noqa: E731
    y, h, mean, rstd = actcomp.dropout_add_layer_norm(f(x), f(res), f(w), f(b), p, seed)
    grads = actcomp.dropout_add_layer_norm_backward(f(dy), h, f(w), mean, rstd, p, seed, dh=f(dh))
    args = [x, res, w, b]
    rng = np.random.default_rng(0)
    for i, got in enumerate(grads):
        flat = args[i].reshape(-1)
        for j in rng.integers(0, flat.numel(), 40):
            old, d = float(flat[j]), []
            for s in (1e-4, -1e-4):
                flat[j] = old + s
                d.append(float(loss(*args)))
            flat[j] = old
            want = (d[0] - d[1]) / 2e-4
            assert abs(float(got.reshape(-1)[j]) - want) <= 2e-5 * (1 + abs(want)), (i, j)


# ---------------------------------------------------------------- the fused forward
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 5), (9, 64), (300, 1032), (2, 1001), (7, 4096), (3, 11008),
                                       (2, 16385), (3, 20000), (700, 4097), (640, 9001), (620, 16384), (5000, 19)])
def test_branch_forward(dtype, rows, cols):
    import actcomp

    x, res = data(rows, cols, dtype, 1, 2.0), data(rows, cols, dtype, 2)
    w, b = data(1, cols, dtype, 3)[0], data(1, cols, dtype, 4)[0]
    p, seed, off = 0.2, 31, (1 << 32) - 2  # the row counter passes 32 bits
    y, h, mean, rstd = actcomp.dropout_add_layer_norm(x.cuda(), res.cuda(), w.cuda(), b.cuda(), p, seed, off)
    keep = keep_mask(rows, cols, p, seed, off)
    rh = res.double() + torch.where(keep, x.double() * held_scale(p), 0.0)
    ry, rm, rr = ln64(rh, w.double(), b.double(), 1e-5)
    mag = (rh.abs() + x.double().abs() * 2).amax(-1)
    close(h, rh, U[dtype] + 2 * E, 2 * E * mag[:, None])
    close(mean, rm, E, ROW * E * mag)
    close(rstd, rr, 8 * E, ROW * E * rr ** 3 * (2 * mag) ** 2)
    k = (2 * mag * rr).clamp_min(1.0)
    close(y, ry, U[dtype] + 2 * E,
          (ROW * E * k * (1 + k * k))[:, None] * w.double().abs() + 4 * E * b.double().abs())


@pytest.mark.gpu
def test_refusals():
    import actcomp as A

    x = torch.randn(4, 64, device="cuda")
    w, m = torch.ones(64, device="cuda"), torch.zeros(4, device="cuda")
    for bad in (lambda: A.dropout(x, 1.5, 0), lambda: A.dropout(x, 0.5, -1), lambda: A.dropout(x, 0.5, 1 << 64),
                lambda: A.dropout(x, 0.5, 0, -3), lambda: A.dropout(x, 0.5, torch.zeros(1, device="cuda")),
                lambda: A.dropout(x, 0.5, 0, out=x.half()), lambda: A.dropout(x, float("nan"), 0),
                lambda: A.layer_norm(x, w[:63]), lambda: A.layer_norm(x, eps=-1.0), lambda: A.layer_norm(x[:, :0]),
                lambda: A.dropout_add_layer_norm(x, x[:3], w, None, 0.1, 0),
                lambda: A.layer_norm_backward(x[:3], x, w, m, m), lambda: A.layer_norm_backward(x, x, w, m[:3], m),
                lambda: A.layer_norm_backward(x, x, w, m.double(), m),
                lambda: A.dropout_add_layer_norm_backward(x, x, w, m, m, 0.1, 0, dh=x.half())):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: A.dropout(x.double(), 0.5, 0), lambda: A.layer_norm(x, w.half()),
                lambda: A.layer_norm(x.half(), w, w.half())):
        with pytest.raises(TypeError):
            bad()


# ---------------------------------------------------------------- custom ops and the example
def test_custom_ops_have_fake_forms():
    from torch._subclasses.fake_tensor import FakeTensorMode

    import actcomp.ops  # noqa: F401

    with FakeTensorMode():
        x, w, seed = torch.empty(6, 40), torch.empty(40), torch.empty(1, dtype=torch.int64)
        o = torch.ops.actcomp
        assert o.dropout(x, 0.1, seed, 0).shape == (6, 40)
        y, m, r = o.layer_norm(x, w, w, 1e-5)
        assert m.shape == r.shape == (6,) and m.dtype == torch.float32
        assert [t.shape for t in o.layer_norm_backward(x, x, w, m, r)] == [(6, 40), (40,), (40,)]
        assert len(o.dropout_add_layer_norm(x, x, w, w, 0.1, seed, 0, 1e-5)) == 4
        assert o.dropout_add_layer_norm_backward(x, x, w, m, r, 0.1, seed, 0, None)[2].shape == (40,)
        c, s = o.mx4_quantize(x, True)
        assert c.shape == (40, 16) and s.shape == (512,)
        c, s = o.mx4_quantize(x, False)
        assert o.mx4_linear(x, c, s, torch.bfloat16).shape == (6, 6)


@pytest.mark.gpu
def test_custom_ops_run_the_operators():
    import actcomp
    import actcomp.ops  # noqa: F401
    from actcomp import mx4

    o = torch.ops.actcomp
    x, w = data(64, 256, torch.bfloat16, 1).cuda(), data(1, 256, torch.bfloat16, 2).cuda()[0]
    seed = torch.tensor([5], device="cuda")
    assert torch.equal(o.dropout(x, 0.2, seed, 3), actcomp.dropout(x, 0.2, 5, 3))
    for a, b in zip(o.dropout_add_layer_norm(x, x, w, w, 0.2, seed, 0, 1e-5),
                    actcomp.dropout_add_layer_norm(x, x, w, w, 0.2, 5)):
        assert torch.equal(a, b)
    y, m, r = o.layer_norm(x, w, w, 1e-5)
    for a, b in zip(o.dropout_add_layer_norm_backward(y, x, w, m, r, 0.2, seed, 0, x),
                    actcomp.dropout_add_layer_norm_backward(y, x, w, m, r, 0.2, 5, dh=x)):
        assert torch.equal(a, b)
    c, s = o.mx4_quantize(x, False)
    assert torch.equal(o.mx4_linear(x, c, s, torch.bfloat16), mx4.linear(x, mx4.quantize(x)))


@pytest.mark.gpu
def test_captured_graph_draws_new_masks_from_a_seed_tensor():
    import actcomp

    x, seed = data(32, 512, torch.bfloat16, 1).cuda(), torch.tensor([7], device="cuda")
    actcomp.dropout(x, 0.3, seed)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = actcomp.dropout(x, 0.3, seed)
    for s in (7, 8):
        seed.fill_(s)
        g.replay()
        assert torch.equal(y, actcomp.dropout(x, 0.3, s))


@pytest.mark.gpu
def test_residual_step_example():
    """Against the float32 step.  e2m1 has one mantissa bit: rounding to it is off
    by at most 1/4 of a value above a block's smallest step, saturation by 1/4, and
    the step itself bounds small values: under 0.15 of a block's norm for normal
    values, so under 0.25 for a product of two such operands (errors add in squares:
    0.15 sqrt 2 = 0.21).  What needs no 4-bit gradient input is far closer."""
    import importlib.util

    path = os.path.join(ROOT, "triton-kernel-test_b200", "examples", "residual_step.py")
    spec = importlib.util.spec_from_file_location("residual_step", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    r = m.main(tokens=512, channels=256, out=384)
    for rep in r.values():
        assert all(v < 0.25 for k, v in rep.items() if k != "bytes"), rep
    assert r[True]["bytes"] < 0.75 * r[False]["bytes"]
