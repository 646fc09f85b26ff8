"""Cross entropy of a linear layer without stored logits, against float64.

Tolerances.  u: the input type's unit roundoff.  A logit is within
ez = H 2^-23 sum|x w| (float32 accumulation, additions rounded or truncated).  An
exponential's argument is rounded twice more relative to |z|, |lse| (4 2^-24), the
hardware's exponential is within 2^-22, and a sum's terms are added in chains of at most
64 + parts: SUM = 200 units of 2^-24 and the number of partial sums bound them.  So
  lse   max ez + 2^-21 + (200 + parts) 2^-24 + 4 2^-24 max|z|,   loss twice ez
  dz    dp = p (ez + 8 2^-24 (|z| + |lse|) + 2^-21), times its factor, + u |dz| + what a
        value of fp16 may be off near 0 (2^-24 of the token's factor)
  dx    sum_v (err dz)|w| + (V 2^-23) sum_v |dz||w| + u |dx|
  dW    the same over tokens; x's scaled copy is exact in bf16, and in fp16 within 2^-24
        of the largest factor for each token."""
import ctypes
import os
import subprocess
import sys

import pytest
import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
E = 2.0 ** -24
IGNORE = -100


def make(tokens, channels, vocab, dtype, seed=0, gone=0.2, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(tokens, channels, generator=g) * spread).to(dtype)
    w = (torch.randn(vocab, channels, generator=g) / channels ** 0.5).to(dtype)
    t = torch.randint(0, vocab, (tokens,), generator=g)
    t[torch.rand(tokens, generator=g) < gone] = IGNORE
    return x, w, t


def loss64(x, w, t, ignore=IGNORE):
    z = x @ w.t()
    lse = torch.logsumexp(z, -1)
    at = z.gather(1, t.clamp(0, w.shape[0] - 1)[:, None])[:, 0]
    return torch.where(t == ignore, torch.zeros_like(lse), lse - at), lse, z


def dz64(z, lse, t, dloss, dlse, ignore=IGNORE):
    d = torch.where(t == ignore, torch.zeros_like(dloss), dloss)
    a = d if dlse is None else d + dlse
    p = (z - lse[:, None]).exp()
    hit = torch.zeros_like(z)
    live = t != ignore
    hit[live, t[live]] = 1
    return p * a[:, None] - hit * d[:, None], p, a, d


def check_forward(x, w, t, loss, lse, ignore=IGNORE):
    x, w, t = x.double().cuda(), w.double().cuda(), t.cuda()
    want, n, z = loss64(x, w, t, ignore)
    ez = x.shape[1] * 2.0 ** -23 * (x.abs() @ w.abs().t()).amax(1)
    parts = 2 * (-(-w.shape[0] // 256))
    tol = ez + 2.0 ** -21 + (200 + parts) * E + 4 * E * z.abs().amax(1)
    assert ((lse.double() - n).abs() <= tol + E * n.abs()).all(), float((lse - n).abs().max())
    assert ((loss.double() - want).abs() <= tol + ez + E * want.abs()).all(), float((loss - want).abs().max())
    assert (loss[t == ignore] == 0).all()


def check_backward(x, w, t, dloss, dlse, lse, dx, dw, ignore=IGNORE):
    u = U[x.dtype]
    x, w, t, n = x.double().cuda(), w.double().cuda(), t.cuda(), lse.double()
    dloss, dlse = dloss.double(), None if dlse is None else dlse.double()
    _, _, z = loss64(x, w, t, ignore)
    g, p, a, d = dz64(z, n, t, dloss, dlse, ignore)
    ez = x.shape[1] * 2.0 ** -23 * (x.abs() @ w.abs().t())
    big = torch.maximum(a.abs(), d.abs())
    tiny = E * big if u == 2.0 ** -11 else torch.zeros_like(big)
    err = p * a.abs()[:, None] * (ez + 8 * E * (z.abs() + n.abs()[:, None]) + 2.0 ** -21) + u * g.abs() * 1.01 \
        + 2 * tiny[:, None] + 2 * E * g.abs()
    if dx is not None:
        ref = g @ w
        tol = err @ w.abs() * 1.01 + w.shape[0] * 2.0 ** -23 * (g.abs() @ w.abs()) + u * ref.abs() * 1.01 + 1e-7 * (u < 2e-3)
        assert ((dx.double() - ref).abs() <= tol + 1e-38).all(), float((dx - ref).abs().max())
    if dw is not None:
        ref = g.t() @ x
        tol = err.t() @ x.abs() * 1.01 + x.shape[0] * 2.0 ** -23 * (g.abs().t() @ x.abs()) + u * ref.abs() * 1.01
        if u == 2.0 ** -11:  # x's scaled copy, and the result's subnormals
            tol = tol + (g != 0).double().t() @ (2 * E * big.max() * torch.ones_like(x)) + 1e-7
        assert ((dw.double() - ref).abs() <= tol + 1e-38).all(), float((dw - ref).abs().max())


# ---------------------------------------------------------------- CPU
def test_formula_against_differences():
    g = torch.Generator().manual_seed(3)
    x, w = torch.randn(4, 6, generator=g, dtype=torch.float64), torch.randn(9, 6, generator=g, dtype=torch.float64)
    t, dloss, dlse = torch.tensor([3, IGNORE, 0, 8]), *torch.randn(2, 4, generator=g, dtype=torch.float64)

    def f(x, w):
        loss, lse, _ = loss64(x, w, t)
        return (loss * dloss).sum() + (lse * dlse).sum()

    _, lse, z = loss64(x, w, t)
    dz = dz64(z, lse, t, dloss, dlse)[0]
    for v, grad in ((x, dz @ w), (w, dz.t() @ x)):
        for i in range(v.numel()):
            s = torch.zeros(v.numel(), dtype=torch.float64)
            s[i] = 1e-5
            s = s.view(v.shape)
            num = f(x + s, w) - f(x - s, w) if v is x else f(x, w + s) - f(x, w - s)
            assert abs(float(num / 2e-5 - grad.flatten()[i])) < 1e-8


def test_entry_points_validate_without_gpu():
    from actcomp import _lib

    lib = _lib.load()
    P, I, A, N = 1 << 20, _lib.ACT_E_INVALID, _lib.ACT_E_ALIGN, _lib.ACT_E_UNSUPPORTED
    base = dict(tokens=8, channels=64, vocab=500, x=P, ldx=64, weight=P, ldw=64, target=P, ignore_index=-100, loss=P, lse=P,
                dtype=1)
    need = lib.actcomp_xent_workspace(8, 500)
    assert need == 8 * 2 * 2 * 8 and lib.actcomp_xent_workspace(0, 5) == 0
    f = lambda ws=P, n=need, **k: lib.actcomp_xent(ctypes.byref(_lib.XentArgs(**{**base, **k})), ws, n, None)  # noqa: E731
    assert lib.actcomp_xent(None, P, need, None) == I and f(tokens=0) == _lib.ACT_OK
    for bad in (dict(channels=0), dict(vocab=0), dict(dtype=0), dict(x=None), dict(target=None), dict(lse=None), dict(loss=None),
                dict(ldx=63), dict(ldw=56), dict(tokens=-1)):
        assert f(**bad) == I, bad
    for bad in (dict(x=P + 8), dict(ldx=68), dict(weight=P + 2), dict(target=P + 4), dict(lse=P + 2)):
        assert f(**bad) == A, bad
    assert f(vocab=1 << 31) == N and f(n=need - 1) == _lib.ACT_E_WORKSPACE and f(ws=None) == _lib.ACT_E_WORKSPACE
    wsb = lib.actcomp_xent_bwd_workspace(8, 64, 500, 0)
    gr = dict(dloss=P, dx=P, lddx=64, dweight=P, lddw=64)
    b = lambda ws=P, n=wsb, piece=0, a={}, **k: lib.actcomp_xent_bwd(  # noqa: E731
        ctypes.byref(_lib.XentArgs(**{**base, **a})), ctypes.byref(_lib.XentGrads(**{**gr, **k})), piece, ws, n, None)
    assert wsb > 0 and lib.actcomp_xent_bwd_workspace(8, 64, 500, 256) > 0
    for bad in (dict(dloss=None), dict(dx=None, dweight=None), dict(lddx=63), dict(lddw=8), dict(piece=-1)):
        assert b(**bad) == I, bad
    assert b(dx=P + 1) == A and b(dlse=P + 2) == A and b(n=wsb - 1) == _lib.ACT_E_WORKSPACE
    assert b(ws=P + 128) == _lib.ACT_E_WORKSPACE and b(a=dict(lse=None)) == I


def test_pieces_larger_than_the_vocabulary():
    """Any piece above the vocabulary is the whole of it, up to the largest integer (in
    its own process: a division by zero ends one)."""
    code = ("from actcomp import _lib\nf = _lib.load().actcomp_xent_bwd_workspace\n"
            "for tokens, channels, vocab in ((100, 512, 16000), (1, 8, 1), (8, 64, 256)):\n"
            "    whole = f(tokens, channels, vocab, (vocab + 255) // 256 * 256)\n"
            "    for piece in (vocab + 256, 2 ** 31, 2 ** 62, 2 ** 63 - 512, 2 ** 63 - 1):\n"
            "        assert f(tokens, channels, vocab, piece) == whole > 0, (vocab, piece)\n")
    import actcomp

    root = os.path.dirname(os.path.dirname(os.path.abspath(actcomp.__file__)))
    env = dict(os.environ, PYTHONPATH=root + os.pathsep + os.environ.get("PYTHONPATH", ""))
    subprocess.run([sys.executable, "-c", code], check=True, env=env, timeout=300)


def test_struct_layouts_match_the_header():
    import os
    import subprocess
    import tempfile

    from actcomp import _lib
    from conftest import ROOT

    structs = {"actcomp_xent_args": _lib.XentArgs, "actcomp_xent_grads": _lib.XentGrads, "actcomp_fp8": _lib.Fp8Desc,
               "actcomp_rms_args": _lib.RmsArgs, "actcomp_rms_bwd_args": _lib.RmsBwdArgs}
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{os.path.join(ROOT, "include", "actcomp.h")}"',
             "int main(void){"]
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


def test_cpu_tensors_are_refused():
    import actcomp

    x, w, t = torch.zeros(2, 8).bfloat16(), torch.zeros(5, 8).bfloat16(), torch.zeros(2, dtype=torch.long)
    with pytest.raises(ValueError, match="CUDA"):
        actcomp.linear_cross_entropy(x, w, t)
    with pytest.raises(ValueError, match="CUDA"):
        actcomp.linear_cross_entropy_backward(torch.zeros(2), x, w, t, torch.zeros(2))


# ---------------------------------------------------------------- forward
SIZES = [(1, 8, 1), (1, 64, 300), (5, 100, 7), (3, 7, 33), (130, 64, 256), (257, 257, 257), (300, 512, 1000), (40, 64, 5000),
         (64, 1032, 2049), (700, 96, 129)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("tokens,channels,vocab", SIZES)
def test_forward(dtype, tokens, channels, vocab):
    import actcomp

    x, w, t = make(tokens, channels, vocab, dtype)
    loss, lse = actcomp.linear_cross_entropy(x.cuda(), w.cuda(), t.cuda())
    assert loss.dtype == lse.dtype == torch.float32
    check_forward(x, w, t, loss, lse)
    # other strides, and rows that are not 16-byte aligned
    pad = lambda v: torch.nn.functional.pad(v, (3, 2)).cuda()[:, 3:3 + channels]  # noqa: E731
    again = actcomp.linear_cross_entropy(pad(x), pad(w), t.cuda())
    assert torch.equal(again[0], loss) and torch.equal(again[1], lse)


@pytest.mark.gpu
def test_forward_large_logits_and_certain_targets():
    """Logits of several hundred, a target that has all the weight, and one that has none."""
    import actcomp

    x, w, t = make(200, 256, 3000, torch.bfloat16, gone=0, spread=60.0)
    z = x.double() @ w.double().t()
    t[:100], t[100:150] = z[:100].argmax(1), z[100:150].argmin(1)
    loss, lse = actcomp.linear_cross_entropy(x.cuda(), w.cuda(), t.cuda())
    assert torch.isfinite(loss).all() and (loss[:100] < 1e-2).any() and (loss >= -1e-3).all()
    check_forward(x, w, t, loss, lse)


@pytest.mark.gpu
def test_shapes_ignored_and_outside_targets():
    import actcomp

    x, w, t = make(24, 64, 500, torch.bfloat16, gone=0)
    t[3], t[5], t[7], t[9] = 500, -1, IGNORE, 499
    x[7] = float("nan")
    loss, lse = actcomp.linear_cross_entropy(x.cuda().view(2, 3, 4, 64), w.cuda(), t.cuda().view(2, 3, 4))
    assert loss.shape == lse.shape == (2, 3, 4)
    loss, lse = loss.flatten(), lse.flatten()
    assert loss[[3, 5]].isnan().all() and loss[7] == 0 and torch.isfinite(lse[[3, 5]]).all()
    ok = torch.ones(24, dtype=torch.bool)
    ok[[3, 5, 7]] = False
    check_forward(x[ok], w, t[ok], loss[ok.cuda()], lse[ok.cuda()])
    # a weight row of NaN or infinity shows in every loss, as in the formula
    w2 = w.clone()
    w2[300] = float("nan")
    assert actcomp.linear_cross_entropy(x.cuda(), w2.cuda(), t.cuda())[1].isnan().all()
    # another ignore_index, inside the vocabulary
    l2, _ = actcomp.linear_cross_entropy(x.cuda(), w.cuda(), t.cuda(), ignore_index=499)
    assert l2[9] == 0 and l2[7].isnan() and torch.equal(l2[10:], loss[10:])
    # one token without a leading dimension, weight rows and targets at a stride
    l3, n3 = actcomp.linear_cross_entropy(x[9].cuda(), torch.cat([w, w], 1).cuda()[:, :64], t[9].cuda())
    assert l3.shape == n3.shape == () and torch.equal(l3, loss[9]) and torch.equal(n3, lse[9])
    dx, dw = actcomp.linear_cross_entropy_backward(torch.ones((), device="cuda"), x[9].cuda(), w.cuda(), t[9].cuda(), n3)
    assert dx.shape == (64,) and dw.shape == w.shape
    wide = torch.stack([t, t + 1], 1).cuda()
    assert torch.equal(actcomp.linear_cross_entropy(x.cuda(), w.cuda(), wide[:, 0])[0][10:], loss[10:])
    # no token
    e = actcomp.linear_cross_entropy(x[:0].cuda(), w.cuda(), t[:0].cuda())
    assert e[0].shape == (0,)
    dx, dw = actcomp.linear_cross_entropy_backward(e[0], x[:0].cuda(), w.cuda(), t[:0].cuda(), e[1])
    assert dx.shape == (0, 64) and not dw.any()


@pytest.mark.gpu
def test_refusals():
    import actcomp

    x, w, t = (v.cuda() for v in make(6, 64, 500, torch.bfloat16))
    f = actcomp.linear_cross_entropy
    for bad in (lambda: f(x, w[:, :32], t), lambda: f(x, w.half(), t), lambda: f(x, w, t[:3]), lambda: f(x, w, t.int()),
                lambda: f(x, w, t.cpu()), lambda: f(x, w[:0], t), lambda: f(x, w[0], t), lambda: f(x[:, :0], w[:, :0], t)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        f(x.float(), w.float(), t)
    loss, lse = f(x, w, t)
    b = actcomp.linear_cross_entropy_backward
    for bad in (lambda: b(loss[:2], x, w, t, lse), lambda: b(loss, x, w, t, lse.double()), lambda: b(loss, x, w, t, lse, dlse=lse[:1]),
                lambda: b(loss, x, w, t, lse, x_grad=False, weight_grad=False), lambda: b(loss, x, w, t, lse, vocab_piece=-1)):
        with pytest.raises(ValueError):
            bad()


# ---------------------------------------------------------------- backward
def run_backward(dtype, tokens, channels, vocab, dlse, piece=0, seed=0, factors=1.0):
    import actcomp

    x, w, t = make(tokens, channels, vocab, dtype, seed)
    g = torch.Generator().manual_seed(seed + 1)
    dloss = (torch.rand(tokens, generator=g) + 0.2) / tokens * factors
    dl = (0.1 * torch.randn(tokens, generator=g) / tokens).cuda() if dlse else None
    loss, lse = actcomp.linear_cross_entropy(x.cuda(), w.cuda(), t.cuda())
    dx, dw = actcomp.linear_cross_entropy_backward(dloss.cuda(), x.cuda(), w.cuda(), t.cuda(), lse, dlse=dl,
                                                   vocab_piece=piece)
    check_backward(x, w, t, dloss.cuda(), dl, lse, dx, dw)
    return x, w, t, dloss.cuda(), dl, lse, dx, dw


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("tokens,channels,vocab", SIZES)
def test_backward(dtype, tokens, channels, vocab):
    import actcomp

    for dlse in (False, True):
        x, w, t, dloss, dl, lse, dx, dw = run_backward(dtype, tokens, channels, vocab, dlse)
    pad = lambda v: torch.nn.functional.pad(v, (3, 2)).cuda()[:, 3:3 + channels]  # noqa: E731
    f = actcomp.linear_cross_entropy_backward
    for xg, wg in ((True, True), (True, False), (False, True)):
        a, b = f(dloss, pad(x), pad(w), t.cuda(), lse, dlse=dl, x_grad=xg, weight_grad=wg)
        assert (torch.equal(a, dx) if xg else a is None) and (torch.equal(b, dw) if wg else b is None)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("tokens,channels,vocab,piece", [
    (40, 64, 5000, 256), (40, 64, 5000, 2304), (300, 96, 1100, 512), (2, 130, 9000, 4096), (600, 40, 2000, 300),
    (64, 257, 4400, 1), (1, 64, 70000, 0), (33, 512, 20000, 7000)])
def test_backward_in_pieces(dtype, tokens, channels, vocab, piece):
    """Pieces of the vocabulary, a last one that is shorter, and dx's contraction in parts."""
    run_backward(dtype, tokens, channels, vocab, True, piece)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("factor", [1e-7, 1e6])
def test_backward_factors_of_any_size(dtype, factor):
    """dloss far below and above what fp16 holds, and of different size from token to token."""
    import actcomp

    x, w, t = make(90, 128, 700, dtype, 5, spread=1.0)
    lse = actcomp.linear_cross_entropy(x.cuda(), w.cuda(), t.cuda())[1]
    dloss = factor * torch.exp2(torch.randint(-6, 1, (90,), generator=torch.Generator().manual_seed(1)).float()).cuda()
    if dtype == torch.float16 and factor > 1:
        dloss = dloss * 1e-3  # the gradient itself has to fit
    dx, dw = actcomp.linear_cross_entropy_backward(dloss, x.cuda(), w.cuda(), t.cuda(), lse)
    check_backward(x, w, t, dloss, None, lse, dx, dw)
    if dtype == torch.bfloat16:
        assert (dx.abs().amax(1)[t.cuda() != IGNORE] > 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(U))
def test_tokens_without_a_gradient_add_nothing(dtype):
    """Ignored tokens and tokens of weight 0 may hold NaN; all tokens may be such."""
    import actcomp

    x, w, t = make(300, 64, 700, dtype, 2, gone=0.5)
    dloss = torch.rand(300, generator=torch.Generator().manual_seed(4))
    dloss[10:60] = 0
    dead = (t == IGNORE) | (dloss == 0)
    bad = x.clone()
    bad[dead] = float("nan")
    bad[11], dloss[t == IGNORE] = float("inf"), float("nan")
    lse = actcomp.linear_cross_entropy(bad.cuda(), w.cuda(), t.cuda())[1]
    assert lse[dead.cuda()].isnan().all()
    dx, dw = actcomp.linear_cross_entropy_backward(dloss.cuda(), bad.cuda(), w.cuda(), t.cuda(), lse, vocab_piece=512)
    assert (dx[dead.cuda()] == 0).all()
    keep = ~dead
    check_backward(x[keep], w, t[keep], dloss[keep].cuda(), None, lse[keep.cuda()], dx[keep.cuda()], dw)
    dx, dw = actcomp.linear_cross_entropy_backward(dloss.cuda(), bad.cuda(), w.cuda(), torch.full_like(t, IGNORE).cuda(), lse)
    assert not dx.any() and not dw.any()
    # the normaliser's gradient alone reaches ignored tokens
    lse = actcomp.linear_cross_entropy(x.cuda(), w.cuda(), t.cuda())[1]
    one = torch.ones(300)
    dx, dw = actcomp.linear_cross_entropy_backward(one.cuda(), x.cuda(), w.cuda(), torch.full_like(t, IGNORE).cuda(), lse,
                                                   dlse=one.cuda())
    check_backward(x, w, torch.full_like(t, IGNORE), one.cuda(), one.cuda(), lse, dx, dw)
    # a target outside the vocabulary
    t2 = t.clone()
    t2[0] = 700
    dx, dw = actcomp.linear_cross_entropy_backward(one.cuda(), x.cuda(), w.cuda(), t2.cuda(), lse)
    assert dx[0].isnan().all() and not dx[1:].isnan().any() and dw.isnan().all()


# ---------------------------------------------------------------- streams and graphs
@pytest.mark.gpu
def test_repeats_other_stream_and_graph():
    import actcomp

    x, w, t = (v.cuda() for v in make(200, 128, 3000, torch.bfloat16, 1))

    def step():
        loss, lse = actcomp.linear_cross_entropy(x, w, t)
        return (loss, lse) + actcomp.linear_cross_entropy_backward(lse / 200, x, w, t, lse, dlse=loss, vocab_piece=1024)

    want = [v.clone() for v in step()]
    assert all(torch.equal(a, b) for a, b in zip(step(), want))
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
    for v in (make(200, 128, 3000, torch.bfloat16, 8)[0].cuda(), first):
        x.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_no_logits_in_memory():
    """The forward pass of 2048 tokens against 100000 allocates far less than their logits."""
    import actcomp

    x, w, t = (v.cuda() for v in make(2048, 64, 100000, torch.bfloat16, 1))
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    loss, lse = actcomp.linear_cross_entropy(x, w, t)
    assert torch.cuda.max_memory_allocated() - before < 2048 * 100000 * 2 / 16
    check_forward(x.cpu(), w.cpu(), t.cpu(), loss, lse)
