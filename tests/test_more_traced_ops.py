"""Traced forms of the root-mean-square norm, the 8-bit linear layer and the cross
entropy: the fake results have the real ones' shapes and types, and the ops give what the
functions give."""
import pytest
import torch


def calls(dev):
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g).bfloat16().to(dev)  # noqa: E731
    x, w, head = r(3, 11, 72), r(72), r(200, 72)
    t = torch.randint(0, 200, (3, 11), generator=g).to(dev)
    rstd = torch.rand(3, 11, generator=g).to(dev)
    o = torch.ops.actcomp
    yield "rms", lambda: o.rms_norm(x, w, 1e-5)
    yield "add", lambda: o.add_rms_norm(x, x, None, 1e-5)
    yield "bwd", lambda: o.rms_norm_backward(x, x, w.float(), rstd, None)
    yield "bwd without", lambda: o.rms_norm_backward(x, x, None, rstd, x)
    for transpose, tiles in ((False, False), (True, False), (False, True)):
        yield f"quantize {transpose} {tiles}", lambda: o.fp8_quantize(x, transpose, tiles, "e4m3")
    c, s = torch.empty(200, 80, dtype=torch.uint8, device=dev), torch.empty(2, dtype=torch.uint8, device=dev)
    yield "linear", lambda: o.fp8_linear(x, c.zero_(), s.fill_(127), "e4m3", torch.float32)
    yield "xent", lambda: o.linear_cross_entropy(x, head, t, -100)
    yield "xent bwd", lambda: o.linear_cross_entropy_backward(rstd, x, head, t, rstd + 9, None, -100, 0)


def meta(v):
    return [(tuple(t.shape), t.dtype) for t in ((v,) if torch.is_tensor(v) else v)]


def fake():
    from torch._subclasses.fake_tensor import FakeTensorMode

    import actcomp.ops  # noqa: F401

    with FakeTensorMode(allow_non_fake_inputs=True):
        return {n: meta(f()) for n, f in calls("cpu")}


def test_fake_forms():
    out = fake()
    assert out["rms"] == [((3, 11, 72), torch.bfloat16), ((3, 11), torch.float32)]
    assert out["quantize True False"] == [((33, 80), torch.uint8), ((128,), torch.uint8)]
    assert out["bwd without"][1] == ((0,), torch.bfloat16) and out["xent bwd"][1] == ((200, 72), torch.bfloat16)


@pytest.mark.gpu
def test_real_forms_are_as_the_fake_ones():
    import actcomp
    import actcomp.ops  # noqa: F401

    want = fake()
    for n, f in calls("cuda"):
        assert meta(f()) == want[n], n
    g = torch.Generator(device="cuda").manual_seed(2)
    x, w = torch.randn(9, 64, generator=g, device="cuda").half(), torch.randn(30, 64, generator=g, device="cuda").half()
    t = torch.arange(9, device="cuda")
    assert all(torch.equal(a, b) for a, b in zip(torch.ops.actcomp.linear_cross_entropy(x, w, t, -100),
                                                 actcomp.linear_cross_entropy(x, w, t)))
    q = actcomp.fp8.quantize_weight(w)
    assert torch.equal(torch.ops.actcomp.fp8_linear(x, q.codes, q.scales, "e4m3", x.dtype), actcomp.fp8.linear(x, q))
