"""The norms, the 8-bit linear layers and the cross entropy together, as
examples/language_step.py runs them.

Tolerance of the gradients against float32 autograd: a value of a block in e4m3 is
within 2^-4 relative, 2^-4 / sqrt(3) = 3.6 % in the mean square, so a product of two
such operands 5.1 %; the longest way through the step passes six products (both layers
forward, their four gradients): 5.1 % sqrt(6) = 12.5 %, plus bf16's roundings (each 2^-8)
and what the errors share, 20 %.  The loss is a mean over hundreds of tokens of values near
log(vocabulary) that the errors move by part of a logit: 2 %."""
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    from conftest import PKG

    sys.path.insert(0, os.path.join(PKG, "examples"))
    import language_step

    return language_step


def test_gradients(example):
    report = example.main()
    assert report.pop("loss") < 0.02, report
    assert set(report) == {"d" + n for n in example.NAMES} and max(report.values()) < 0.2, report


def test_captured_step_equals_the_eager_one(example):
    args = example.inputs(tokens=130, channels=264, hidden=520, vocab=1003)
    loss, grads = example.step(*args)
    want = [t.clone() for t in (loss, *grads)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, grads = example.step(*args)
    first, other = args[0].clone(), example.inputs(tokens=130, channels=264, hidden=520, vocab=1003)[1]
    for x in (other, first):
        args[0].copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        again, g = example.step(*args)
        assert all(torch.equal(a, b) for a, b in zip((loss, *grads), (again, *g)))
    assert all(torch.equal(a, b) for a, b in zip((loss, *grads), want))


def test_two_streams_at_once(example):
    """Two steps in flight beside each other, and served tokens beside them."""
    from actcomp import fp8

    sets = [example.inputs(tokens=t, channels=512, hidden=1408, vocab=2003) for t in (300, 77)]
    want = [example.step(*a) for a in sets]
    x, r, n1, w1 = (t[:9] if i < 2 else t for i, t in enumerate(sets[0][:4]))
    q1 = fp8.quantize_weight(w1)
    y, h = example.serve(x, r, n1, q1)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(5):
        got = [None] * 3
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = example.step(*sets[i]) if i < 2 else example.serve(x, r, n1, q1)
        torch.cuda.synchronize()
        for (loss, grads), (l2, g2) in zip(got[:2], want):
            assert torch.equal(loss, l2) and all(torch.equal(a, b) for a, b in zip(grads, g2))
        assert torch.equal(got[2][0], y) and torch.equal(got[2][1], h)


def test_served_tokens(example):
    """One token to more than the few-token kernel takes: each token's result is the same
    whichever batch it came in, up to the order of the sums."""
    x, r, n1, w1 = example.inputs(tokens=300)[:4]
    from actcomp import fp8

    q1 = fp8.quantize_weight(w1)
    ref = example.serve(x, r, n1, q1)[0].float()
    h = (x.float() + r.float())
    z = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-5) * n1.float()
    plain = z @ w1.float().t()
    assert ((ref - plain).norm() / plain.norm()) < 0.08  # two operands of 3.6 % each, and bf16
    for n in (1, 2, 16, 17, 128, 129):
        y = example.serve(x[:n], r[:n], n1, q1)[0].float()
        assert ((y - ref[:n]).abs() <= 2.0 ** -7 * ref[:n].abs() + 1e-3 * ref.abs().max()).all()
