"""Captured graphs in which the operators' launches, which carry programmatic
dependence on the kernel before them, follow something else: a copy or a fill, another
stream's work through an event, nothing at all; and two graphs in turn."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def operands():
    import actcomp
    from actcomp import fp8

    g = torch.Generator(device="cuda").manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()  # noqa: E731
    x, w, head = r(300, 256), r(520, 256), r(700, 256)
    t = torch.randint(0, 700, (300,), generator=g, device="cuda")
    wq = fp8.quantize_weight(w)
    q, few = fp8.quantize(x), fp8.quantize(x[:9])
    return {"product": lambda: fp8.matmul(q, wq), "few rows": lambda: fp8.matmul(few, wq),
            "loss": lambda: actcomp.linear_cross_entropy(x, head, t)[0],
            "gradient": lambda: actcomp.linear_cross_entropy_backward(torch.ones(300, device="cuda"), x, head, t,
                                                                      torch.full((300,), 9.0, device="cuda"))[1],
            "norm": lambda: fp8.dequantize(fp8.rms_norm(x)[0])}, x


@pytest.mark.parametrize("name", ["product", "few rows", "loss", "gradient", "norm"])
def test_what_comes_before(name):
    calls, x = operands()
    call = calls[name]
    want = call()
    side, scratch, other = torch.cuda.Stream(), torch.empty(1 << 20, device="cuda"), torch.empty(1 << 20, device="cuda")

    def nothing():
        return call()

    def fill():
        scratch.zero_()
        return call()

    def copy():
        scratch.copy_(other)
        return call()

    def forked():
        here = torch.cuda.current_stream()
        scratch.add_(1)
        side.wait_stream(here)
        with torch.cuda.stream(side):
            out = call()
        scratch.mul_(2)
        here.wait_stream(side)
        return out + call() * 0

    def joined():
        here = torch.cuda.current_stream()
        side.wait_stream(here)
        with torch.cuda.stream(side):
            other.add_(1)
        scratch.add_(1)
        here.wait_stream(side)
        return call()

    graphs = []
    for f in (nothing, fill, copy, forked, joined):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = f()
        graphs.append((graph, out, f.__name__))
    for _ in range(2):
        for graph, out, _ in graphs:
            out.fill_(7)
            graph.replay()
        torch.cuda.synchronize()
        for _, out, what in graphs:
            assert torch.equal(out, want), what


def test_weight_written_just_before():
    """A weight that the kernels before have just written, over and over."""
    from actcomp import fp8

    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(4, 4096, generator=g, device="cuda").bfloat16()
    ws = [torch.randn(4096, 4096, generator=g, device="cuda").bfloat16() for _ in range(3)]
    want = [fp8.linear(x, fp8.quantize_weight(w)) for w in ws]
    torch.cuda.synchronize()
    w = torch.empty_like(ws[0])
    got = []
    for i in range(12):
        w.copy_(ws[i % 3])
        got.append(fp8.matmul(fp8.quantize(x), fp8.quantize_weight(w)))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i % 3]) for i, y in enumerate(got))
