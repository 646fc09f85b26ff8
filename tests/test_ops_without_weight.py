"""The traced forms of layer norm without a weight: what the forward op takes,
the backward op takes too (the weight's gradient is then an empty tensor)."""
import pytest
import torch


def test_fake_forms():
    from torch._subclasses.fake_tensor import FakeTensorMode

    import actcomp.ops  # noqa: F401

    with FakeTensorMode():
        o = torch.ops.actcomp
        x, b = torch.empty(6, 40, dtype=torch.bfloat16), torch.empty(40)
        seed = torch.empty(1, dtype=torch.int64)
        y, m, r = o.layer_norm(x, None, b, 1e-5)
        for out in (o.layer_norm_backward(x, x, None, m, r, torch.float32),
                    o.dropout_add_layer_norm_backward(x, x, None, m, r, 0.1, seed, 0, None, torch.float32)[1:]):
            assert [t.shape for t in out] == [(6, 40), (0,), (40,)]
            assert out[2].dtype == torch.float32
        assert o.layer_norm_backward(x, x, None, m, r)[2].dtype == torch.bfloat16


@pytest.mark.gpu
def test_ops_run_without_a_weight():
    import actcomp
    import actcomp.ops  # noqa: F401

    o = torch.ops.actcomp
    x, dy = (torch.randn(33, 96, generator=torch.Generator().manual_seed(i)).bfloat16().cuda() for i in (0, 1))
    seed = torch.tensor([5], device="cuda")
    y, m, r = o.layer_norm(x, None, None, 1e-5)
    got = o.layer_norm_backward(dy, x, None, m, r, torch.float32)
    want = actcomp.layer_norm_backward(dy, x, None, m, r, bias_dtype=torch.float32)
    assert torch.equal(got[0], want[0]) and got[1].numel() == 0 and torch.equal(got[2], want[2])
    got = o.dropout_add_layer_norm_backward(dy, x, None, m, r, 0.2, seed, 0, dy)
    want = actcomp.dropout_add_layer_norm_backward(dy, x, None, m, r, 0.2, 5, dh=dy)
    assert all(torch.equal(a, b) for a, b in zip((got[0], got[1], got[3]), (want[0], want[1], want[3])))
    assert got[2].numel() == 0
