"""Layer norm with a bias and no weight: the bias's gradient is in the bias's
dtype, a float32 one unrounded.  Tolerance: a sum of n float32 terms in any
order is within n 2^-24 sum|terms|, then one rounding to the output's type."""
import pytest
import torch

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
pytestmark = pytest.mark.gpu


def inputs(rows, cols, dtype):
    g = torch.Generator().manual_seed(rows + cols)
    return [torch.randn(rows, cols, generator=g).to(dtype).cuda() for _ in range(2)]


@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(700, 96), (65, 1003), (3, 20000)])
def test_bias_gradient_is_in_the_bias_dtype(dtype, rows, cols, fused):
    import actcomp

    x, dy = inputs(rows, cols, dtype)
    for bt in {dtype, torch.float32}:
        b = torch.randn(cols, generator=torch.Generator().manual_seed(1)).to(bt).cuda()
        if fused:
            _, h, mean, rstd = actcomp.dropout_add_layer_norm(x, dy, None, b, 0.25, 3)
            dw, db = actcomp.dropout_add_layer_norm_backward(dy, h, None, mean, rstd, 0.25, 3, bias_dtype=bt)[2:]
        else:
            _, mean, rstd = actcomp.layer_norm(x, None, b)
            dw, db = actcomp.layer_norm_backward(dy, x, None, mean, rstd, bias_dtype=bt)[1:]
        assert dw is None and db.dtype == bt and db.shape == (cols,)
        ref, mag = dy.double().sum(0), dy.double().abs().sum(0)
        assert ((db.double() - ref).abs() <= U[bt] * ref.abs() + (rows + 64) * 2.0 ** -24 * mag).all()


def test_bias_dtype_refusals():
    import actcomp

    x, dy = inputs(8, 64, torch.bfloat16)
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    _, mean, rstd = actcomp.layer_norm(x)
    for weight, bt in ((None, torch.float16), (None, torch.float64), (w, torch.float32)):
        with pytest.raises(TypeError):
            actcomp.layer_norm_backward(dy, x, weight, mean, rstd, bias_dtype=bt)
    assert actcomp.layer_norm_backward(dy, x, w, mean, rstd, bias_dtype=torch.bfloat16)[2].dtype == torch.bfloat16
    assert actcomp.layer_norm_backward(dy, x, None, mean, rstd)[2].dtype == torch.bfloat16  # as the activation's
