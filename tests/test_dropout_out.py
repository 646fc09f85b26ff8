"""Dropout into a tensor that lies over other parts of its input."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(2, 8), (40, 513), (3000, 1024)])
def test_out_over_other_parts_of_the_input(dtype, rows, cols):
    import actcomp

    g = torch.Generator().manual_seed(rows)
    n = rows * cols
    src = torch.randn(2 * n + 16, generator=g).to(dtype)
    views = {  # x and out of one buffer
        "a row back": lambda b: (b[cols:cols + n].view(rows, cols), b[:n].view(rows, cols)),
        "a row on": lambda b: (b[:n].view(rows, cols), b[cols:cols + n].view(rows, cols)),
        "one value on": lambda b: (b[:n].view(rows, cols), b[1:1 + n].view(rows, cols)),
        "strided": lambda b: (b[:2 * n].view(rows, 2 * cols)[:, :cols], b[:n].view(rows, cols)),
        "transposed": lambda b: (b[:n].view(cols, rows).t(), b[:n].view(rows, cols)),
        "itself": lambda b: (b[:n].view(rows, cols), b[:n].view(rows, cols)),
        "apart": lambda b: (b[:n].view(rows, cols), b[n:2 * n].view(rows, cols)),
    }
    for name, view in views.items():
        x, out = view(src.cuda())
        want = actcomp.dropout(x.contiguous().clone(), 0.3, 5, 7)
        got = actcomp.dropout(x, 0.3, 5, 7, out=out)
        assert got.data_ptr() == out.data_ptr() and torch.equal(out, want), name
