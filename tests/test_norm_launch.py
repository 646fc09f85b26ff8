"""Launch shapes of the layer norm kernels, seen through the workspace: the
backward pass keeps one partial weight gradient (dweight and dbias, float32) per
CTA of its grid, and a grid of persistent CTAs is no larger than what is
resident."""
import pytest
import torch


def _sms():
    return torch.cuda.get_device_properties(0).multi_processor_count if torch.cuda.is_available() else 148


@pytest.mark.parametrize("cols,per_sm", [(4096, 2), (5120, 2), (6144, 1), (8192, 1), (8200, 1), (8704, 1), (9216, 1),
                                         (9300, 1)])
def test_backward_grid_is_what_an_sm_holds(cols, per_sm):
    """Rows of 4097 to 5120 values have a form of up to 320 threads that fits an SM
    twice; past that, and so past 8192 where a thread holds four segments, a
    kernel of up to 512 threads at 128 registers fits once."""
    from actcomp import _lib

    need = _lib.load().actcomp_layer_norm_bwd_workspace(1 << 20, cols)
    parts = _sms() * per_sm
    assert need == (parts * 2 * cols * 4 + 255) // 256 * 256
