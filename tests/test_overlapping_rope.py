"""The table rotations on views whose rows overlap in memory."""

import pytest
import torch

import attnax_b200 as ax
from attnax_b200 import rope
from tests.test_overlapping_views import rows_apart, windows


@pytest.mark.parametrize("step", [1, 8, 64])
@pytest.mark.parametrize("b,h,s", [(2, 2, 8), (1, 1, 8), (1, 4, 1)])
def test_layout_of_results(b, h, s, step):
    """On the host alone: the kernel steps by the first three strides and takes a row's channels as neighbours."""
    x = windows(b, h, s, 64, step)
    for y in (x, x.transpose(1, 2), x[:, :1].expand(b, h, s, 64)):
        assert rows_apart(rope._out_for(y, None)) and rope._out_for(y, None).shape == y.shape


def test_results_that_the_kernel_cannot_write_are_refused():
    x = torch.zeros(2, 3, 5, 8)
    assert rope._out_for(x, x) is x
    for out in (torch.zeros(2, 3, 4, 8), torch.zeros(2, 3, 5, 6), x.half(), torch.zeros(2, 3, 8, 5).transpose(2, 3)):
        with pytest.raises(ValueError, match="out must be"):
            rope._out_for(x, out)


@pytest.mark.gpu
@pytest.mark.parametrize("step", [1, 8, 40])
def test_rotations(step):
    x = windows(2, 3, 9, 64, step, torch.bfloat16, "cuda")
    cos, sin = ax.rope_cos_sin_table(16, 64, 10000.0, x.dtype, x.device)
    assert torch.equal(ax.apply_rope_table(x, cos, sin), ax.apply_rope_table(x.contiguous(), cos, sin))
    assert torch.equal(ax.apply_rope(x, cos[:9], sin[:9]), ax.apply_rope(x.contiguous(), cos[:9], sin[:9]))
