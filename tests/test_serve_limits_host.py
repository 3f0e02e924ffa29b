"""What the 8-bit serving calls refuse at the ends of their arguments' ranges,
without a GPU: nothing here is launched (pointers are made up)."""
import pytest

import omni_attn as oa
from test_serve_host import attend, prompt


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf"), 3e38, -3e38])
def test_scales_past_the_range_of_base_2(scale):
    """The kernels multiply by scale log2(e): infinite from 2.36e38 on, which made NaN of every score of 0."""
    assert attend(scale_=scale) == oa.EINVAL and b"scale" in oa.load().omni_attn_last_error()
    assert prompt(scale=scale) == oa.EINVAL and b"scale" in oa.load().omni_attn_last_error()
