"""Decode over the 8-bit cache at the ends of its range: values of V next to the
largest that 32 bits hold, and tokens and pages that a row does not see."""
import numpy as np
import pytest
import torch

import omni_attn as oa
from test_q8_gpu import FORMATS, Decode

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rise", [0.5, 4, 7.5])
def test_values_of_v_up_to_2_to_121(fmt, rise):
    """Scores of 0 in keys 0-31 and of `rise` (in base 2) in keys 128-159, which one wave takes after them, the rest far
    below: the result is an average of V, finite, while 2^rise times V is not. With weights p <= 1 the largest sum on the
    way is 32 keys of 2^121.8 or less: below 2^127."""
    d = Decode([300], 1, 1, 16, fmt, seed=1)
    score = torch.full((300,), -16.0)
    score[:32], score[128:160] = 0, rise
    byte = score if fmt == torch.float8_e4m3fn else score * 4  # the integers' K in quarters
    for t in range(300):
        b = int(d.pages[t // 16])
        k = d.kv[b, 0].view(16, 128)
        k[t % 16] = torch.zeros(128, device="cuda").to(fmt)
        k[t % 16, 0] = float(byte[t])
    e = d.sc.view(torch.uint8)
    e[:, 0] = 127 if fmt == torch.float8_e4m3fn else 125
    e[:, 1] = 127 + (113 if fmt == torch.float8_e4m3fn else 114)  # 448 2^113, 127 2^114: below 2^121.9
    d.q.zero_()
    d.q[0, 0] = 1
    scale = float(np.log(2.0))
    for chunk in (0, 1024):
        d.run(chunk=chunk, scale=scale)
        assert bool(d.out.isfinite().all())
        d.check(scale)
