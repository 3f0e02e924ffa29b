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


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("chunk", [0, 64])
def test_pages_and_blocks_past_a_row_are_not_followed(page, chunk):
    """Page ids past a row's last key name a page of NaN bytes with exponents of 255 (infinity): whatever weighs one of
    its blocks, even by 0, is NaN. The blocks past the row in its last page hold the same."""
    lens, at = [17, 16, 100, 300, 200], [3, 15, 63, 100, 199]
    d = Decode(lens, 8, 2, page, torch.float8_e4m3fn, seed=page, rows_of=list(enumerate(at)))
    per = page // 16
    spare = next(p for p in range(d.kv.shape[0] // per) if p not in d.pages)

    def poison(block):
        d.kv.view(torch.uint8)[block] = 0x7F
        d.sc.view(torch.uint8)[block] = 255

    for b in range(per):
        poison(spare * per + b)
    for s, p in d.rows:
        lo, hi = int(d.indptr[s]), int(d.indptr[s + 1])
        last = lo + p // page
        for b in range(p % page // 16 + 1, per):
            poison(int(d.pages[last]) * per + b)
        d.pages[last + 1:hi] = spare
    assert (d.pages == spare).sum() > 0
    d.run(chunk=chunk)
    d.check()
    d.run(chunk=chunk, ragged=False, max_len=400)
    d.check()
