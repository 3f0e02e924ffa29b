"""prompt_run: what its mirror asks of a work list on the device, and what rows that a
row does not see may hold."""
import pytest
import torch

import omni_attn as oa
from test_prompt_gpu import make, parts, run

pytestmark = pytest.mark.gpu


def test_a_work_list_shorter_than_its_plan_is_refused():
    b = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device="cuda")
    pp = oa.prompt_plan([300, 20], 4, 2)
    args = [b(320, 512), b(320, 256), b(320, 256), b(320, 512), 0.1]
    oa.prompt_run(pp, *args)
    for work in (pp.work[:-1], pp.work[:0]):
        with pytest.raises(oa.OmniAttnError, match="work must be a contiguous int32 tensor of at least"):
            oa.prompt_run(oa.Prompt(pp.plan, work), *args)
    torch.cuda.synchronize()


@pytest.mark.parametrize("lens,hq,hk,at", [([300], 4, 2, 201), ([1200, 1100, 1300], 32, 8, 129), ([700, 650], 16, 16, 640)])
@pytest.mark.parametrize("exact_p", [False, True])
def test_what_later_rows_hold_does_not_matter(lens, hq, hk, at, exact_p):
    """Rows from `at` on of every prompt get other finite values of V, and K of NaN, infinities and large values: the rows
    before keep their bits. (A later V row must be finite: a masked key weighs 0.)"""
    qkv = make(lens, hq, hk, seed=at)
    want = run(qkv, lens, hq, hk, exact_p)
    g = torch.Generator(device="cuda").manual_seed(at)
    for bad in (float("nan"), float("inf"), -float("inf"), 3e38, None):
        x, start = qkv.clone(), 0
        for n in lens:
            q, k, v = (t[start + at:start + n] for t in parts(x, hq, hk))
            k.fill_(bad) if bad is not None else k.copy_(torch.randn(k.shape, device="cuda", generator=g) * 30)
            v.copy_(torch.randn(v.shape, device="cuda", generator=g) * 1e30)
            start += n
        out, start = run(x, lens, hq, hk, exact_p), 0
        for n in lens:
            assert torch.equal(out[start:start + at], want[start:start + at]), (bad, n)
            start += n
