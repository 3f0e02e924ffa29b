"""What prompt_run's mirror asks of a work list on the device."""
import pytest
import torch

import omni_attn as oa

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
