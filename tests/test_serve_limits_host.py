"""What the 8-bit serving calls refuse at the ends of their arguments' ranges,
without a GPU: nothing here is launched (pointers are made up)."""
import os
import subprocess
import sys

import pytest

import omni_attn as oa
from test_serve_host import P, attend, prompt, write


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf"), 3e38, -3e38])
def test_scales_past_the_range_of_base_2(scale):
    """The kernels multiply by scale log2(e): infinite from 2.36e38 on, which made NaN of every score of 0."""
    assert attend(scale_=scale) == oa.EINVAL and b"scale" in oa.load().omni_attn_last_error()
    assert prompt(scale=scale) == oa.EINVAL and b"scale" in oa.load().omni_attn_last_error()


def unsupported(rc):
    """Refused by its arguments: a launch that fails (ELAUNCH, as every launch here without a GPU) is not that."""
    return rc == oa.EUNSUPPORTED


def test_writes_that_no_grid_holds():
    """Threads of a launch stay below 2^32 in x (2^24 workgroups of 256), workgroups in y at 65,535 or less: of few rows
    (hk + 1) / 2 + hk + (hq + 3) / 4 of them; of many, 4 workgroups for 16 rows and one for 1 to 16 rows of q."""
    ld = lambda hq, hk: dict(hq=hq, hk=hk, ld=(hq + 2 * hk) * 128, q_ld=hq * 128, k_ld=hk * 128)
    assert unsupported(write(rows=1, **ld(1, 50000)))
    assert unsupported(write(rows=1, **ld(1, 43690))) and unsupported(write(rows=1, **ld(17485, 40776)))
    for rows, hq in ((1 << 24, 9), (1 << 24, 40), (1 << 25, 8), (1 << 26, 1), (2**31 - 1, 1)):
        assert unsupported(write(rows=rows, **ld(hq, 1))), (rows, hq)


def test_decodes_that_no_grid_holds():
    """The merge has a workgroup for each row and head, decode one in x for each split: below 2^24 of either."""
    for args in ((65535, 272, 17, 16, 1000, 512), (2**16 - 1, 257, 257, 16, 1000, 512), (1, 8, 8, 16, 2**30, 64)):
        with pytest.raises(oa.OmniAttnError) as e:
            oa.decode_plan_q8(*args)
        assert e.value.code == oa.EUNSUPPORTED
    assert oa.decode_plan_q8(65535, 272, 17, 16, 1000, 1024).splits == 1  # no merge
    assert oa.decode_plan_q8(65535, 256, 16, 16, 1000, 512).splits == 2
    assert oa.decode_plan_q8(1, 8, 8, 16, 2**30 - 64, 64).splits == 2**24 - 1
    plan = oa.decode_plan_q8(65535, 272, 17, 16, 1000, 1024)
    plan.chunk, plan.splits, plan.workspace_bytes = 512, 2, 65535 * 272 * 2 * 129 * 4
    assert unsupported(attend(plan, hq=272, hk=17, stride=272 * 128, ws=P))


def test_prompts_that_no_grid_holds():
    """512 threads for each (tile of 256 rows and heads, K/V head): below 2^23 of them."""
    lens = [2**30 // 4, 2**30 // 4, 2**30 // 4, 2**30 // 4]
    with pytest.raises(oa.OmniAttnError) as e:
        oa.prompt_plan(lens, 4, 2, device="cpu")
    assert e.value.code == oa.EUNSUPPORTED


NO_MEMORY = """
import ctypes, resource, sys
import numpy as np
import omni_attn as oa
L = oa.load()
p = lambda a: a.ctypes.data_as(ctypes.c_void_p)
if sys.argv[1] == "prompt":
    lens, work, plan = np.array([1 << 27], np.int32), np.zeros(16 + 4 * (1 << 22), np.int32), oa.PromptPlan()
    call = lambda: L.omni_attn_prompt_plan_init(1, p(lens), 8, 1, p(work), len(work), ctypes.byref(plan))
else:  # a tile for every row
    pos, work, plan = np.zeros(1 << 21, np.int32), np.zeros(16 + 4 * (1 << 21), np.int32), oa.PrefillPlan()
    call = lambda: L.omni_attn_prefill_plan_init(1 << 21, 8, 1, 16, p(pos), p(pos), p(work), len(work), ctypes.byref(plan))
size = int(open("/proc/self/statm").read().split()[0]) * resource.getpagesize() + (4 << 20)
resource.setrlimit(resource.RLIMIT_AS, (size, size))
rc = call()
assert rc == oa.EUNSUPPORTED and b"memory" in L.omni_attn_last_error(), rc
print("refused")
"""


@pytest.mark.parametrize("which", ["prompt", "prefill"])
def test_plans_without_host_memory_return_an_error(which):
    """A plan's tiles (64 and 32 MiB here) are host memory; where there is none the C call says so, and throws nothing."""
    here = os.path.dirname(oa.__file__)
    r = subprocess.run([sys.executable, "-c", NO_MEMORY, which], capture_output=True, text=True, env={**os.environ, "PYTHONPATH": here})
    assert r.returncode == 0 and "refused" in r.stdout, (r.returncode, r.stderr[-500:])
