"""step_tables with a ring: what a step may ask for, and the calls that read such
tables (those with a context cap)."""
import numpy as np
import pytest
import torch

import omni_attn as oa
from gpu_util import assert_close, dev_bits, host_bits
from test_tables_gpu import Step, i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("leased", [False, True])
@pytest.mark.parametrize("ring,first,count,bad", [
    (48, [10, 500], [48, 1], False), (48, [10, 500], [1, 49], True), (48, [0, 0], [2, 300], True), (1, [7, 3], [1, 1], False),
    (1, [7, 3], [2, 1], True), (33, [0, 40], [33, -1], False), (33, [0, 40], [34, -1], True), (0, [0, 40], [90, 64], False),
])
def test_a_step_of_more_rows_than_the_ring_is_refused(ring, first, count, bad, leased):
    """count > ring would give several rows of one call the same slot: code 1, nothing built and nothing taken."""
    st = Step(2, 2, 40, 60, 200, 90, seed=ring, ring=ring, leased=leased)
    st.fill(first, [0, 1])
    d = st.device()
    st.call(d, i32(first), i32(count), None)
    if not bad:
        assert st.check(d, np.array(first), np.array(count), None)["status"][0] == 0
        slots = d["slots"].cpu().numpy()
        slots = slots[slots >= 0]
        if not leased:  # (a leased table of random pages may hold one twice)
            assert len(set(slots.tolist())) == len(slots)
        return
    assert d["status"].tolist() == [1, 0, 0] + ([0, 0] if leased else st.state.tolist())
    for name in ("pos", "slots", "seq"):
        assert bool((d[name] == -1).all()), name
    assert not bool(d["row_indptr"].any()) and not bool(d["indptr"].any()) and bool((d["pages"] == 5).all())
    assert np.array_equal(d["table"].cpu().numpy(), st.table)
    if not leased:
        assert np.array_equal(d["free"].cpu().numpy(), st.free)


def test_ring_tables_are_read_by_the_calls_with_a_context_cap(oracle):
    """Positions up to and past the ring: lm_attend with context = ring reads the tables as they are."""
    heads, ring, page = 4, 50, 16
    first, count = np.array([20, 49, 50, 333], np.int32), np.array([1, 1, 1, 1], np.int32)
    st = Step(4, 4, 4, 20, 4, 20, seed=2, page=page, ring=ring)
    st.fill(first, range(4))
    d = st.device()
    st.call(d, i32(first), i32(count), None)
    want = st.check(d, first, count, None)
    rng = np.random.default_rng(3)
    bf16 = lambda *s: oracle.f32_to_bf16(rng.standard_normal(s).astype(np.float32))
    qkv, kv = bf16(4, 3 * heads * 128), bf16(20 * page, 2 * heads * 128)
    plan = oa.decode_plan(4, heads, heads, page, ring)
    out = torch.zeros(4, heads * 128, dtype=torch.bfloat16, device="cuda")
    oa.lm_attend(dev_bits(qkv), dev_bits(kv), d["pos"], d["seq"], 0, d["indptr"], d["pages"], page, out, heads, 0.09, ring, plan,
                 oa.workspace_for(plan))
    torch.cuda.synchronize()
    a = lambda x: np.array(x, np.int32)
    assert_close(host_bits(out), oracle.paged_attend(qkv, kv, a(want["pos"]), a(want["seq"]), 0, a(want["indptr"]), a(want["pages"]),
                                                     page, heads, heads, 0.09, ring), what="ring tables")
    # Each row's new key is the one that its slot names.
    for n, (f, s) in enumerate(zip(first, want["slots"])):
        q = int(f) % ring
        assert s == want["pages"][want["indptr"][n] + q // page] * page + q % page
