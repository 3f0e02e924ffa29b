"""NaN in V of a token, over the 8-bit cache: the rows of a call that see earlier keys only keep their bits, whatever rows share a group,
a tile or a split with them; the rows that see it are NaN in the dims that hold it, and keep the others' bits."""
import numpy as np
import pytest
import torch

import omni_attn as oa
from test_multi_gpu import APART, SCALE, Cache, bf16, i32

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


def run(c, counts, hq, pos, chunk, exact=False, max_len=None):
    rows = sum(counts)
    q = bf16(torch.Generator(device="cuda").manual_seed(5), rows, hq * 128)
    out = torch.full((rows, hq * 128), 7.0, dtype=torch.bfloat16, device="cuda")
    mp = oa.extend_plan(counts, hq, c.hk, max_len or max(c.lens), c.lens, chunk, exact_p=exact)
    oa.qwen3_extend_q8(mp, q, c.kv, c.sc, i32(pos), c.indptr, c.pages, c.page, out, SCALE, oa.workspace_for(mp.plan))
    torch.cuda.synchronize()
    return mp, out.view(rows, c.hk, hq // c.hk, 128)


def check(c, counts, hq, bad, chunk, pos=None, exact=False, max_len=None):
    """bad: (sequence, token, K/V head, dim, byte) of each NaN. Both calls, bit by bit."""
    if pos is None:
        pos = [n - k + i for n, k in zip(c.lens, counts) for i in range(k)]
    mp, want = run(c, counts, hq, pos, chunk, exact, max_len)
    assert not bool(want.isnan().any())
    want = want.clone()
    raw, at, starts = c.kv.view(torch.uint8), 0, np.cumsum([0] + counts)
    kept = raw.clone()
    for s, t, h, d, byte in bad:
        slot = c.slots[s][t]
        raw[slot // 16, c.hk + h].view(128, 16)[d, slot % 16] = byte
        for i in range(starts[s], starts[s + 1]):
            if pos[i] >= t:
                want[i, h, :, d] = float("nan")
    _, got = run(c, counts, hq, pos, chunk, exact, max_len)
    raw.copy_(kept)
    nan = want.isnan()
    assert torch.equal(got.isnan(), nan), [x.tolist() for x in (got.isnan() != nan).nonzero()[:5]]
    same = got.view(torch.int16) == want.view(torch.int16)
    assert bool((same | nan).all()), [x.tolist() for x in (~(same | nan)).nonzero()[:5]]
    return mp


def spots(rng, lens, counts, hk, n):
    """NaNs among a sequence's last tokens and a little before, in a few dims, of either sign."""
    out = []
    for s, (m, k) in enumerate(zip(lens, counts)):
        for _ in range(n if k else 0):
            t = int(rng.integers(max(0, m - k - 2), m))
            out.append((s, t, int(rng.integers(hk)), int(rng.integers(128)), int(rng.choice([0x7f, 0xff]))))
    return out


@pytest.mark.parametrize("hq,hk", [(1, 1), (4, 2), (3, 1), (8, 2), (16, 2), (14, 1), (16, 1)])
def test_groups(hq, hk):
    """Groups of one and two column blocks, unsplit and in splits, where the new rows' keys begin and end in any place of a tile and block."""
    g = hq // hk
    counts = [16 // g, max(32 // g - 1, 1), 1, 32 // g, 2, 16 // g + 1 if 16 // g + 1 <= 32 // g else 1]
    rng = np.random.default_rng(hq)
    for chunk in (64, APART):
        lens = [c + int(x) for c, x in zip(counts, (0, 37, 200, 300, 15, 95))]
        c = Cache(hq + chunk, lens, hk, 16, E4M3)
        for n in (1, 6):
            mp = check(c, counts, hq, spots(rng, lens, counts, hk, n), chunk)
            assert mp.plan.tiles == 0


def test_groups_at_any_positions():
    lens, counts = [300, 75], [8, 3]
    c = Cache(6, lens, 2, 16, E4M3)
    pos = [299, 0, -1, 150, 150, 31, 32, -7, 74, -1, 3]
    bad = [(0, 0, 1, 5, 0x7f), (0, 31, 0, 127, 0xff), (0, 32, 0, 0, 0x7f), (0, 151, 1, 64, 0x7f), (0, 299, 0, 63, 0x7f), (1, 4, 0, 9, 0x7f), (1, 74, 1, 9, 0x7f)]
    for chunk in (64, 0):
        for spot in bad:
            check(c, counts, 4, [spot], chunk, pos)
        check(c, counts, 4, bad, chunk, pos)
    check(c, counts, 4, bad, 64, pos, max_len=65)  # splits that grow past the plan's bound
