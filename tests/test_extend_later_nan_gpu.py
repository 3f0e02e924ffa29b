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


@pytest.mark.parametrize("exact", [False, True])
@pytest.mark.parametrize("hq,hk", [(1, 1), (4, 2), (8, 2), (16, 2), (16, 1), (3, 1), (10, 2), (6, 1), (14, 2)])
def test_tiles(hq, hk, exact):
    """Whole tiles and parts of them, with a sequence in a group beside them: NaNs in any block of the keys that the rows end in."""
    g = hq // hk
    counts = [32 // g + 1, 64 // g + 3, 256 // g, 1, 256 // g + 1, 0, 2]
    rng = np.random.default_rng(hq)
    lens = [counts[0], 129, 256 // g, 70, 256 // g + 128, 5, 300]
    c = Cache(hq, lens, hk, 16, E4M3)
    for n in (1, 9):
        mp = check(c, counts, hq, spots(rng, lens, counts, hk, n), APART, exact=exact)
        assert mp.plan.tiles == 5 and mp.plan.group_rows == 3
    check(c, counts, hq, spots(rng, lens, counts, hk, 3), 0, exact=exact)


@pytest.mark.parametrize("exact", [False, True])
@pytest.mark.parametrize("seqs,hk", [(1, 2), (12, 8), (20, 16)])
def test_every_form_of_a_tile(seqs, hk, exact):
    """Quarters, halves, whole tiles."""
    rng = np.random.default_rng(seqs)
    counts = [int(x) for x in rng.integers(34, 128, seqs)]
    lens = [c + int(x) for c, x in zip(counts, rng.integers(0, 260, seqs))]
    mp = check(Cache(seqs, lens, hk, 16, E4M3), counts, 2 * hk, spots(rng, lens, counts, hk, 4), APART, exact=exact)
    items = mp.plan.tile_units * hk
    assert mp.plan.split_tiles == 0 and (items <= 64, items <= 128) == ((True, True), (False, True), (False, False))[(1, 12, 20).index(seqs)]


@pytest.mark.parametrize("exact", [False, True])
@pytest.mark.parametrize("hq,hk", [(4, 1), (2, 2), (5, 1), (16, 1)])
def test_tiles_in_splits(hq, hk, exact):
    """Rows that end in other splits than the NaN's, in the same one, and rows that are none."""
    lens, counts = [2600, 700, 90], [70, 40, 40]
    c = Cache(hq, lens, hk, 16, E4M3)
    pos = [2599 - 37 * i if i % 3 else -1 for i in range(70)] + [i for i in range(40)] + [-1] * 40
    bad = [(0, t, t % hk, 11 * i, 0x7f) for i, t in enumerate((3, 127, 128, 900, 1500, 2563, 2599))] + [(1, 20, 0, 3, 0xff), (2, 5, 0, 9, 0x7f)]
    for most in (None, 1100):
        for spot in (*([b] for b in bad[:4]), bad):
            mp = check(c, counts, hq, spot, APART, pos, exact, most)
        assert mp.plan.split_tiles > 0
    check(c, counts, hq, bad, 0, pos, exact)


@pytest.mark.parametrize("chunk", [64, APART])
@pytest.mark.parametrize("rows", [3, 150])
def test_values_that_round_up_past_bf16(rows, chunk):
    """E4M3 rounds 1.99 2^127 to 2^128, which no bf16 holds: rows before it keep their bits; rows that see it take it as 2^128 in groups, as
    the largest bf16 value in tiles (2^-8 less)."""
    import multi_refs as M

    n, hk, hq = 400, 1, 2
    c = Cache(rows, [n], hk, 16, E4M3)
    pos = list(range(n - rows, n))
    t = n - 16 - rows // 3  # the first token of the block is the huge one; nothing else of the block has a value of V
    t -= t % 16
    slot, raw = c.slots[0][t], c.kv.view(torch.uint8)
    v = raw[slot // 16, hk].view(128, 16)
    v.zero_()
    _, want = run(c, [rows], hq, pos, chunk)
    want = want.clone()
    v[::3, slot % 16] = 0x78  # 256
    v[1::3, slot % 16] = 0xf8
    c.sc.view(torch.uint8)[slot // 16, hk] = 247  # 2^120
    mp, got = run(c, [rows], hq, pos, chunk)
    assert (mp.plan.tiles > 0) == (rows > 16)
    before = [i for i in range(rows) if pos[i] < t]
    assert rows == 3 or before
    assert torch.equal(got[before], want[before])
    q = bf16(torch.Generator(device="cuda").manual_seed(5), rows, hq * 128)
    ref, size = M.rows_of(q.cpu().view(rows, hq, 128), *c.tokens(0), [p + 1 for p in pos], SCALE)
    bound = M.bound(ref, size, mp.plan.tiles > 0) + (2.0 ** -8 * size if mp.plan.tiles else 0.0)
    assert float(ref.abs().max()) > 1e33 and bool(((got.view(rows, hq, 128).cpu().double() - ref).abs() <= bound).all())


@pytest.mark.parametrize("counts,chunk", [([5, 9], 64), ([5, 9], APART), ([90, 40], APART)])
def test_nan_in_k(counts, chunk):
    """NaN in K of a later token leaves the rows before it their bits; the rows that see it are NaN."""
    lens, hk, hq = [180, 77], 2, 4
    c = Cache(44, lens, hk, 16, E4M3)
    pos = [n - k + i for n, k in zip(lens, counts) for i in range(k)]
    _, want = run(c, counts, hq, pos, chunk)
    want = want.clone()
    starts = [0, counts[0]]
    for s, h, back in ((0, 1, 2), (1, 0, 4)):
        t = lens[s] - back
        slot = c.slots[s][t]
        c.kv.view(torch.uint8)[slot // 16, h].view(16, 128)[slot % 16, 77] = 0x7f
        for i in range(counts[s]):
            if pos[starts[s] + i] >= t:
                want[starts[s] + i, h] = float("nan")
    _, got = run(c, counts, hq, pos, chunk)
    nan = want.isnan()
    assert torch.equal(got.isnan(), nan) and bool(((got.view(torch.int16) == want.view(torch.int16)) | nan).all())
