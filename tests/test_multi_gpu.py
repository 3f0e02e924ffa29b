"""Several rows per sequence over the 8-bit cache, and rows over encoder states, on the
GPU: against 64 bits, at the counts, lengths and head layouts where groups, tiles and
splits begin and end; with rubbish in every place that no row sees; in graphs."""
import math

import numpy as np
import pytest
import torch

import multi_refs as M
import omni_attn as oa
import serve_refs as R

pytestmark = pytest.mark.gpu

FORMATS = [torch.float8_e4m3fn, torch.int8]
SCALE = 128 ** -0.5
APART = 1 << 14  # a chunk: groups unsplit, and sequences of more than 32 packed rows in tiles


def i32(a):
    return torch.from_numpy(np.array(a, dtype=np.int32).copy()).cuda()


def bf16(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g).to(torch.bfloat16)


class Cache:
    """Sequences of the given lengths in an 8-bit cache; every token that is none of theirs is NaN (E4M3) or the largest integer
    under the largest exponent."""

    def __init__(self, seed, lens, hk, page, fmt, spare=3):
        rng = np.random.default_rng(seed)
        g = torch.Generator(device="cuda").manual_seed(seed)
        need = [-(-n // page) for n in lens]
        pool, per = sum(need) + spare, page // 16
        self.kv, self.sc = oa.q8_cache(pool, page, hk, fmt)
        x = torch.randn(self.kv.shape, device="cuda", generator=g)
        self.kv.copy_((x * 90).clamp(-448, 448).to(fmt) if fmt == torch.float8_e4m3fn else (x * 40).round().clamp(-127, 127).to(fmt))
        self.sc.view(torch.uint8).copy_(torch.randint(116, 123, self.sc.shape, device="cuda", generator=g).to(torch.uint8))
        ids = rng.permutation(pool)
        self.hk, self.page, self.lens = hk, page, lens
        indptr, pages = [0], []
        live = torch.zeros(pool * page, dtype=torch.bool)
        self.slots = []
        for n, c in zip(lens, need):
            mine = [int(x) for x in ids[len(pages):len(pages) + c]]
            pages += mine
            indptr.append(len(pages))
            at = [mine[t // page] * page + t % page for t in range(n)]
            self.slots.append(at)
            live[at] = True
        self.indptr, self.pages = i32(indptr), i32(pages if pages else [0])
        raw = self.kv.view(torch.uint8)
        bad = 0x7f
        dead = (~live).view(-1, 16).cuda()
        k = raw[:, :hk].view(-1, hk, 16, 128)
        k[dead[:, None].expand(-1, hk, -1)] = bad
        v = raw[:, hk:].view(-1, hk, 128, 16).transpose(2, 3)
        v[dead[:, None].expand(-1, hk, -1)] = bad
        self.sc.view(torch.uint8)[dead.all(1)] = 254
        assert per >= 1

    def tokens(self, s):
        if not hasattr(self, "_t"):
            self._t = R.Cache(self.kv, self.sc, self.hk).tokens()
        return self._t[0][self.slots[s]], self._t[1][self.slots[s]]


def extend(c, counts, hq, pos=None, chunk=0, keys=True, extra=2, seed=1, max_len=None, stream=None, stride=0, scale=SCALE):
    """Runs the call on the last counts[s] tokens of each sequence (or at `pos`), checks it against 64 bits; the plan and the output."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows = sum(counts)
    if pos is None:
        pos = [n - k + i for n, k in zip(c.lens, counts) for i in range(k)]
    q = bf16(g, rows + extra, hq * 128 + stride)[:, :hq * 128]
    out = torch.full((rows + extra, hq * 128), 7.0, dtype=torch.bfloat16, device="cuda")
    mp = oa.extend_plan(counts, hq, c.hk, max_len or max(c.lens + [1]), c.lens if keys else None, chunk)
    ws = oa.workspace_for(mp.plan)
    if ws is not None:
        ws.fill_(0xff)
    torch.cuda.synchronize()
    oa.qwen3_extend_q8(mp, q, c.kv, c.sc, i32(pos if rows else [0]), c.indptr, c.pages, c.page, out, scale, ws, stream)
    torch.cuda.synchronize()
    assert bool((out[rows:] == 7).all())
    at = 0
    for s, k in enumerate(counts):
        if k:
            kk, vv = c.tokens(s)
            lim = [p + 1 for p in pos[at:at + k]]
            want, size = M.rows_of(q[at:at + k].cpu().view(k, hq, 128), kk, vv, lim, scale)
            got = out[at:at + k].cpu().double().view(k, hq, 128)
            err = (got - want).abs() - M.bound(want, size, mp.plan.tiles > 0)
            assert bool((err <= 0).all()), f"sequence {s}: {float(err.max()):.3g} at {int(err.argmax())}, {err.isnan().any()}"
            for i, n in enumerate(lim):
                if n <= 0:
                    assert bool((out[at + i] == 0).all())
        at += k
    return mp, out


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("hq,hk", [(1, 1), (4, 2), (3, 1), (8, 2), (5, 1), (16, 2), (14, 1), (16, 1)])
def test_extend_of_few_rows(hq, hk, fmt):
    """Groups of one row to a little more than two groups', lengths about a tile and a block, a sequence without rows."""
    g = hq // hk
    counts = [1, 16 // g, 0, 16 // g + 1, 32 // g, 32 // g + 1, 2, 3]
    lens = [1, 16 // g + 31, 9, 32 + 16 // g, 32 // g, 130, 33, 64]
    c = Cache(hq * 7 + hk, lens, hk, 16, fmt)
    mp, _ = extend(c, counts, hq)
    assert mp.plan.rows == sum(counts)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("page", [16, 48, 256])
@pytest.mark.parametrize("chunk", [64, 128, 0])
def test_extend_in_splits(page, chunk, fmt):
    """Rows that end in different splits, rows in the first split alone, one to thirty splits."""
    lens = [1900, 700, 129, 128, 64, 65, 5]
    counts = [4, 70, 3, 1, 2, 5, 5]
    c = Cache(page + chunk, lens, 2, page, fmt)
    extend(c, counts, 8, chunk=chunk, keys=chunk != 128)
    extend(c, counts, 2, chunk=chunk, seed=2)


def test_extend_past_the_plans_bound():
    """Rows longer than max_len run in splits that grow."""
    c = Cache(5, [900, 40], 2, 16, torch.float8_e4m3fn)
    mp, _ = extend(c, [3, 2], 4, chunk=64, max_len=128)
    assert mp.plan.splits == 2


def test_extend_at_any_positions():
    """Positions in no order, twice the same, far behind, and rows that are none."""
    c = Cache(6, [300, 75], 2, 16, torch.int8)
    pos = [299, 0, -1, 150, 150, 31, 32, -7, 74, -1, 3]
    for chunk in (0, 64):
        extend(c, [8, 3], 4, pos=pos, chunk=chunk)
    extend(c, [8, 3], 4, pos=[-1] * 11, chunk=64)


def test_extend_equals_decode_on_single_rows():
    """One row a sequence: the row of omni_qwen3_attend_q8, to the rounding of the output."""
    lens = [1, 17, 500, 1234]
    c = Cache(9, lens, 2, 16, torch.float8_e4m3fn)
    mp, out = extend(c, [1] * 4, 8, extra=0)
    g = torch.Generator(device="cuda").manual_seed(1)
    q = bf16(g, 4, 8 * 128)
    plan = oa.decode_plan_q8(4, 8, 2, 16, max(lens))
    other = torch.zeros_like(out)
    oa.qwen3_attend_q8(q, c.kv, c.sc, i32([n - 1 for n in lens]), None, 0, c.indptr, c.pages, 16, other, 8, 2, SCALE, plan, oa.workspace_for(plan))
    torch.cuda.synchronize()
    assert bool(((out.float() - other.float()).abs() <= 2.0 ** -7 * other.float().abs() + 2.0 ** -12).all())


@pytest.mark.parametrize("scale", [0.0, -SCALE, 3.0, -40.0])
def test_extend_scales(scale):
    c = Cache(12, [80, 41], 1, 16, torch.int8)
    if abs(scale) < 1:
        extend(c, [5, 20], 2, scale=scale)
        return
    # One key takes nearly all the weight: which one is a matter of the scores' own rounding; finite, and within the values.
    g = torch.Generator(device="cuda").manual_seed(1)
    q = bf16(g, 25, 256)
    out = torch.zeros_like(q)
    mp = oa.extend_plan([5, 20], 2, 1, 80)
    oa.qwen3_extend_q8(mp, q, c.kv, c.sc, i32(list(range(75, 80)) + list(range(21, 41))), c.indptr, c.pages, 16, out, scale, oa.workspace_for(mp.plan))
    torch.cuda.synchronize()
    assert bool(torch.isfinite(out).all()) and float(out.abs().max()) <= 127 * 2.0 ** (122 - 127) * 1.01


@pytest.mark.parametrize("stride", [8, 128])
def test_extend_of_strided_rows_on_another_stream(stride):
    c = Cache(13, [90, 33], 2, 32, torch.int8)
    extend(c, [20, 1], 4, stride=stride, stream=torch.cuda.Stream())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("hq,hk,page", [(1, 1, 16), (4, 2, 48), (8, 2, 16), (16, 2, 256), (3, 1, 16), (10, 2, 16), (6, 1, 32), (14, 2, 16), (16, 1, 16)])
def test_extend_in_tiles(hq, hk, page, fmt):
    """Tiles of a few packed rows to more than one, keys about one and two key tiles; with sequences in groups beside them."""
    g = hq // hk
    counts = [32 // g + 1, 64 // g + 3, 256 // g, 1, 256 // g + 1, 0, 2]
    lens = [counts[0], 129, 256 // g, 70, 256 // g + 128, 5, 300]
    mp, _ = extend(Cache(hq + page, lens, hk, page, fmt), counts, hq, chunk=APART)
    assert mp.plan.tiles == 5 and sum(mp.plan.groups) == 2


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("seqs,hk", [(1, 2), (12, 8), (20, 16)])
def test_extend_in_every_form_of_a_tile(seqs, hk, fmt):
    """Quarters, halves and whole tiles: the plan splits none of these."""
    rng = np.random.default_rng(seqs)
    counts = [int(x) for x in rng.integers(34, 130, seqs)]
    lens = [c + int(x) for c, x in zip(counts, rng.integers(0, 260, seqs))]
    mp, _ = extend(Cache(seqs, lens, hk, 16, fmt), counts, 2 * hk, chunk=APART)
    assert mp.plan.tiles * hk in ((2, 96, 320) if seqs < 20 else (320,)) or mp.plan.tiles >= seqs
    assert mp.plan.split_tiles == 0


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("hq,hk", [(4, 1), (2, 2), (5, 1), (16, 1)])
def test_extend_of_tiles_in_splits(hq, hk, fmt):
    """Few tiles over long contexts, rows that see nothing of the later splits, and (a bound below the lengths) splits that grow."""
    c = Cache(hq, [2600, 700, 90], hk, 16, fmt)
    counts = [70, 40, 40]
    for most in (None, 1100):
        mp, _ = extend(c, counts, hq, max_len=most, seed=3, chunk=APART)
        assert mp.plan.split_tiles > 0
    pos = [2599 - 37 * i if i % 3 else -1 for i in range(70)] + [i for i in range(40)] + [-1] * 40
    extend(c, counts, hq, pos=pos, seed=4, chunk=APART)
    extend(c, counts, hq, pos=pos, seed=4)


def test_extend_of_tiles_at_any_positions():
    """Rows in no order, rows that are none, a tile and a part of one without any."""
    for hk, n in ((1, 300), (8, 40)):
        c = Cache(30 + hk, [500, 90], hk, 16, torch.float8_e4m3fn)
        rng = np.random.default_rng(hk)
        pos = [int(x) for x in rng.integers(-3, 500, n)] + [-1] * 40
        pos[:20] = [-1] * 20
        extend(c, [n, 40], 4 * hk, pos=pos, chunk=APART)
        extend(c, [n, 40], 4 * hk, pos=pos)


@pytest.mark.parametrize("scale", [0.0, -SCALE])
def test_extend_of_tiles_scales_strides_streams(scale):
    c = Cache(41, [200, 150], 2, 16, torch.int8)
    extend(c, [120, 60], 4, scale=scale, stride=24, stream=torch.cuda.Stream(), chunk=APART)


def test_a_tile_whose_row_sees_nothing_leaves_the_others_alone():
    """NaN in V of a token that only later rows see: the rows of other sequences keep their bits."""
    c = Cache(42, [150, 150], 1, 16, torch.float8_e4m3fn)
    _, a = extend(c, [100, 100], 2, chunk=APART)
    raw = c.kv.view(torch.uint8)
    slot = c.slots[0][149]
    raw[slot // 16, 1].view(128, 16)[:, slot % 16] = 0x7f
    q = bf16(torch.Generator(device="cuda").manual_seed(1), 202, 256)
    out = torch.zeros(202, 256, dtype=torch.bfloat16, device="cuda")
    mp = oa.extend_plan([100, 100], 2, 1, 150, c.lens, APART)
    assert mp.plan.tiles > 0
    pos = i32(list(range(50, 150)) * 2)
    oa.qwen3_extend_q8(mp, q, c.kv, c.sc, pos, c.indptr, c.pages, 16, out, SCALE, oa.workspace_for(mp.plan))
    torch.cuda.synchronize()
    assert bool(out[99].isnan().any()) and torch.equal(out[100:200], a[100:200])


# ------------------------------------------------------------------ cross
def cross(seed, counts, lens, hq, hk, chunk=0, keys=True, of=None, max_len=None, extra=2, layout="one", stream=None, scale=SCALE):
    """Sources of the given lengths in any order, NaN between them; the call against 64 bits."""
    rng = np.random.default_rng(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    order = rng.permutation(len(lens))
    first, at = [0] * len(lens), 1
    for e in order:
        first[e] = at
        at += max(0, lens[e]) + int(rng.integers(0, 3))
    total = at + 1
    k, v = bf16(g, total, hk * 128), bf16(g, total, hk * 128)
    live = torch.zeros(total, dtype=torch.bool)
    for e, n in enumerate(lens):
        live[first[e]:first[e] + max(0, n)] = True
    k[~live.cuda()], v[~live.cuda()] = math.nan, math.nan
    if layout == "one":  # parts of one row
        kv = torch.cat([k, v], 1)
        k, v = kv[:, :hk * 128], kv[:, hk * 128:]
    elif layout == "apart":
        pad = torch.zeros(total, hk * 128 + 8, dtype=torch.bfloat16, device="cuda")
        pad[:, 8:] = v
        v = pad[:, 8:]
    rows = sum(counts)
    q = bf16(g, rows + extra, hq * 128)
    out = torch.full((rows + extra, hq * 128), 7.0, dtype=torch.bfloat16, device="cuda")
    named = list(range(len(counts))) if of is None else of
    mp = oa.cross_plan(counts, hq, hk, max_len or max(lens + [1]), [max(0, lens[e]) for e in named] if keys else None, chunk)
    ws = oa.workspace_for(mp.plan)
    if ws is not None:
        ws.fill_(0xff)
    torch.cuda.synchronize()
    oa.cross_run(mp, q, k, v, None if of is None else i32(of), i32(first), i32(lens), out, scale, ws, stream)
    torch.cuda.synchronize()
    assert bool((out[rows:] == 7).all())
    at = 0
    for s, c in enumerate(counts):
        e = named[s]
        n = max(0, lens[e])
        part = slice(first[e], first[e] + n)
        want, size = M.rows_of(q[at:at + c].cpu().view(c, hq, 128), k[part].cpu().view(n, hk, 128), v[part].cpu().view(n, hk, 128), [n] * c, scale)
        got = out[at:at + c].cpu().double().view(c, hq, 128)
        err = (got - want).abs() - M.bound(want, size, mp.plan.tiles > 0)
        assert c == 0 or bool((err <= 0).all()), f"sequence {s}: {float(err.max()):.3g}, {err.isnan().any()}"
        at += c
    return mp, out


@pytest.mark.parametrize("hq,hk", [(1, 1), (4, 2), (3, 1), (8, 2), (5, 1), (16, 2), (14, 1), (16, 1), (4, 4)])
@pytest.mark.parametrize("layout", ["own", "one", "apart"])
def test_cross_of_few_rows(hq, hk, layout):
    g = hq // hk
    counts = [1, 16 // g, 0, 16 // g + 1, 32 // g, 32 // g + 1, 2, 3, 5]
    lens = [1, 31, 9, 32, 33, 130, 0, 64, -3]
    cross(hq * 5 + hk, counts, lens, hq, hk, layout=layout)


@pytest.mark.parametrize("chunk", [64, 128, 0])
def test_cross_in_splits(chunk):
    cross(chunk, [4, 70, 3, 1, 2, 5, 5], [1900, 700, 129, 128, 0, 65, 5], 8, 2, chunk=chunk, keys=chunk != 128)


@pytest.mark.parametrize("hq,hk", [(1, 1), (4, 2), (8, 2), (16, 2), (3, 1), (10, 2), (6, 1), (14, 2), (16, 1)])
@pytest.mark.parametrize("layout", ["own", "one", "apart"])
def test_cross_in_tiles(hq, hk, layout):
    g = hq // hk
    counts = [32 // g + 1, 64 // g + 3, 256 // g, 1, 256 // g + 1, 0, 2, 40]
    lens = [1, 129, 128, 70, 257, 5, 300, 0]
    mp, _ = cross(hq, counts, lens, hq, hk, layout=layout, chunk=APART)
    assert mp.plan.tiles == sum(-(-c // (256 // g)) for c in counts if c > 32 // g)


@pytest.mark.parametrize("seqs,hk", [(1, 2), (12, 8), (20, 16)])
def test_cross_in_every_form_of_a_tile(seqs, hk):
    rng = np.random.default_rng(seqs)
    counts = [int(x) for x in rng.integers(34, 130, seqs)]
    mp, _ = cross(seqs, counts, [int(x) for x in rng.integers(0, 300, seqs)], 2 * hk, hk, chunk=APART)
    assert mp.plan.split_tiles == 0


@pytest.mark.parametrize("seqs,hk,g", [(1, 1, 16), (4, 4, 16), (12, 8, 16), (1, 1, 5), (6, 4, 3), (6, 8, 7)])
def test_every_form_of_other_head_layouts(seqs, hk, g):
    rng = np.random.default_rng(seqs + g)
    counts = [int(x) for x in rng.integers(34, 130, seqs)]
    lens = [c + int(x) for c, x in zip(counts, rng.integers(0, 260, seqs))]
    e, _ = extend(Cache(seqs, lens, hk, 16, torch.float8_e4m3fn), counts, g * hk, chunk=APART)
    x, _ = cross(seqs, counts, lens, g * hk, hk, chunk=APART)
    assert e.plan.tiles == x.plan.tiles == sum(-(-c // (256 // g)) for c in counts) and e.plan.split_tiles == x.plan.split_tiles == 0


@pytest.mark.parametrize("most", [None, 1100])
@pytest.mark.parametrize("hq", [4, 7, 16])
def test_cross_of_tiles_in_splits(hq, most):
    mp, _ = cross(6, [70, 40, 40, 50], [2600, 700, 90, 0], hq, 1, max_len=most, chunk=APART)
    assert mp.plan.split_tiles > 0


@pytest.mark.parametrize("scale", [0.0, -SCALE])
def test_cross_of_tiles_scales_streams(scale):
    cross(7, [120, 60], [200, 150], 4, 2, scale=scale, stream=torch.cuda.Stream(), chunk=APART)


def test_cross_over_shared_sources():
    cross(3, [5, 5, 1, 40, 2], [300, 77, 12], 4, 2, of=[1, 0, 1, 1, 2])


def test_cross_past_the_plans_bound():
    mp, _ = cross(4, [3, 2], [900, 40], 4, 2, chunk=64, max_len=128)
    assert mp.plan.splits == 2


@pytest.mark.parametrize("scale", [0.0, -SCALE])
def test_cross_scales_on_another_stream(scale):
    cross(5, [3, 20], [200, 40], 2, 1, scale=scale, stream=torch.cuda.Stream())


def test_the_mirror_refuses_what_the_kernels_do_not_take():
    hq, hk = 4, 2
    b = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device="cuda")
    kv, sc = oa.q8_cache(4, 16, hk)
    z = i32([0] * 8)

    def refused(f, *a):
        with pytest.raises(oa.OmniAttnError):
            f(*a)

    e, x = oa.extend_plan([2, 1], hq, hk, 300, chunk=64), oa.cross_plan([2, 1], hq, hk, 300, chunk=64)
    ws = oa.workspace_for(e.plan)
    good = [e, b(3, 512), kv, sc, z[:3], z[:3], z, 16, b(3, 512), SCALE, ws]
    oa.qwen3_extend_q8(*good)
    for at, bad in ((0, x), (1, b(2, 512)), (1, b(3, 256)), (1, b(3, 512).float()), (2, kv.view(torch.uint8)), (2, kv[:, :2]), (3, sc[:3]),
                    (3, sc.cpu()), (4, z[:2]), (5, z[:2]), (5, z[:3].long()), (7, 24), (8, b(2, 512)), (8, b(512, 3).t()), (10, ws[:-1]), (10, None),
                    (10, ws.cpu()), (0, oa.Multi(e.plan, e.work[:4])), (1, b(3, 516)[:, 2:514])):
        refused(oa.qwen3_extend_q8, *good[:at], bad, *good[at + 1:])
    ws = oa.workspace_for(x.plan)
    good = [x, b(3, 512), b(9, 256), b(9, 256), z[:2], z[:5], z[:5], b(3, 512), SCALE, ws]
    oa.cross_run(*good)
    for at, bad in ((0, e), (1, b(2, 512)), (2, b(9, 128)), (3, b(9, 256).float()), (2, b(256, 9).t()), (4, z[:1]), (5, z[:5].float()), (6, z[:4]),
                    (7, b(3, 256)), (9, ws[:-1]), (9, None), (0, oa.Multi(x.plan, x.work[:4])), (3, b(9, 260)[:, 2:258])):
        refused(oa.cross_run, *good[:at], bad, *good[at + 1:])
    refused(oa.cross_run, x, b(3, 512), b(9, 256), b(9, 256), None, z[:1], z[:5], b(3, 512), SCALE, ws)  # a source for each sequence
    torch.cuda.synchronize()


def test_no_rows_and_no_sequences():
    for counts in ([], [0, 0]):
        mp = oa.cross_plan(counts, 4, 2, 10)
        out = torch.full((2, 512), 7.0, dtype=torch.bfloat16, device="cuda")
        q, k = torch.zeros(1, 512, dtype=torch.bfloat16, device="cuda"), torch.zeros(1, 256, dtype=torch.bfloat16, device="cuda")
        oa.cross_run(mp, q, k, k, None, i32([0, 0]), i32([0, 0]), out, SCALE)
        torch.cuda.synchronize()
        assert bool((out == 7).all())


@pytest.mark.parametrize("hq,hk", [(1, 1), (3, 1), (14, 2), (16, 1)])
def test_one_tile_in_many_splits(hq, hk):
    """Waves share a row's splits: all of them, as many as one wave takes at once, one, none; rows that see only the first; rows * G that
    are no multiple of four."""
    g = hq // hk
    rows = 32 // g + 1
    c = Cache(hq, [9000], hk, 16, torch.int8)
    for last in (8999, 1900, 1000, 129, 60, -1):
        pos = [max(last - 3 * i, -1) if i % 4 else min(last, 5) for i in range(rows)]
        mp, _ = extend(c, [rows], hq, pos=pos)
        assert mp.plan.tile_segments > 8 * mp.plan.split_tiles > 0
    for n in (9000, 1900, 1000, 129, 60, 0):
        mp, _ = cross(hq, [rows], [n], hq, hk, max_len=9000, keys=False)
        assert mp.plan.tile_segments > 8 * mp.plan.split_tiles > 0


@pytest.mark.parametrize("counts", [[3, 1], [40, 1]])
def test_a_bound_that_bounds_nothing(counts):
    c = Cache(3, [700, 90], 1, 16, torch.int8)
    extend(c, counts, 4, max_len=2**31 - 1, keys=False)
    cross(3, counts, [700, 90], 4, 1, max_len=2**31 - 1, keys=False)


@pytest.mark.parametrize("hq,hk,rows", [(1, 1, 1), (3, 1, 5), (14, 2, 4), (16, 1, 2), (9, 3, 7)])
def test_groups_in_many_splits(hq, hk, rows):
    """Waves share a row's splits: all of them, a batch more than one wave takes at once, one batch, two splits, one, none; a row alone in
    its workgroup."""
    c = Cache(hq, [9000, 40], hk, 16, torch.float8_e4m3fn)
    for last in (8999, 2100, 1000, 100, 60, -1):
        pos = [max(last - 3 * i, -1) if i % 4 < 3 else min(last, 5) for i in range(rows)] + [39]
        mp, _ = extend(c, [rows, 1], hq, pos=pos, chunk=64)
        assert mp.plan.splits > 32 and mp.plan.tiles == 0
    for n in (9000, 2100, 1000, 100, 60, 0):
        mp, _ = cross(hq, [rows, 1], [n, 33], hq, hk, max_len=9000, keys=False, chunk=64)
        assert mp.plan.splits > 32 and mp.plan.tiles == 0


# ------------------------------------------------------------------ all sequences in one kernel
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("hq,hk", [(1, 1), (4, 2), (3, 1), (8, 2), (16, 2), (16, 1)])
def test_small_calls_run_in_one_kernel(hq, hk, fmt):
    """A row, what one and two column blocks of groups hold, and more: all as groups over 900 and 60 keys, as tiles over 1200 if more is
    there, as groups in splits if not."""
    g = hq // hk
    for longest, last in ((900, 64 // g + 3), (60, 64 // g + 3), (1200, 64 // g + 3), (6000, 2)):
        counts = [1, 16 // g, 0, 16 // g + 1, 32 // g, last, 2]
        lens = [max(n, c) for n, c in zip((longest, 33, 7, 41, 64, longest - 7, 16), counts)]
        tiles = longest == 1200
        e, _ = extend(Cache(hq + longest, lens, hk, 16, fmt), counts, hq)
        x, _ = cross(hq + longest, counts, lens, hq, hk)
        for p in (e.plan, x.plan):
            assert (p.tiles > 0, p.group_rows) == ((True, 0) if tiles else (False, sum(counts))) and p.groups[0] == 0
            assert p.splits > 1 or longest < 6000


# ------------------------------------------------------------------ odd heads, far offsets
@pytest.mark.parametrize("hq,hk", [(3, 3), (10, 5), (22, 11)])
def test_kv_heads_that_are_no_power_of_two(hq, hk):
    """Few rows and tiles, split and not, apart and together."""
    for chunk in (64, 0):
        extend(Cache(50 + hk, [900, 200, 70], hk, 16, torch.int8), [3, 70, 40], hq, chunk=chunk)
        extend(Cache(51 + hk, [2600, 700], hk, 16, torch.float8_e4m3fn), [40, 3], hq, chunk=chunk)
        cross(52 + hk, [3, 70, 40], [900, 200, 70], hq, hk, chunk=chunk)
        cross(53 + hk, [40, 3], [2600, 700], hq, hk, chunk=chunk)


def test_extend_past_32_bits():
    """Blocks at the end of a cache of 4.5 GiB."""
    hk, blocks = 8, 147_500
    kv = torch.zeros(blocks, 2 * hk, 2048, dtype=torch.int8, device="cuda")
    sc = torch.full((blocks, 2 * hk), 120, dtype=torch.uint8, device="cuda")
    n = 12
    g = torch.Generator(device="cuda").manual_seed(3)
    kv[-n:] = torch.randint(-127, 128, kv[-n:].shape, dtype=torch.int8, device="cuda", generator=g)
    small_kv, small_sc = kv[-n:].clone(), sc[-n:].clone()
    q = bf16(g, 40, 16 * 128)
    for counts, lens in (([3, 2], [100, 90]), ([37, 3], [100, 90])):
        rows = sum(counts)
        pos = i32([l - c + i for l, c in zip(lens, counts) for i in range(c)])
        out = torch.zeros(2, rows, 16 * 128, dtype=torch.bfloat16, device="cuda")
        for i, (k, s, first) in enumerate(((kv, sc, blocks - n), (small_kv, small_sc, 0))):
            mp = oa.extend_plan(counts, 16, hk, 100, lens, 64)
            pages = i32([first + x for x in (7, 3, 11, 0, 9, 1, 2, 4, 5, 6, 8, 10, 11)])
            oa.qwen3_extend_q8(mp, q, k, s, pos, i32([0, 7, 13]), pages, 16, out[i], SCALE, oa.workspace_for(mp.plan))
        torch.cuda.synchronize()
        assert torch.equal(out[0], out[1]) and bool(out[0].any())


def test_cross_past_32_bits():
    """Sources behind 5 GiB of k and v rows."""
    hk, total, n = 8, 1_250_000, 300
    kv = torch.zeros(total, 2 * hk * 128, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(3)
    kv[-n:] = bf16(g, n, 2 * hk * 128)
    small = kv[-n:].clone()
    q = bf16(g, 40, 16 * 128)
    for counts in ([3, 2], [37, 3]):
        rows = sum(counts)
        out = torch.zeros(2, rows, 16 * 128, dtype=torch.bfloat16, device="cuda")
        for i, (x, first) in enumerate(((kv, total - n), (small, 0))):
            mp = oa.cross_plan(counts, 16, hk, 200, [200, 100], 64)
            oa.cross_run(mp, q, x[:, :hk * 128], x[:, hk * 128:], None, i32([first, first + 200]), i32([200, 100]), out[i], SCALE,
                         oa.workspace_for(mp.plan))
        torch.cuda.synchronize()
        assert torch.equal(out[0], out[1]) and bool(out[0].any())


# ------------------------------------------------------------------ graphs
def test_two_graphs_with_workspaces_of_their_own():
    """Extend and cross captured together, twice; lengths and positions move on between replays, eager work in between."""
    hq, hk, lens, counts = 8, 2, [1400, 90, 33], [40, 20, 2]
    c = Cache(21, lens, hk, 16, torch.float8_e4m3fn)
    g = torch.Generator(device="cuda").manual_seed(4)
    rows = sum(counts)
    q = bf16(g, rows, hq * 128)
    kv = bf16(g, 500, 2 * hk * 128)
    k, v = kv[:, :hk * 128], kv[:, hk * 128:]
    start = [max(n - m + i - 30, -1) for n, m in zip(lens, counts) for i in range(m)]
    pos, first, length = i32(start), i32([0, 200, 333]), i32([150, 3, 0])

    def make():
        e, x = oa.extend_plan(counts, hq, hk, 1400, lens, 64), oa.cross_plan(counts, hq, hk, 1200, None, 64)
        assert e.plan.split_tiles > 0 and x.plan.split_tiles > 0 and e.plan.splits > 1 and e.plan.groups[0] > 0 and x.plan.tiles > 0
        return e, oa.workspace_for(e.plan), x, oa.workspace_for(x.plan), torch.zeros(2, rows, hq * 128, dtype=torch.bfloat16, device="cuda")

    def step(m, s=None):
        oa.qwen3_extend_q8(m[0], q, c.kv, c.sc, pos, c.indptr, c.pages, 16, m[4][0], SCALE, m[1], s)
        oa.cross_run(m[2], q, k, v, None, first, length, m[4][1], SCALE, m[3], s)

    sets = [make() for _ in range(3)]
    torch.cuda.synchronize()
    graphs, s = [], torch.cuda.Stream()
    for m in sets[1:]:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=s):
            step(m)
    for rep in range(12):
        step(sets[0])
        torch.cuda.synchronize()
        for gr, m in zip(graphs, sets[1:]):
            m[4].zero_()
            gr.replay()
        torch.cuda.synchronize()
        for m in sets[1:]:
            assert torch.equal(m[4], sets[0][4]), rep
        pos += 2
        length += i32([3, 7, 11])
