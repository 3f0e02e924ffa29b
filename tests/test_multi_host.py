"""Plans of extend and cross attention, and what the calls refuse before any launch (CPU)."""
import ctypes
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import omni_attn as oa

P = 4096  # stands for a device pointer: nothing is launched
PLANS = [oa.extend_plan, oa.cross_plan]


def groups_of(mp):
    n0, n1 = mp.plan.groups
    skip = mp.plan.work_bytes // 4 - 4 * (n0 + n1)
    it = mp.work.numpy()[skip:skip + 4 * (n0 + n1)].reshape(-1, 4)
    return it[:n0], it[n0:]


@pytest.mark.parametrize("make", PLANS)
@pytest.mark.parametrize("hq,hk", [(3, 1), (5, 1), (10, 2), (9, 1), (15, 1), (12, 1), (16, 1), (7, 7), (8, 2)])
def test_groups_cover_every_row_once(make, hq, hk):
    g = hq // hk
    counts = [0, 1, 16 // g, 16 // g + 1, 32 // g, 2, 0, 3]
    if g > 8:
        counts += [32 // g + 1, 100]
    mp = make(counts, hq, hk, 500, device="cpu")
    starts = np.cumsum([0] + counts)
    seen = np.zeros(sum(counts), int)
    at = 0
    for cols, list_ in zip((16, 32), groups_of(mp)):
        for s, first, rows, ws in list_:
            assert starts[s] <= first and first + rows <= starts[s + 1] and 1 <= rows and rows * g <= cols and ws == at
            seen[first:first + rows] += 1
            at += rows
    assert (seen == 1).all() and mp.plan.group_rows == at == mp.plan.rows == sum(counts)


@pytest.mark.parametrize("make", PLANS)
def test_long_sequences_come_first(make):
    mp = make([1, 1, 4, 1], 4, 4, 900, [5, 800, 20, 300], device="cpu")
    assert groups_of(mp)[0][:, 0].tolist() == [1, 3, 2, 0]


@pytest.mark.parametrize("make", PLANS)
def test_plan_bounds(make):
    for counts, keys, hq, hk, n, chunk, code in (
            ([-1], None, 4, 2, 9, 0, oa.EINVAL), ([1], [-1], 4, 2, 9, 0, oa.EINVAL), ([1], [1, 2], 4, 2, 9, 0, oa.EINVAL),
            ([1], None, 5, 2, 9, 0, oa.EINVAL), ([1], None, 0, 1, 9, 0, oa.EINVAL), ([1], None, 4, 0, 9, 0, oa.EINVAL),
            ([1], None, 4, 2, 0, 0, oa.EINVAL), ([1], None, 4, 2, 9, 65, oa.EINVAL), ([1], None, 17, 1, 9, 0, oa.EUNSUPPORTED),
            ([2**31 - 1, 2**31 - 1], None, 1, 1, 9, 0, oa.EUNSUPPORTED),
            ([2**31 - 1] * 3, None, 2**31 - 1, 2**31 - 1, 9, 0, oa.EUNSUPPORTED)):
        with pytest.raises(oa.OmniAttnError) as e:
            make(counts, hq, hk, n, keys, chunk, device="cpu")
        assert e.value.code == code, (counts, hq, hk)
    mp = make([], 4, 2, 9, device="cpu")
    assert mp.plan.rows == 0 and mp.plan.work_bytes == 0 and mp.plan.workspace_bytes == 0


@pytest.mark.parametrize("make", PLANS)
def test_a_bound_that_bounds_nothing(make):
    for counts in ([1], [1, 0, 8], [40], [300, 2]):
        p = make(counts, 4, 1, 2**31 - 1, device="cpu").plan
        assert p.rows == sum(counts) and p.splits >= 1 and p.tile_chunk > 0


@pytest.mark.parametrize("init", ["omni_attn_extend_plan_init", "omni_attn_cross_plan_init"])
def test_plan_capacity(init):
    f, plan = getattr(oa.load(), init), oa.MultiPlan()
    counts, work = np.array([3, 1], np.int32), np.zeros(8, np.int32)
    ptr = lambda a: a.ctypes.data_as(ctypes.c_void_p)
    assert f(2, ptr(counts), None, 4, 2, 50, 0, ptr(work), 7, ctypes.byref(plan)) == oa.EWORKSPACE and plan.work_bytes == 32
    assert f(2, ptr(counts), None, 4, 2, 50, 0, None, 99, ctypes.byref(plan)) == oa.EWORKSPACE
    assert f(2, ptr(counts), None, 4, 2, 50, 0, ptr(work), 8, ctypes.byref(plan)) == oa.OK
    assert f(2, None, None, 4, 2, 50, 0, ptr(work), 8, ctypes.byref(plan)) == oa.EINVAL
    assert f(-1, ptr(counts), None, 4, 2, 50, 0, ptr(work), 8, ctypes.byref(plan)) == oa.EINVAL
    assert f(2, ptr(counts), None, 4, 2, 50, 0, ptr(work), 8, None) == oa.EINVAL


@pytest.mark.parametrize("make", PLANS)
def test_splits_follow_the_chunk(make):
    mp = make([1, 2], 4, 2, 1000, None, 128, device="cpu")
    p = mp.plan
    assert (p.chunk, p.splits) == (128, 8) and p.workspace_bytes == 3 * 4 * 8 * 129 * 4 + 16  # partials, and the splits of two groups
    assert make([1, 2], 4, 2, 1000, None, 1024, device="cpu").plan.workspace_bytes == 0


def extend(plan=None, **k):
    plan = plan or oa.extend_plan([3, 2], 4, 2, 100, chunk=128, device="cpu").plan
    a = dict(plan=ctypes.byref(plan), q=P, stride=512, kv=P, scale=P, fmt=0, pos=P, indptr=P, pages=P, page=16, out=P, s=0.1, work=P, ws=None)
    a.update(k)
    if a.pop("plan_", None):
        a["plan"] = None
    return oa.load().omni_qwen3_extend_q8(*a.values(), None)


def cross(plan=None, **k):
    plan = plan or oa.cross_plan([3, 2], 4, 2, 100, chunk=128, device="cpu").plan
    a = dict(plan=ctypes.byref(plan), q=P, stride=512, k=P, ks=256, v=P, vs=256, of=P, first=P, len=P, out=P, s=0.1, work=P, ws=None)
    a.update(k)
    if a.pop("plan_", None):
        a["plan"] = None
    return oa.load().omni_attn_cross_run(*a.values(), None)


BAD = [dict(q=None), dict(out=None), dict(work=None), dict(q=P + 8), dict(out=P + 8), dict(work=P + 4), dict(stride=504), dict(stride=516),
       dict(s=float("nan")), dict(s=3e38), dict(ws=P + 8)]


@pytest.mark.parametrize("bad", BAD + [
    dict(fmt=2), dict(fmt=-1), dict(kv=None), dict(scale=None), dict(pos=None), dict(indptr=None), dict(pages=None), dict(kv=P + 8), dict(page=0)])
def test_extend_refusals(bad):
    assert extend(**bad) == oa.EINVAL
    assert b"extend" in oa.load().omni_attn_last_error()


@pytest.mark.parametrize("bad", BAD + [
    dict(k=None), dict(v=None), dict(first=None), dict(len=None), dict(k=P + 8), dict(v=P + 2), dict(ks=248), dict(vs=260), dict(ks=(1 << 22) + 8)])
def test_cross_refusals(bad):
    assert cross(**bad) == oa.EINVAL
    assert b"cross" in oa.load().omni_attn_last_error()


def test_other_codes():
    assert extend(plan_=1) == oa.EINVAL and cross(plan_=1) == oa.EINVAL
    assert extend(page=24) == oa.EUNSUPPORTED
    split = oa.extend_plan([3, 2], 4, 2, 100, chunk=64, device="cpu").plan
    assert extend(split) == oa.EWORKSPACE
    split = oa.cross_plan([3, 2], 4, 2, 100, chunk=64, device="cpu").plan
    assert cross(split) == oa.EWORKSPACE
    none = oa.cross_plan([0], 4, 2, 100, device="cpu").plan
    assert cross(none, q=None, k=None, out=None, work=None) == oa.OK
    none = oa.extend_plan([0], 4, 2, 100, device="cpu").plan
    assert extend(none, q=None, kv=None, out=None, work=None) == oa.OK
    # Each call takes its own plans.
    assert extend(oa.cross_plan([3], 4, 2, 100, device="cpu").plan) == oa.EINVAL
    assert cross(oa.extend_plan([3], 4, 2, 100, device="cpu").plan) == oa.EINVAL


@pytest.mark.parametrize("field,value", [
    ("rows", -1), ("hq", 5), ("hq", 0), ("hk", 0), ("hq", 64), ("max_len", 0), ("max_len", 300), ("group_rows", -1), ("group_rows", 6), ("chunk", 0),
    ("chunk", 65), ("splits", 2), ("splits", 0), ("tiles", -1), ("tiles", 1), ("tile_chunk", 0), ("tile_chunk", 64), ("tile_units", 3), ("split_tiles", 1), ("tile_segments", 2), ("work_bytes", 0),
    ("workspace_bytes", 16)])
def test_plans_that_do_not_agree(field, value):
    for make, call in ((oa.extend_plan, extend), (oa.cross_plan, cross)):
        plan = make([3, 2], 4, 2, 100, chunk=128, device="cpu").plan
        setattr(plan, field, value)
        assert call(plan) == oa.EINVAL, field
    for at in (0, 1):
        plan = oa.cross_plan([3, 2], 4, 2, 100, chunk=128, device="cpu").plan
        plan.groups[at] += 1
        assert cross(plan) == oa.EINVAL
        plan.groups[at] = -1
        assert cross(plan) == oa.EINVAL


def test_the_mirror_refuses_host_tensors_and_other_shapes():
    b = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)
    z = torch.zeros(8, dtype=torch.int32)
    kv, sc = oa.q8_cache(4, 16, 2, device="cpu")
    e, x = oa.extend_plan([3], 4, 2, 50, device="cpu"), oa.cross_plan([3], 4, 2, 50, device="cpu")
    for call in (lambda: oa.qwen3_extend_q8(e, b(3, 512), kv, sc, z, z, z, 16, b(3, 512), 0.1),
                 lambda: oa.cross_run(x, b(3, 512), b(9, 256), b(9, 256), z, z, z, b(3, 512), 0.1)):
        with pytest.raises(oa.OmniAttnError) as err:
            call()
        assert err.value.code == oa.EINVAL


def test_launches_that_no_grid_holds():
    for make in PLANS:
        with pytest.raises(oa.OmniAttnError) as e:
            make([1] * 3000, 128, 128, 64 * 100000, None, 64, device="cpu")
        assert e.value.code == oa.EUNSUPPORTED


def tile_items(mp):
    p = mp.plan
    work = mp.work.numpy()
    n = 16 + 8 * p.tile_units * p.hk
    return work[:16], work[16:n].reshape(-1, 8), work[n:n + 4 * p.split_tiles * p.hk].reshape(-1, 4)


def check_tiles(mp, counts, keys, causal):
    """Every row of a sequence in tiles once for each split of its tile and each head; segments and the combine's list agree."""
    p = mp.plan
    g = p.hq // p.hk
    starts = np.cumsum([0] + counts)
    if p.tiles == 0:
        ranges, items, split = [0] * 9, [], []
    else:
        ranges, items, split = tile_items(mp)
    assert ranges[0] == 0 and ranges[8] == len(items) == p.tile_units * p.hk and np.ptp(np.diff(ranges[:9])) <= 1
    seen, segments, which = {}, {}, {}
    for s, first, rows, head, k, n, seg, at in items:
        assert (counts[s] > 32 // g or p.group_rows == 0) and starts[s] <= first and first + rows <= starts[s + 1] and 1 <= rows <= 256 // g
        assert (first - starts[s]) % (256 // g) == 0 and 0 <= k < n
        last = min(max(keys[s] - (starts[s + 1] - first - rows if causal else 0), 0), p.max_len)
        assert n == max(1, -(-last // p.tile_chunk))
        seen.setdefault((first, rows, head, n), []).append(k)
        if n > 1:
            assert segments.setdefault(seg, (first, head, k)) == (first, head, k) and 0 <= seg < p.tile_segments * p.hk
            assert tuple(split[at]) == (first, rows + 512 * n, head, seg - k)
            which[at] = True
    assert all(sorted(ks) == list(range(n)) for (_, _, _, n), ks in seen.items())
    covered = np.zeros((sum(counts), p.hk), int)
    for first, rows, head, _ in seen:
        covered[first:first + rows, head] += 1
    for list_ in groups_of(mp):
        for s, first, rows, _ in list_:
            covered[first:first + rows] += 1
    assert (covered == 1).all() and len(segments) == p.tile_segments * p.hk and len(which) == p.split_tiles * p.hk
    # An XCD's splits run longest first.
    for x in range(8):
        def cost(i):
            s, first, rows, _, k, n = i[:6]
            last = min(max(keys[s] - (starts[s + 1] - first - rows if causal else 0), 0), p.max_len)
            steps = max(1, -(-last // 128))
            return (2.4 if rows * g <= 128 else 3.9) * min(p.tile_chunk // 128, steps - k * (p.tile_chunk // 128))
        costs = [cost(i) for i in items[ranges[x]:ranges[x + 1]]]
        assert costs == sorted(costs, reverse=True)


@pytest.mark.parametrize("make", PLANS)
@pytest.mark.parametrize("hq,hk", [(1, 1), (8, 4), (8, 2), (16, 2), (3, 3), (3, 1), (10, 2), (6, 1), (14, 2), (16, 1)])
def test_tiles_and_groups_cover_every_row_once(make, hq, hk):
    g = hq // hk
    counts = [1, 32 // g, 32 // g + 1, 0, 256 // g, 256 // g + 1, 1000, 2]
    for reach in (160, 9000):
        keys = [c + reach + 13 * i for i, c in enumerate(counts)]
        mp = make(counts, hq, hk, max(keys) - 5, keys, device="cpu")
        check_tiles(mp, counts, keys, make is oa.extend_plan)
        assert mp.plan.group_rows == 0 and mp.plan.tiles == sum(-(-c // (256 // g)) for c in counts)  # few keys: all of them tiles
        for chunk in (0, 512):
            mp = make(counts, hq, hk, 500, None, chunk, device="cpu")  # lengths not known: the longest
            check_tiles(mp, counts, [500] * len(counts), make is oa.extend_plan)
        # With a chunk, by their rows.
        assert mp.plan.group_rows == sum(c for c in counts if c <= 32 // g) and all(mp.plan.groups)
        assert mp.plan.tiles == sum(-(-c // (256 // g)) for c in counts if c > 32 // g)


@pytest.mark.parametrize("make", PLANS)
@pytest.mark.parametrize("hq,hk", [(1, 1), (8, 2), (16, 2)])
def test_calls_that_mix_run_in_one_kernel_where_keys_are_few(make, hq, hk):
    g = hq // hk
    small, large, tall = 16 // g, 32 // g, 32 // g + 1
    tiles = lambda counts: sum(-(-c // (256 // g)) for c in counts)

    def plan(counts, reach):
        keys = [max(reach - 3 * (i % 5), 0) for i in range(len(counts))]
        mp = make(counts, hq, hk, reach, keys, device="cpu")
        check_tiles(mp, counts, keys, make is oa.extend_plan)
        return mp.plan.tiles, list(mp.plan.groups)

    mixed = [small, large, 0, tall, 1]
    assert plan(mixed, 1152) == (0, [0, 5])                                  # groups of 32: a CU gets one at most
    assert plan(mixed, 1153) == (4, [0, 0])                                  # tiles
    assert plan([300 * 32 // g] + mixed, 1152) == (tiles([300 * 32 // g] + mixed), [0, 0])  # more groups than CUs
    assert plan([257 * 256 // g] + mixed, 1153) == (tiles([257 * 256 // g, tall]), [0, 3])  # more tiles than CUs
    assert plan([small, large], 1153) == (0, [0, 2])
    assert plan([small, 1], 1153) == (0, [2, 0])
    # Many keys: what is no tile as groups.
    limit = 128_000_000 // 256 if make is oa.extend_plan else 2_000_000_000 // 512
    assert plan(mixed, limit // (3 * hk) - 100) == (4, [0, 0])
    assert plan(mixed, limit // (3 * hk) + 100) == (1, [0, 3])
    assert plan([small, 1], limit // hk) == (0, [2, 0])


@pytest.mark.parametrize("make", PLANS)
def test_tiles_are_split_where_they_are_few(make):
    few = make([100], 4, 1, 30000, device="cpu").plan
    assert few.tiles == few.split_tiles == 2 and few.tile_units > 32 and few.tile_segments == few.tile_units
    assert few.workspace_bytes >= few.tile_units * 256 * 130 * 4
    many = make([2000] * 8, 32, 8, 30000, device="cpu").plan
    assert many.tile_units == many.tiles and many.split_tiles == many.workspace_bytes == 0
    short = make([100], 4, 1, 200, device="cpu").plan
    assert short.split_tiles == 0  # not worth it
    # Tiles of unlike lengths: the long ones are split.
    p = make([60, 60, 60], 4, 4, 20000, [20000, 300, 0], device="cpu").plan
    assert 1 <= p.split_tiles < p.tiles


@pytest.mark.parametrize("field,by", [("tile_units", 1), ("tile_units", -1), ("split_tiles", 1), ("split_tiles", -1), ("tile_segments", 1),
                                      ("tile_segments", -1), ("tile_chunk", 64), ("workspace_bytes", -16), ("work_bytes", 4)])
def test_plans_of_tiles_that_do_not_agree(field, by):
    for make, call in ((oa.extend_plan, extend), (oa.cross_plan, cross)):
        plan = make([100, 3], 4, 2, 30000, device="cpu").plan
        assert plan.split_tiles > 0
        setattr(plan, field, getattr(plan, field) + by)
        assert call(plan, ws=P) == oa.EINVAL


NO_MEMORY = """
import ctypes, resource, sys
import numpy as np
import omni_attn as oa
L = oa.load()
p = lambda a: a.ctypes.data_as(ctypes.c_void_p)
f = getattr(L, "omni_attn_%s_plan_init" % sys.argv[1])
counts, plan = np.full(1 << 21, 3, np.int32), oa.MultiPlan()
work = np.zeros(4 << 21, np.int32)
size = int(open("/proc/self/statm").read().split()[0]) * resource.getpagesize() + (4 << 20)
resource.setrlimit(resource.RLIMIT_AS, (size, size))
rc = f(len(counts), p(counts), None, 3, 1, 100, 0, p(work), len(work), ctypes.byref(plan))
assert rc == oa.EUNSUPPORTED and b"memory" in L.omni_attn_last_error(), rc
print("refused")
"""


@pytest.mark.parametrize("which", ["extend", "cross"])
def test_plans_without_host_memory_return_an_error(which):
    """The groups of two million sequences (32 MiB) are host memory; where there is none the C call says so, and throws nothing."""
    here = os.path.dirname(oa.__file__)
    r = subprocess.run([sys.executable, "-c", NO_MEMORY, which], capture_output=True, text=True, env={**os.environ, "PYTHONPATH": here})
    assert r.returncode == 0 and "refused" in r.stdout, (r.returncode, r.stderr[-500:])


@pytest.mark.parametrize("make", PLANS)
def test_counts_that_no_grid_holds_are_refused_before_their_lists_are_made(make):
    for counts, hq, hk in (([2**31 - 1], 3, 1), ([2**31 - 1], 4, 4), ([10**8], 12, 1), ([1] * 70000, 512, 512)):
        with pytest.raises(oa.OmniAttnError) as e:
            make(counts, hq, hk, 100, device="cpu")
        assert e.value.code == oa.EUNSUPPORTED


def test_the_mirrors_plan_is_the_headers(tmp_path):
    fields = [f[0] for f in oa.MultiPlan._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "omni_attn.h"\nint main(void) {\n  printf("%zu", sizeof(omni_attn_multi_plan));\n'
                   + "".join(f'  printf(" %zu", offsetof(omni_attn_multi_plan, {f}));\n' for f in fields) + "  return 0;\n}\n")
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    exe = str(tmp_path / "layout")
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I" + include, str(src), "-o", exe], check=True)
    got = [int(x) for x in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(oa.MultiPlan)] + [getattr(oa.MultiPlan, f).offset for f in fields]
