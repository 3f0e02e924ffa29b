"""A plan's exact_p for several rows per sequence: P in 16 bits in tiles as in groups, against 64 bits under the bound of
groups (2^-8 of the result, for its rounding to bf16, and 2^-13 of sum p |v|), whichever kernel the plan takes."""
import numpy as np
import pytest
import torch

import omni_attn as oa
import test_multi_gpu as T
from test_multi_host import cross as cross_call, extend as extend_call

MANY = 1 << 14


@pytest.mark.parametrize("make,call", [(oa.extend_plan, extend_call), (oa.cross_plan, cross_call)])
def test_the_field(make, call):
    mp = make([40, 2], 4, 2, 100, chunk=128, device="cpu")
    assert mp.plan.exact_p == 0 and mp.plan.tiles > 0
    assert make([40, 2], 4, 2, 100, chunk=128, device="cpu", exact_p=True).plan.exact_p == 1
    for bad in (2, -1):
        mp.plan.exact_p = bad
        assert call(mp.plan) == oa.EINVAL and b"exact_p" in oa.load().omni_attn_last_error()


def exactly(monkeypatch):
    """The calls of test_multi_gpu with plans that carry P in 16 bits, held to the bound of groups."""
    for name in ("extend_plan", "cross_plan"):
        plain = getattr(oa, name)
        monkeypatch.setattr(oa, name, lambda *a, _p=plain, **k: _p(*a, **k, exact_p=True))
    bound = T.M.bound
    monkeypatch.setattr(T.M, "bound", lambda want, size, tiles: bound(want, size, False))


LAYOUTS = [(1, 1), (4, 2), (8, 2), (16, 2), (3, 1), (10, 2), (6, 1), (14, 2), (16, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", T.FORMATS)
@pytest.mark.parametrize("hq,hk", LAYOUTS)
def test_extend(hq, hk, fmt, monkeypatch):
    """Whole tiles beside groups, unsplit; the same rows with the choice left to the plan."""
    exactly(monkeypatch)
    g = hq // hk
    counts = [32 // g + 1, 64 // g + 3, 256 // g, 1, 256 // g + 1, 0, 2]
    lens = [counts[0], 129, 256 // g, 70, 256 // g + 128, 5, 300]
    for chunk in (MANY, 0):
        mp, _ = T.extend(T.Cache(hq, lens, hk, 16, fmt), counts, hq, chunk=chunk)
        assert mp.plan.exact_p == 1 and (mp.plan.tiles > 0 or chunk == 0)


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hk", LAYOUTS)
def test_cross(hq, hk, monkeypatch):
    exactly(monkeypatch)
    g = hq // hk
    counts = [32 // g + 1, 64 // g + 3, 256 // g, 1, 256 // g + 1, 0, 2, 40]
    for chunk in (MANY, 0):
        mp, _ = T.cross(hq, counts, [1, 129, 128, 70, 257, 5, 300, 0], hq, hk, chunk=chunk)
        assert mp.plan.exact_p == 1 and (mp.plan.tiles > 0 or chunk == 0)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", T.FORMATS)
@pytest.mark.parametrize("seqs,hk,g", [(1, 2, 2), (12, 8, 2), (20, 16, 2), (1, 1, 16), (4, 4, 16), (12, 8, 16)])
def test_every_form_of_a_tile(seqs, hk, g, fmt, monkeypatch):
    exactly(monkeypatch)
    rng = np.random.default_rng(seqs)
    counts = [int(x) for x in rng.integers(34, 130, seqs)]
    lens = [c + int(x) for c, x in zip(counts, rng.integers(0, 260, seqs))]
    mp, _ = T.extend(T.Cache(seqs, lens, hk, 16, fmt), counts, g * hk, chunk=MANY)
    assert mp.plan.tiles >= seqs and mp.plan.split_tiles == 0
    if fmt == torch.int8:
        T.cross(seqs, counts, [int(x) for x in rng.integers(0, 300, seqs)], g * hk, hk, chunk=MANY)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", T.FORMATS)
@pytest.mark.parametrize("hq,hk", [(4, 1), (2, 2), (5, 1), (16, 1)])
def test_tiles_in_splits(hq, hk, fmt, monkeypatch):
    exactly(monkeypatch)
    c = T.Cache(hq, [2600, 700, 90], hk, 16, fmt)
    mp, _ = T.extend(c, [70, 40, 40], hq, chunk=MANY)
    assert mp.plan.split_tiles > 0
    pos = [2599 - 37 * i if i % 3 else -1 for i in range(70)] + [i for i in range(40)] + [-1] * 40
    T.extend(c, [70, 40, 40], hq, pos=pos, seed=4, chunk=MANY)
    mp, _ = T.cross(6, [70, 40, 40, 50], [2600, 700, 90, 0], hq, hk, chunk=MANY)
    assert mp.plan.split_tiles > 0


@pytest.mark.gpu
def test_rows_of_groups_keep_their_bits():
    """exact_p changes nothing where no row runs in a tile."""
    c = T.Cache(3, [500, 70], 2, 16, torch.float8_e4m3fn)
    outs = []
    for exact in (False, True):
        q = T.bf16(torch.Generator(device="cuda").manual_seed(1), 5, 8 * 128)
        out = torch.zeros_like(q)
        mp = oa.extend_plan([3, 2], 8, 2, 500, chunk=64, exact_p=exact)
        assert mp.plan.tiles == 0
        oa.qwen3_extend_q8(mp, q, c.kv, c.sc, T.i32([497, 498, 499, 68, 69]), c.indptr, c.pages, 16, out, T.SCALE, oa.workspace_for(mp.plan))
        torch.cuda.synchronize()
        outs.append(out)
    assert torch.equal(*outs)


@pytest.mark.gpu
def test_in_graphs_beside_a_plan_that_rounds():
    """Extend and cross with exact_p captured, with groups and split tiles, replayed as positions move on, beside eager calls of both kinds
    on other streams with workspaces of their own."""
    hq, hk, lens, counts = 8, 2, [1400, 90, 33], [40, 20, 2]
    c = T.Cache(21, lens, hk, 16, torch.float8_e4m3fn)
    g = torch.Generator(device="cuda").manual_seed(4)
    rows = sum(counts)
    q, kv = T.bf16(g, rows, hq * 128), T.bf16(g, 500, 2 * hk * 128)
    k, v = kv[:, :hk * 128], kv[:, hk * 128:]
    pos = T.i32([max(n - m + i - 30, -1) for n, m in zip(lens, counts) for i in range(m)])
    first, length = T.i32([0, 200, 333]), T.i32([150, 3, 0])

    def make(exact):
        e, x = (f(counts, hq, hk, 1400, None, 64, exact_p=exact) for f in (oa.extend_plan, oa.cross_plan))
        assert e.plan.split_tiles > 0 and x.plan.split_tiles > 0 and e.plan.group_rows > 0
        return e, oa.workspace_for(e.plan), x, oa.workspace_for(x.plan), torch.zeros(2, rows, hq * 128, dtype=torch.bfloat16, device="cuda")

    def step(m, s=None):
        oa.qwen3_extend_q8(m[0], q, c.kv, c.sc, pos, c.indptr, c.pages, 16, m[4][0], T.SCALE, m[1], s)
        oa.cross_run(m[2], q, k, v, None, first, length, m[4][1], T.SCALE, m[3], s)

    eager, captured, rounded, other = make(True), make(True), make(False), make(False)
    torch.cuda.synchronize()
    s, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        step(captured)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for rep in range(8):
        step(eager)
        step(rounded)
        torch.cuda.synchronize()
        for m in (captured, other):
            m[4].zero_()
        torch.cuda.synchronize()
        graph.replay()
        step(other, streams[0])
        step(eager, streams[1])
        torch.cuda.synchronize()
        assert torch.equal(captured[4], eager[4]) and torch.equal(other[4], rounded[4]), rep
        assert not torch.equal(captured[4], rounded[4])
        pos += 2
        length += T.i32([3, 7, 11])
