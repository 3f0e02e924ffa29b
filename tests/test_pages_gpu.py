"""Pages that requests share, on the GPU: fork, free, compact and copy against host
loops, with equal bits (the results are whole numbers and bytes); what they refuse
on the device; and a server of forked requests that are given back and compacted."""
import numpy as np
import pytest
import torch

import omni_attn as oa
import pages_refs as R

pytestmark = pytest.mark.gpu


def i32(a):
    return torch.from_numpy(np.array(a, dtype=np.int32).copy()).cuda()


def host(t):
    return t.cpu().numpy().astype(np.int64)


class Pool:
    """A table of requests of the given lengths, their pages anywhere in the pool, the free ones anywhere in the queue."""

    def __init__(self, rng, lens, page, spare, more_lines=0, width=None):
        self.page, self.lens = page, list(lens)
        held = [-(-n // page) for n in lens]
        self.total = max(1, sum(held) + spare)
        ids = rng.permutation(self.total)
        self.lines = [int(x) for x in rng.permutation(len(lens) + more_lines)]
        self.table = np.full((len(lens) + more_lines, width or max(held + [0]) + 2), -1, np.int64)
        at = 0
        for line, n in zip(self.lines, held):
            self.table[line, :n] = ids[at:at + n]
            at += n
        self.avail = self.total - at
        self.head = int(rng.integers(self.total))
        self.free = np.full(self.total, -1, np.int64)
        for k, p in enumerate(ids[at:]):
            self.free[(self.head + k) % self.total] = p
        self.shares = np.zeros(self.total, np.int64)
        self.state = [self.head, self.avail]

    def upload(self):
        self.d = {n: i32(getattr(self, n)) for n in ("table", "free", "shares", "state")}
        return self.d

    def same(self):
        for n in ("table", "free", "shares"):
            assert np.array_equal(host(self.d[n]), getattr(self, n)), n


def fork(pool, parents, children, tokens, stream=None):
    d, n = pool.d, len(tokens)
    src, dst, status = i32([7] * n), i32([7] * n), i32([9] * 5)
    oa.pages_fork(i32(parents), i32(children), i32(tokens), d["table"], d["free"], d["state"], d["shares"], src, dst, status, pool.page, stream)
    torch.cuda.synchronize()
    want = R.fork(parents, children, tokens, pool.page, pool.table, pool.free, pool.state, pool.shares)
    assert [src.tolist(), dst.tolist(), status.tolist()] == [list(want[0]), list(want[1]), [int(x) for x in want[2]]]
    pool.same()
    pool.state, d["state"] = want[2][3:], status[3:5]
    return want


def give_back(pool, lines, tokens):
    d = pool.d
    status = i32([9] * 5)
    oa.pages_free(i32(lines), i32(tokens), d["table"], d["free"], d["state"], d["shares"], status, pool.page)
    torch.cuda.synchronize()
    want = R.give_back(lines, tokens, pool.page, pool.table, pool.free, pool.state, pool.shares)
    assert status.tolist() == [int(x) for x in want]
    pool.same()
    pool.state, d["state"] = want[3:], status[3:5]
    return want


@pytest.mark.parametrize("page", [1, 16, 24, 256])
@pytest.mark.parametrize("parents,each,hi", [(1, 1, 1), (1, 8, 187), (5, 3, 40), (32, 7, 700), (3, 300, 33)])
def test_fork_and_free(page, parents, each, hi):
    rng = np.random.default_rng(parents * 1000 + page)
    n = parents * each
    pool = Pool(rng, rng.integers(0, hi + 1, parents), page, n + 3, n)
    pool.upload()
    par = [pool.lines[i // each] for i in range(n)]
    chi = pool.lines[parents:]
    tok = [int(rng.integers(0, pool.lens[i // each] + 1)) if i % 3 else pool.lens[i // each] for i in range(n)]
    for i in range(0, n, 5):
        tok[i] = -1 if n > 5 else tok[i]
    assert fork(pool, par, chi, tok)[2][0] == 0
    # Some children end, then the parents, then the other children: a page leaves with its last holder.
    first, rest = list(range(0, n, 2)), list(range(1, n, 2))
    assert give_back(pool, [chi[i] for i in first], [tok[i] for i in first])[0] == 0
    assert give_back(pool, pool.lines[:parents], pool.lens)[0] == 0
    if rest:
        assert give_back(pool, [chi[i] for i in rest], [tok[i] for i in rest])[0] == 0
    assert pool.state[1] == pool.total and (pool.shares == 0).all()
    assert sorted(pool.free.tolist()) == list(range(pool.total))


def test_one_call_takes_all_holders_of_a_page():
    """A parent and its children end in one call: each page comes free once."""
    rng = np.random.default_rng(4)
    pool = Pool(rng, [100], 16, 9, 6)
    pool.upload()
    fork(pool, [pool.lines[0]] * 6, pool.lines[1:], [100, 64, 16, 15, 0, 96])
    status = give_back(pool, pool.lines, [100, 100, 64, 16, 15, 0, 96])
    assert status[0] == 0 and pool.state[1] == pool.total


def test_a_child_of_a_child():
    rng = np.random.default_rng(5)
    pool = Pool(rng, [50], 16, 12, 3)
    pool.upload()
    a, b, c, e = pool.lines
    fork(pool, [a], [b], [50])
    fork(pool, [b, b], [c, e], [50, 33])
    assert pool.shares.max() == 3
    give_back(pool, [b, a], [50, 50])
    give_back(pool, [e, c], [33, 50])
    assert pool.state[1] == pool.total


@pytest.mark.parametrize("parents,children,tokens,state,code", [
    ([0, 0], [1, 1], [5, 5], None, 1), ([0, 1], [1, 2], [5, 5], None, 1), ([0], [0], [5], None, 1), ([-1], [1], [5], None, 1),
    ([0], [9], [5], None, 1), ([9], [1], [5], None, 1), ([0], [1], [81], None, 4), ([0, 0, 0], [1, 2, 3], [5, 5, 5], [0, 2], 5),
    ([0], [1], [5], [0, 999], 1), ([0], [1], [5], [-1, 2], 1), ([0], [9], [-1], None, 0), ([0], [1], [64], [0, 0], 0)])
def test_forks_that_cannot_be_made_change_nothing(parents, children, tokens, state, code):
    pool = Pool(np.random.default_rng(1), [70, 20], 16, 8, 4, width=5)
    pool.lines = list(range(6))
    if state:
        pool.state = state
    before = pool.table.copy()
    pool.upload()
    assert fork(pool, parents, children, tokens)[2][0] == code
    if code:
        assert np.array_equal(pool.table, before)


@pytest.mark.parametrize("lines,tokens,state,code", [
    ([0, 0], [5, 5], None, 1), ([9], [5], None, 1), ([-2], [5], None, 1), ([0], [99], None, 4), ([0], [5], [0, -1], 1), ([9], [-1], None, 0),
    ([0], [0], None, 0)])
def test_frees_that_cannot_be_made_change_nothing(lines, tokens, state, code):
    pool = Pool(np.random.default_rng(2), [70, 20], 16, 8, 4, width=5)
    if state:
        pool.state = state
    pool.upload()
    assert give_back(pool, lines, tokens)[0] == code


def test_pages_that_nobody_holds():
    """A line that is given back twice: the queue holds more pages than were in use."""
    pool = Pool(np.random.default_rng(3), [70], 16, 2, 0)
    pool.upload()
    assert give_back(pool, [pool.lines[0]], [70])[0] == 0
    assert give_back(pool, [pool.lines[0]], [70])[0] == 6


def test_page_ids_outside_the_pool_are_passed_over():
    pool = Pool(np.random.default_rng(3), [70, 40], 16, 4, 2)
    pool.table[pool.lines[0], 1] = 99999
    pool.table[pool.lines[0], 2] = -5
    pool.upload()
    fork(pool, [pool.lines[0]], [pool.lines[2]], [66])
    give_back(pool, [pool.lines[2]], [66])


@pytest.mark.parametrize("pages", [1, 63, 64, 65, 5000, 70001])
def test_the_queue_of_larger_pools(pages):
    rng = np.random.default_rng(pages)
    pool = Pool(rng, [pages], 1, 7, 1)
    pool.upload()
    fork(pool, [pool.lines[0]], [pool.lines[1]], [pages // 2])
    give_back(pool, [pool.lines[0]], [pages])
    give_back(pool, [pool.lines[1]], [pages // 2])
    assert pool.state[1] == pool.total


def compact(pool, limit, cap, in_place=False):
    d = pool.d
    o = {n: torch.full_like(d[n], 77) for n in ("table", "free", "shares")}
    if in_place:
        o["table"] = d["table"]
    ids, src, dst, status = i32([77] * pool.total), i32([77] * cap), i32([77] * cap), i32([9] * 5)
    oa.pages_compact(d["table"], d["free"], d["state"], d["shares"], limit, o["table"], o["free"], o["shares"], ids, src, dst, status)
    torch.cuda.synchronize()
    want, st = R.compact(pool.table, pool.free, pool.state, pool.shares, limit, cap)
    assert status.tolist() == [int(x) for x in st]
    if want is None:
        assert all(bool((x == 77).all()) for x in (o["free"], o["shares"], ids, *([] if in_place else [o["table"]])))
        assert bool((src == -1).all()) and bool((dst == -1).all())
        return st
    for n, t in (("table", o["table"]), ("free", o["free"]), ("shares", o["shares"]), ("new_ids", ids), ("src", src), ("dst", dst)):
        assert np.array_equal(host(t), want[n]), n
    pool.table, pool.free, pool.shares, pool.state = want["table"], want["free"], want["shares"], st[3:]
    d.update(o, state=status[3:5])
    return st, src, dst, status


@pytest.mark.parametrize("total,keep", [(1, 1.0), (2, 0.5), (255, 0.6), (256, 0.51), (257, 1.0), (3001, 0.55), (70000, 0.6)])
def test_compact(total, keep):
    rng = np.random.default_rng(total)
    pool = Pool(rng, [max(0, total // 4)] * 2, 1, total - 2 * (total // 4), 3)
    assert pool.total == total
    pool.shares[pool.table[pool.lines[0], :total // 4]] = rng.integers(0, 4, total // 4)
    pool.table[pool.lines[-1], 0] = total + 5  # no page of the pool
    pool.upload()
    st = compact(pool, int(total * keep), total, in_place=total % 2 == 1)
    assert st[0][0] == 0
    used = host(pool.d["table"])
    assert used[(used >= 0) & (used < total)].size == 0 or used[(used >= 0) & (used < total)].max() < max(1, int(total * keep))
    # And once more, to itself: nothing moves.
    assert compact(pool, int(total * keep), 4)[0][1] == 0


def test_compact_of_a_pool_as_large_as_one_may_be():
    """2^19 pages: every bit of the map is in use."""
    rng = np.random.default_rng(8)
    total = 1 << 19
    pool = Pool(rng, [total // 2], 1, total - total // 2, 0)
    pool.upload()
    assert compact(pool, total // 2 + 1000, total // 2)[0][0] == 0


@pytest.mark.parametrize("limit,cap,state,code", [(3, 99, None, 5), (0, 99, None, 5), (9, 1, None, 3), (9, 99, [0, 99], 1), (9, 99, [-1, 3], 1)])
def test_compactions_that_cannot_be_made(limit, cap, state, code):
    pool = Pool(np.random.default_rng(6), [90, 60], 16, 6, 1)
    if state:
        pool.state = state
    pool.upload()
    assert compact(pool, limit, cap)[0] == code


def test_a_queue_that_lists_a_page_twice():
    pool = Pool(np.random.default_rng(6), [90, 60], 16, 6, 1)
    pool.free[pool.head] = pool.free[(pool.head + 1) % pool.total]
    pool.upload()
    assert compact(pool, 11, 99)[0] == 1
    pool.free[pool.head] = pool.total
    pool.upload()
    assert compact(pool, 11, 99)[0] == 1


# ------------------------------------------------------------------ copy
def raw(t):
    return t.view(torch.uint8) if t.dtype != torch.bfloat16 else t.view(torch.int16)


@pytest.mark.parametrize("kind,hk,page,layers", [("e4m3", 1, 16, 0), ("e4m3", 8, 16, 3), ("int8", 3, 64, 0), ("int8", 2, 256, 2),
                                                 ("bf16", 2, 16, 0), ("bf16", 1, 1, 3), ("bf16", 4, 24, 2), ("e4m3", 5, 32, 1)])
def test_copy(kind, hk, page, layers):
    pages, n = 23, 9
    g = torch.Generator(device="cuda").manual_seed(hk + page)
    lead = [layers] if layers else []
    if kind == "bf16":
        kv, sc = torch.randn(*lead, pages * page, 2 * hk, 128, device="cuda", generator=g).to(torch.bfloat16), None
    else:
        kv = torch.randint(0, 256, (*lead, pages * page // 16, 2 * hk, 2048), dtype=torch.uint8, device="cuda", generator=g)
        kv = kv.view(torch.float8_e4m3fn if kind == "e4m3" else torch.int8)
        sc = torch.randint(1, 255, (*lead, pages * page // 16, 2 * hk), dtype=torch.uint8, device="cuda", generator=g)
    ids = np.random.default_rng(page).permutation(pages)
    src, dst = ids[:n].copy(), ids[n:2 * n].copy()
    src[2], dst[4], src[5], dst[6] = -1, -1, pages, pages + 3
    want = [None if t is None else raw(t).clone().view(max(layers, 1), pages, -1) for t in (kv, sc)]
    for k in range(n - 1):  # the count leaves the last pair out
        if 0 <= src[k] < pages and 0 <= dst[k] < pages:
            for w in want:
                if w is not None:
                    w[:, dst[k]] = w[:, src[k]].clone()
    oa.pages_copy(kv, sc, i32(src), i32(dst), page, i32([n - 1]))
    torch.cuda.synchronize()
    for t, w in zip((kv, sc), want):
        assert t is None or torch.equal(raw(t).view(w.shape), w)
    oa.pages_copy(kv, sc, i32(src[-1:]), i32(dst[-1:]), page)  # without a count, all
    torch.cuda.synchronize()
    for w in want:
        if w is not None:
            w[:, dst[-1]] = w[:, src[-1]].clone()
    for t, w in zip((kv, sc), want):
        assert t is None or torch.equal(raw(t).view(w.shape), w)


@pytest.mark.parametrize("count", [0, -4, 3, 100])
def test_copy_counts(count):
    kv, sc = oa.q8_cache(8, 16, 1, torch.int8)
    kv.copy_(torch.arange(8, device="cuda", dtype=torch.int8)[:, None, None].expand(kv.shape))
    oa.pages_copy(kv, sc, i32([0, 1, 2, 3]), i32([4, 5, 6, 7]), 16, i32([count]))
    torch.cuda.synchronize()
    n = max(0, min(4, count))
    assert kv[:, 0, 0].tolist() == [0, 1, 2, 3] + [0, 1, 2, 3][:n] + [4, 5, 6, 7][n:]
    oa.pages_copy(kv, sc, i32([]), i32([]), 16)


def test_offsets_past_32_bits():
    """The last page of a cache of more than 4 GiB, in its second layer."""
    hk, page, pages = 8, 256, 4500  # 512 KiB a page and layer
    kv = torch.zeros(2, pages * 16, 2 * hk, 2048, dtype=torch.int8, device="cuda")
    sc = torch.ones(2, pages * 16, 2 * hk, dtype=torch.uint8, device="cuda")
    kv[1, -16:] = 5
    sc[1, -1] = 9
    oa.pages_copy(kv, sc, i32([pages - 1, 0]), i32([pages - 2, 1]), page)
    torch.cuda.synchronize()
    assert bool((kv[1, -32:] == 5).all()) and not bool(kv[1, :-32].any()) and not bool(kv[0].any())
    assert bool((sc[1, -17] == 9).all()) and bool((sc[0] == 1).all()) and int(sc[1].sum()) == pages * 16 * 2 * hk + 2 * 8 * 2 * hk


# ------------------------------------------------------------------ together
def test_a_step_of_forks_in_a_graph():
    """Fork, copy and free of one set of candidates as one graph, replayed between eager work, against the same calls run eagerly."""
    rng = np.random.default_rng(11)
    pools = []
    for _ in range(2):
        rng = np.random.default_rng(11)
        p = Pool(rng, [187, 40, 96], 16, 40, 9)
        p.upload()
        g = torch.Generator(device="cuda").manual_seed(2)
        p.kv = torch.randint(0, 127, (2, p.total, 4, 2048), dtype=torch.int8, device="cuda", generator=g)
        p.sc = torch.randint(1, 255, (2, p.total, 4), dtype=torch.uint8, device="cuda", generator=g)
        par, chi = [p.lines[i // 3] for i in range(9)], p.lines[3:]
        tok = [p.lens[i // 3] - (i % 3) * 7 for i in range(9)]
        p.a = [i32(x) for x in (par, chi, tok, [0] * 9, [0] * 9)]
        p.st = [i32([0] * 5), i32([0, 0, 0, *p.state])]
        pools.append(p)

    def step(p, stream=None):
        d, (par, chi, tok, src, dst) = p.d, p.a
        oa.pages_fork(par, chi, tok, d["table"], d["free"], p.st[1][3:5], d["shares"], src, dst, p.st[0], 16, stream)
        oa.pages_copy(p.kv, p.sc, src, dst, 16, None, stream)
        oa.pages_free(chi, tok, d["table"], d["free"], p.st[0][3:5], d["shares"], p.st[1], 16, stream)

    a, b = pools
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        step(b)
    for rep in range(12):
        for p in pools:
            p.kv[:, rep] += 1
        step(a)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for n in ("table", "free", "shares"):
            assert torch.equal(a.d[n], b.d[n]), (rep, n)
        assert torch.equal(a.kv, b.kv) and torch.equal(a.sc, b.sc) and torch.equal(a.st[0], b.st[0]) and torch.equal(a.st[1], b.st[1])
        assert int(a.st[0][0]) == 0 and int(a.st[1][0]) == 0 and not bool(a.d["shares"].any())


def test_on_another_stream():
    pool = Pool(np.random.default_rng(7), [100, 30], 16, 9, 4)
    pool.upload()
    torch.cuda.synchronize()
    fork(pool, [pool.lines[0]] * 2, pool.lines[2:4], [100, 50], torch.cuda.Stream())
