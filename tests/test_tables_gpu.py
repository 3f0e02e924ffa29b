"""step_tables on the GPU against host loops: every output equal, over batches
from none to several scans of sequences, rings, leased tables, done requests,
full and wrapped queues, refusals, replays and other streams."""
import numpy as np
import pytest
import torch

import omni_attn as oa
import serve_refs as R

pytestmark = pytest.mark.gpu


def i32(a):
    return torch.from_numpy(np.array(a, dtype=np.int32).copy()).cuda()


class Step:
    def __init__(self, nseq, lines, width, pool, row_cap, page_cap, seed=0, page=16, ring=0, leased=False):
        self.rng = np.random.default_rng(seed)
        self.nseq, self.page, self.ring = nseq, page, ring
        self.rows, self.pcap = row_cap, page_cap
        self.table = np.full((lines, width), -7, np.int32)
        self.free = None if leased else np.full(pool, -9, np.int32)
        self.state = None if leased else np.zeros(2, np.int32)
        self.pool = pool

    def fill(self, first, lines):
        """Gives each line the pages of its first[] tokens and the rest to the queue, from a random place on."""
        ids = self.rng.permutation(self.pool).astype(np.int32)
        at = 0
        for f, line in zip(first, lines):
            n = (min(f, self.ring) if self.ring else f) + self.page - 1
            n //= self.page
            self.table[line, :n] = ids[at:at + n]
            at += n
        if self.free is not None:
            head = int(self.rng.integers(self.pool))
            for i, p in enumerate(ids[at:]):
                self.free[(head + i) % self.pool] = p
            self.state[:] = head, self.pool - at
        else:
            self.table[:] = self.rng.integers(0, self.pool, self.table.shape)

    def device(self):
        d = dict(table=i32(self.table), free=None if self.free is None else i32(self.free),
                 state=None if self.state is None else i32(self.state))
        d.update(pos=i32([5] * self.rows), slots=i32([5] * self.rows), seq=i32([5] * self.rows),
                 row_indptr=i32([5] * (self.nseq + 1)), indptr=i32([5] * (self.nseq + 1)),
                 pages=i32([5] * self.pcap), status=i32([5] * 5))
        return d

    def call(self, d, first, count, lines, stream=None):
        oa.step_tables(first, count, lines, d["table"], d["free"], d["state"], d["pos"], d["slots"], d["seq"],
                       d["row_indptr"], d["indptr"], d["pages"], d["status"], self.page, self.ring, stream)

    def check(self, d, first, count, lines, stale=5):
        want = R.tables(first, count, lines, self.table, self.free, self.state, self.rows, self.pcap, self.page, self.ring)
        for name in ("pos", "slots", "seq"):
            full = np.full(self.rows, -1)
            full[:len(want[name])] = want[name]
            assert np.array_equal(d[name].cpu().numpy(), full), name
        for name in ("row_indptr", "indptr", "status"):
            assert np.array_equal(d[name].cpu().numpy(), want[name]), name
        full = np.full(self.pcap, stale)
        full[:len(want["pages"])] = want["pages"]
        if stale is not None:
            assert np.array_equal(d["pages"].cpu().numpy(), full)
        assert np.array_equal(d["table"].cpu().numpy(), want["table"])
        if self.free is not None:
            assert np.array_equal(d["free"].cpu().numpy(), want["free"])
        return want


def lengths(rng, nseq, ctx, new, done):
    first = rng.integers(0, ctx + 1, nseq)
    count = np.where(rng.random(nseq) < 0.5, 1, rng.integers(0, new + 1, nseq))
    count[rng.random(nseq) < done] = -1
    return first.astype(np.int32), count.astype(np.int32)


@pytest.mark.parametrize("nseq,ctx,new,page,ring,leased", [
    (0, 0, 0, 16, 0, False), (1, 0, 1, 16, 0, False), (1, 100, 1, 16, 0, False), (5, 40, 33, 16, 0, False),
    (64, 2400, 1, 16, 0, False), (64, 300, 200, 16, 0, True), (255, 50, 20, 16, 0, False), (256, 50, 20, 16, 0, False),
    (257, 50, 20, 16, 0, False), (512, 70, 30, 16, 0, False), (513, 90, 9, 16, 0, True), (700, 90, 9, 16, 0, False),
    (1024, 60, 9, 16, 0, False), (1025, 60, 9, 16, 0, False), (2600, 40, 5, 16, 48, False), (30, 400, 90, 10, 0, False), (30, 400, 90, 1, 0, False),
    (40, 900, 60, 16, 300, False), (40, 900, 60, 16, 301, True), (9, 700, 2000, 64, 0, False),
])
def test_matches_host_loops(nseq, ctx, new, page, ring, leased):
    for seed in range(2):
        rng = np.random.default_rng(seed * 100 + nseq)
        first, count = lengths(rng, nseq, ctx, new, 0.2 if nseq > 2 else 0)
        width = (ctx + new + page) // page + 1
        pages = int(sum((f + max(c, 0) + page - 1) // page + 1 for f, c in zip(first, count)))
        rows = int(np.maximum(count, 0).sum())
        st = Step(nseq, nseq + 3, width, pages + 5, rows + 37 * seed, pages + 3, seed, page, ring, leased)
        lines = rng.permutation(nseq + 3)[:nseq].astype(np.int32)
        st.fill(first, lines)
        d = st.device()
        st.call(d, i32(first), i32(count), i32(lines))
        st.check(d, first, count, lines)
        # Again on what it left: the same step gives the same tables and queue.
        st.call(d, i32(first), i32(count), i32(lines))
        st.check(d, first, count, lines)


def test_lines_default_to_the_sequence():
    st = Step(3, 3, 4, 20, 8, 12)
    first, count = np.array([3, 0, 16], np.int32), np.array([1, 2, 1], np.int32)
    st.fill(first, range(3))
    d = st.device()
    st.call(d, i32(first), i32(count), None)
    st.check(d, first, count, None)


@pytest.mark.parametrize("code,first,count,lines,rows,pages", [
    (1, [-1, 3], [1, 1], [0, 1], 4, 4), (1, [0, 2**31 - 2], [1, 2], [0, 1], 4, 4), (1, [0, 0], [1, 1], [0, 2], 4, 4),
    (1, [0, 0], [1, 1], [-1, 1], 4, 4), (2, [0, 0], [3, 2], [0, 1], 4, 4), (3, [20, 20], [1, 1], [0, 1], 4, 3),
    (4, [0, 0], [1, 65], [0, 1], 99, 99), (5, [0, 0], [64, 40], [0, 1], 200, 99), (2, [0, 0], [64, 64], [0, 1], 4, 2),
])
def test_a_step_that_cannot_be_made_changes_nothing(code, first, count, lines, rows, pages):
    st = Step(2, 2, 4, 6, rows, pages)
    st.fill([0, 0], [0, 1])
    d = st.device()
    st.call(d, i32(first), i32(count), i32(lines))
    want = st.check(d, np.array(first), np.array(count), lines)
    assert want["status"][0] == code


@pytest.mark.parametrize("state", [[-1, 2], [6, 2], [0, -1], [0, 7]])
def test_bad_queue_states_are_reported(state):
    st = Step(1, 1, 4, 6, 4, 4)
    st.fill([0], [0])
    st.state[:] = state
    d = st.device()
    st.call(d, i32([0]), i32([1]), i32([0]))
    assert st.check(d, np.array([0]), np.array([1]), [0])["status"][0] == 1


def test_many_steps_with_admissions_and_ends():
    """Requests come, grow and go over 60 steps, two status buffers taking turns: pages are never held twice, and the tables equal the
    host's at every step."""
    rng = np.random.default_rng(5)
    lines, width, pool = 12, 24, 300
    st = Step(lines, lines, width, pool, 750, 400)
    st.fill([0] * lines, range(lines))
    d = st.device()
    other = i32([0] * 5)
    length = np.full(lines, -1)
    for step in range(60):
        live = [s for s in range(lines) if length[s] >= 0]
        first, count, used = [], [], []
        for s in range(lines):
            if length[s] >= 0:
                end = length[s] > 250 or rng.random() < 0.06
                first.append(length[s]), count.append(-1 if end else 1), used.append(s)
                length[s] = -1 if end else length[s] + 1
            elif rng.random() < 0.3:
                n = int(rng.integers(1, 60))
                first.append(0), count.append(n), used.append(s)
                length[s] = n
        n = len(first)
        st.nseq = n
        d["row_indptr"], d["indptr"] = i32([5] * (n + 1)), i32([5] * (n + 1))
        d["pages"].fill_(5)
        d["status"], other = other, d["status"]
        first, count = np.array(first, np.int32), np.array(count, np.int32)
        st.call(d, i32(first), i32(count), i32(used) if n else None)
        want = st.check(d, first, count, used)
        assert want["status"][0] == 0 and len(live) <= lines
        d["state"] = d["status"][3:5]
        st.table, st.free, st.state = want["table"], want["free"], np.array(want["status"][3:], np.int32)
        queue = [int(st.free[(st.state[0] + i) % pool]) for i in range(st.state[1])]
        mine = [int(p) for s in range(lines) if length[s] > 0 for p in st.table[s, :(length[s] + 15) // 16]]
        assert sorted(queue + mine) == list(range(pool))


def test_equals_the_host_row_builder():
    first, count = np.array([0, 33, 100, 15], np.int32), np.array([40, 1, 3, 2], np.int32)
    st = Step(4, 4, 10, 64, 46, 64)
    st.fill(first, range(4))
    d = st.device()
    st.call(d, i32(first), i32(count), None)
    table = d["table"].cpu().numpy()
    rows = oa.Rows(16)
    for s in range(4):
        rows.push(table[s, :(first[s] + count[s] + 15) // 16], int(first[s]), int(count[s]), s)
    got = {n: d[m].cpu().numpy() for n, m in (("pos", "pos"), ("slot", "slots"), ("seq", "seq"), ("indptr", "indptr"))}
    for n, g in got.items():
        assert np.array_equal(g, getattr(rows, n)), n
    assert np.array_equal(d["pages"].cpu().numpy()[:len(rows.pages)], rows.pages)


def test_replays_follow_the_lengths():
    st = Step(6, 6, 30, 200, 64, 200, seed=3)
    first = np.array([0, 10, 20, 30, 40, 50], np.int32)
    st.fill(first, range(6))
    d = st.device()
    f, c, lines = i32(first), i32([1] * 6), i32(range(6))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        st.call(d, f, c, lines)
    torch.cuda.synchronize()
    st.check(d, first, np.ones(6, np.int32), list(range(6)))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        st.call(d, f, c, lines)
    rng = np.random.default_rng(1)
    for rep in range(4):
        count = rng.integers(0, 11, 6).astype(np.int32)
        c.copy_(i32(count))
        d["table"].copy_(i32(st.table)), d["free"].copy_(i32(st.free)), d["pages"].fill_(5)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        st.check(d, first, count, list(range(6)))
