"""Requests with shared prefixes, as a server would run them: prompts, candidates that
are forked from them, prompts behind a prefix and several proposed tokens over the
8-bit cache, cross attention of a request's candidates over its encoder's states, ends,
and the pool compacted in between. Every step against 64 bits over the cache's own
values, and every token of every line where it was put."""
import numpy as np
import pytest
import torch

import multi_refs as M
import omni_attn as oa
import serve_refs as R

pytestmark = pytest.mark.gpu

EPS, THETA, SCALE = 1e-6, 1e6, 128 ** -0.5


def i32(a):
    return torch.from_numpy(np.array(a, dtype=np.int32).copy()).cuda()


class Server:
    def __init__(self, hq, hk, page, fmt, lines=14, pages=120, layers=2, seed=1):
        self.hq, self.hk, self.page, self.pages, self.layers = hq, hk, page, pages, layers
        one = [oa.q8_cache(pages, page, hk, fmt) for _ in range(layers)]
        self.kv = torch.stack([k.view(torch.uint8) for k, _ in one]).view(fmt)
        self.sc = torch.stack([s.view(torch.uint8) for _, s in one])
        self.table = i32(np.full((lines, 40), -1))
        self.free, self.shares = i32(np.random.default_rng(seed).permutation(pages)), i32([0] * pages)
        self.state = i32([0, pages])
        self.gen = torch.Generator(device="cuda").manual_seed(seed)
        self.norms = [(1 + 0.2 * torch.randn(128, device="cuda", generator=self.gen)).to(torch.bfloat16) for _ in range(2)]
        self.len, self.tokens = {}, {}  # line -> tokens; line -> per layer (K, V) of its tokens, as stored

    def bf16(self, *shape):
        return torch.randn(*shape, device="cuda", generator=self.gen).to(torch.bfloat16)

    def slots(self, line):
        ids = self.table[line].tolist()
        return [ids[t // self.page] * self.page + t % self.page for t in range(self.len[line])]

    def look(self, layer):
        return R.Cache(self.kv[layer], self.sc[layer], self.hk).tokens()

    def check_tokens(self):
        """Every line's tokens are the ones that were written; no page is free and held, or held by more lines than it counts."""
        for layer in range(self.layers):
            k, v = self.look(layer)
            for line in self.len:
                at = self.slots(line)
                assert torch.equal(k[at], self.tokens[line][layer][0]) and torch.equal(v[at], self.tokens[line][layer][1]), (layer, line)
        held = {}
        for line, n in self.len.items():
            for p in self.table[line].tolist()[:-(-n // self.page)]:
                held[p] = held.get(p, 0) + 1
        head, avail = self.state.tolist()
        queue = [int(self.free[(head + i) % self.pages]) for i in range(avail)]
        assert len(set(queue)) == avail and not set(queue) & set(held) and avail + len(held) == self.pages
        shares = self.shares.tolist()
        assert all(shares[p] == held.get(p, 1) - 1 for p in range(self.pages))

    def rows(self, lines, counts):
        """New rows of these lines: tables, rotary and write in every layer, attention of the rows over the cache."""
        n, rows = len(lines), sum(counts)
        first = [self.len.get(x, 0) for x in lines]
        t = {k: i32([0] * m) for k, m in (("pos", rows), ("slots", rows), ("seq", rows), ("ri", n + 1), ("indptr", n + 1),
                                          ("pages", 400), ("status", 5))}
        oa.step_tables(i32(first), i32(counts), i32(lines), self.table, self.free, self.state, t["pos"], t["slots"], t["seq"], t["ri"],
                       t["indptr"], t["pages"], t["status"], self.page)
        self.state = t["status"][3:5]
        assert int(t["status"][0]) == 0
        for line, f, c in zip(lines, first, counts):
            self.len[line] = f + c
        last = [f + c for f, c in zip(first, counts)]
        mp = oa.extend_plan(counts, self.hq, self.hk, max(last), last, 64)
        ws = oa.workspace_for(mp.plan)
        for layer in range(self.layers):
            qkv = self.bf16(rows, (self.hq + 2 * self.hk) * 128)
            q = torch.zeros(rows, self.hq * 128, dtype=torch.bfloat16, device="cuda")
            oa.qwen3_rope_q8(qkv, *self.norms, t["pos"], t["slots"], q, None, self.kv[layer], self.sc[layer], self.hq, self.hk, EPS, THETA)
            out = torch.zeros_like(q)
            oa.qwen3_extend_q8(mp, q, self.kv[layer], self.sc[layer], t["pos"], t["indptr"], t["pages"], self.page, out, SCALE, ws)
            torch.cuda.synchronize()
            k, v = self.look(layer)
            at = 0
            for line, f, c in zip(lines, first, counts):
                s = self.slots(line)
                want, size = M.rows_of(q[at:at + c].cpu().view(c, self.hq, 128), k[s], v[s], [f + 1 + i for i in range(c)], SCALE)
                err = (out[at:at + c].cpu().double().view(c, self.hq, 128) - want).abs() - M.bound(want, size, mp.plan.tiles > 0)
                assert bool((err <= 0).all()), (layer, line, float(err.max()))
                at += c
                # What the blocks held before may have been rounded again; whole ones before the first new row were not touched.
                old = self.tokens.get(line, {}).get(layer)
                if old is not None:
                    keep = f // 16 * 16
                    assert torch.equal(k[s[:keep]], old[0][:keep]) and torch.equal(v[s[:keep]], old[1][:keep])
                self.tokens.setdefault(line, {})[layer] = (k[s], v[s])

    def fork(self, parents, children, tokens):
        n = len(parents)
        src, dst, status = i32([0] * n), i32([0] * n), i32([0] * 5)
        oa.pages_fork(i32(parents), i32(children), i32(tokens), self.table, self.free, self.state, self.shares, src, dst, status, self.page)
        oa.pages_copy(self.kv, self.sc, src, dst, self.page)
        self.state = status[3:5]
        assert int(status[0]) == 0
        for p, c, t in zip(parents, children, tokens):
            self.len[c] = t
            self.tokens[c] = {y: (k[:t], v[:t]) for y, (k, v) in self.tokens[p].items()}

    def end(self, lines):
        status = i32([0] * 5)
        oa.pages_free(i32(lines), i32([self.len[x] for x in lines]), self.table, self.free, self.state, self.shares, status, self.page)
        self.state = status[3:5]
        assert int(status[0]) == 0
        for x in lines:
            del self.len[x], self.tokens[x]

    def compact(self, limit):
        out = [torch.zeros_like(x) for x in (self.free, self.shares, self.shares)]
        src, dst, status = i32([0] * self.pages), i32([0] * self.pages), i32([0] * 5)
        oa.pages_compact(self.table, self.free, self.state, self.shares, limit, self.table, *out, src, dst, status)
        oa.pages_copy(self.kv, self.sc, src, dst, self.page, status[1:2])
        self.free, self.shares, self.state = out[0], out[1], status[3:5]
        assert int(status[0]) == 0


@pytest.mark.parametrize("hq,hk,page,fmt", [(8, 2, 16, torch.float8_e4m3fn), (6, 2, 32, torch.int8), (4, 4, 16, torch.int8)])
def test_candidates_of_a_request(hq, hk, page, fmt):
    s = Server(hq, hk, page, fmt)
    s.rows([0, 1], [70, 33])  # two prompts
    s.check_tokens()
    s.fork([0, 0, 0, 1], [2, 3, 4, 5], [70, 64, 45, 33])
    s.check_tokens()
    s.rows([0, 2, 3, 4, 5], [1, 3, 4, 40, 1])  # each goes on for itself: a token, proposals, a prompt behind the prefix
    s.check_tokens()
    s.fork([4, 2], [6, 7], [85, 73])  # candidates of candidates
    s.end([0, 3])
    s.check_tokens()
    used = s.pages - int(s.state[1])
    s.compact(used)
    s.check_tokens()
    assert int(s.table[s.table >= 0].max()) < s.pages
    s.rows([7, 6, 1, 2], [2, 50, 7, 1])
    s.check_tokens()
    s.end([1, 2, 4, 5, 6, 7])
    s.check_tokens()
    assert int(s.state[1]) == s.pages and not bool(s.shares.any())


def test_candidates_share_their_encoder():
    """Self-attention over forked pages and cross attention over the request's states, both for all candidates of two requests."""
    hq, hk = 8, 4
    s = Server(hq, hk, 16, torch.float8_e4m3fn, layers=1)
    s.rows([0, 1], [20, 50])
    s.fork([0, 0, 1], [2, 3, 4], [20, 20, 50])
    lines, of = [[0, 2, 3], [1, 4]], [1, 0]  # candidates of a request stand together; its source
    enc = s.bf16(300, 2 * hk * 128)
    first, length = [0, 100], [100, 200]
    for _ in range(3):
        flat = [x for group in lines for x in group]
        s.rows(flat, [1] * len(flat))
        q = s.bf16(len(flat), hq * 128)
        out = torch.zeros_like(q)
        mp = oa.cross_plan([len(x) for x in lines], hq, hk, 200, [length[e] for e in of])
        oa.cross_run(mp, q, enc[:, :hk * 128], enc[:, hk * 128:], i32(of), i32(first), i32(length), out, SCALE, oa.workspace_for(mp.plan))
        torch.cuda.synchronize()
        at = 0
        for group, e in zip(lines, of):
            n, part = len(group), slice(first[e], first[e] + length[e])
            kv = enc[part].cpu().view(-1, 2 * hk, 128)
            want, size = M.rows_of(q[at:at + n].cpu().view(n, hq, 128), kv[:, :hk], kv[:, hk:], [length[e]] * n, SCALE)
            assert bool(((out[at:at + n].cpu().double().view(n, hq, 128) - want).abs() <= M.bound(want, size, False)).all())
            at += n
    s.check_tokens()
