"""The 8-bit serving calls together, as an engine would use them: row tables from
the request lengths, rotary + quantized write, prompts over their own rows and
new tokens over the cache, for requests that come, grow and end; and a decode
step captured in two graphs that take turns. And what the Python mirror refuses."""
import numpy as np
import pytest
import torch

import omni_attn as oa
import serve_refs as R

pytestmark = pytest.mark.gpu

EPS, THETA, SCALE = 1e-6, 1e6, 128 ** -0.5


def i32(a):
    return torch.from_numpy(np.array(a, dtype=np.int32).copy()).cuda()


class Engine:
    """Device state of a server of `lines` requests at most over `pages` pages."""

    def __init__(self, hq, hk, lines, pages, page, fmt, seed):
        self.hq, self.hk, self.page = hq, hk, page
        self.kv, self.sc = oa.q8_cache(pages, page, hk, fmt)
        self.table = i32(np.full((lines, 64), -1))
        self.free = i32(np.random.default_rng(seed).permutation(pages))
        self.state = i32([0, pages])
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.gen = g
        self.norms = [(1 + 0.2 * torch.randn(128, device="cuda", generator=g)).to(torch.bfloat16) for _ in range(2)]

    def tables(self, first, count, lines, rows, npages):
        n = len(first)
        t = {k: i32(np.zeros(m)) for k, m in (("pos", rows), ("slots", rows), ("seq", rows), ("row_indptr", n + 1),
                                              ("indptr", n + 1), ("pages", npages), ("status", 5))}
        oa.step_tables(i32(first), i32(count), i32(lines), self.table, self.free, self.state, t["pos"], t["slots"], t["seq"],
                       t["row_indptr"], t["indptr"], t["pages"], t["status"], self.page)
        self.state = t["status"][3:5]
        return t

    def write(self, qkv, t):
        rows = qkv.shape[0]
        q = torch.zeros(rows, self.hq * 128, dtype=torch.bfloat16, device="cuda")
        k = torch.zeros(rows, self.hk * 128, dtype=torch.bfloat16, device="cuda")
        oa.qwen3_rope_q8(qkv, *self.norms, t["pos"], t["slots"], q, k, self.kv, self.sc, self.hq, self.hk, EPS, THETA)
        return q, k


@pytest.mark.parametrize("fmt", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("hq,hk,page", [(8, 2, 16), (4, 4, 32)])
def test_requests_come_grow_and_end(fmt, hq, hk, page):
    e = Engine(hq, hk, 6, 60, page, fmt, seed=hq)
    rng = np.random.default_rng(hq + page)
    ref = R.Cache(e.kv, e.sc, hk)
    length, slots_of = {}, {}  # line -> tokens, slots
    for step in range(14):
        running = sorted(length)
        done = [s for s in running if length[s] > 40 and rng.random() < 0.4]
        decode = [s for s in running if s not in done]
        fresh = [s for s in range(6) if s not in length][:2]
        new = [int(rng.choice([1, 15, 33, 70, 129])) for _ in fresh]
        # Decode rows first, then the prompts' rows, so that each is one range of rows.
        seqs = decode + fresh + done
        first = [length[s] for s in decode] + [0] * len(fresh) + [length[s] for s in done]
        count = [1] * len(decode) + new + [-1] * len(done)
        nd, rows = len(decode), len(decode) + sum(new)
        if rows == 0:
            continue
        t = e.tables(first, count, seqs, rows + 5, 200)
        qkv = torch.randn(rows + 5, (hq + 2 * hk) * 128, device="cuda", generator=e.gen).to(torch.bfloat16)
        q, k = e.write(qkv, t)
        out = torch.full((rows + 5, hq * 128), 7.0, dtype=torch.bfloat16, device="cuda")
        v = qkv[:, (hq + hk) * 128:]
        if nd:
            plan = oa.decode_plan_q8(nd, hq, hk, page, max(first[:nd]) + 1, 64)
            oa.qwen3_attend_q8(q[:nd], e.kv, e.sc, t["pos"], t["seq"], 1, t["indptr"], t["pages"], page, out[:nd], hq, hk, SCALE,
                               plan, oa.workspace_for(plan))
        if new:
            oa.prompt_run(oa.prompt_plan(new, hq, hk, exact_p=True), q[nd:], k[nd:], v[nd:], out[nd:], SCALE)
        torch.cuda.synchronize()
        assert t["status"].tolist()[:2] == [0, rows]
        pos, slots, seq = (t[n].cpu().numpy() for n in ("pos", "slots", "seq"))
        assert (slots[rows:] == -1).all() and bool((q[rows:] == 0).all()) and bool((out[rows:] == 7).all())
        kk, vv = k.cpu().double().view(-1, hk, 128), v.cpu().double().view(-1, hk, 128)
        ref.write(slots, kk, vv)
        ref.same_as(e.kv, e.sc)
        ck, cv = ref.tokens()
        for s, c in zip(seqs, count):
            if c < 0:
                del length[s], slots_of[s]
            else:
                length[s] = length.get(s, 0) + c
        for n in range(rows):
            s = seqs[seq[n]]
            slots_of.setdefault(s, []).append(int(slots[n]))
            if n < nd:  # over the quantized cache
                at = slots_of[s]
                want, size = R.attend(q[n].cpu().view(hq, 128), ck[at], cv[at], SCALE)
            else:  # over the prompt's own bf16 rows
                b = n - pos[n]
                want, size = R.attend(q[n].cpu().view(hq, 128), kk[b:n + 1], vv[b:n + 1], SCALE)
            bound = 2.0 ** -8 * want.abs() + 2.0 ** -13 * size
            assert bool(((out[n].cpu().double().view(hq, 128) - want).abs() <= bound).all()), f"step {step} row {n}"
        for s in length:
            assert len(slots_of[s]) == length[s] and len(set(slots_of[s])) == length[s]
        live = sum(len(x) for x in slots_of.values())
        assert len({x for y in slots_of.values() for x in y}) == live  # no slot is anybody else's
    assert length


def test_two_graphs_that_take_turns():
    """A decode step of five requests, captured once for each of two status buffers; 40 replays, pages taken as the requests grow,
    against the same step run eagerly on a state of its own."""
    hq, hk, page, n = 16, 8, 16, 5
    start = [0, 15, 16, 100, 31]

    def make():
        e = Engine(hq, hk, n, 80, page, torch.float8_e4m3fn, seed=3)
        t = e.tables([0] * n, start, list(range(n)), sum(start), 100)
        qkv = torch.randn(sum(start), (hq + 2 * hk) * 128, device="cuda", generator=e.gen).to(torch.bfloat16)
        e.write(qkv, t)
        d = dict(first=i32(start), count=i32([1] * n), lines=i32(range(n)), pos=i32([0] * n), slots=i32([0] * n), seq=i32([0] * n),
                 row_indptr=i32([0] * (n + 1)), indptr=i32([0] * (n + 1)), pages=i32([0] * 100),
                 status=[torch.cat([i32([0, 0, 0]), e.state]), i32([0] * 5)])
        d["qkv"] = torch.zeros(n, (hq + 2 * hk) * 128, dtype=torch.bfloat16, device="cuda")
        d["q"] = torch.zeros(n, hq * 128, dtype=torch.bfloat16, device="cuda")
        d["out"] = torch.zeros(n, hq * 128, dtype=torch.bfloat16, device="cuda")
        d["plan"] = oa.decode_plan_q8(n, hq, hk, page, 200, 64)
        d["ws"] = oa.workspace_for(d["plan"])
        return e, d

    def step(e, d, turn, s=None):
        oa.step_tables(d["first"], d["count"], d["lines"], e.table, e.free, d["status"][turn][3:5], d["pos"], d["slots"], d["seq"],
                       d["row_indptr"], d["indptr"], d["pages"], d["status"][1 - turn], page, 0, s)
        oa.qwen3_rope_q8(d["qkv"], *e.norms, d["pos"], d["slots"], d["q"], None, e.kv, e.sc, hq, hk, EPS, THETA, s)
        oa.qwen3_attend_q8(d["q"], e.kv, e.sc, d["pos"], None, 0, d["indptr"], d["pages"], page, d["out"], hq, hk, SCALE, d["plan"],
                           d["ws"], s)

    (a, da), (b, db) = make(), make()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    graphs = []
    for turn in (0, 1):  # captured, not run
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[turn], stream=s):
            step(b, db, turn)
    g = torch.Generator(device="cuda").manual_seed(9)
    for rep in range(40):
        qkv = torch.randn(da["qkv"].shape, device="cuda", generator=g).to(torch.bfloat16)
        for d in (da, db):
            d["qkv"].copy_(qkv)
        step(a, da, rep % 2)
        torch.cuda.synchronize()
        graphs[rep % 2].replay()
        torch.cuda.synchronize()
        for name in ("pos", "slots", "indptr", "q", "out"):
            assert torch.equal(da[name], db[name]), (rep, name)
        assert torch.equal(da["status"][1 - rep % 2], db["status"][1 - rep % 2]) and int(da["status"][1 - rep % 2][0]) == 0
        assert torch.equal(a.table, b.table) and torch.equal(a.kv.view(torch.uint8), b.kv.view(torch.uint8))
        da["first"] += 1
        db["first"] += 1
    assert int(da["status"][0][4]) < int(a.state[1])  # pages were taken


def test_the_mirror_refuses_what_the_kernels_do_not_take():
    hq, hk, n = 4, 2, 3
    b = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device="cuda")
    kv, sc = oa.q8_cache(4, 16, hk)
    z = i32([0] * 8)

    def refused(f, *a):
        with pytest.raises(oa.OmniAttnError):
            f(*a)

    good = [b(n, 1024), b(128), b(128), z[:n], z[:n], b(n, 512), b(n, 256), kv, sc, hq, hk, EPS, THETA]
    oa.qwen3_rope_q8(*good)
    for at, bad in ((0, b(n - 1, 1024)), (0, b(n, 1024).float()), (0, b(1024, n).t()), (0, b(n, 1025)[:, :1024]), (1, b(64)),
                    (1, b(256)[::2]), (3, z[:n].long()), (3, i32([0] * 6)[::2]), (4, z[:2]), (5, b(n, 256)), (6, b(2, 256)),
                    (7, kv.view(torch.uint8)), (7, kv[:, :2]), (7, kv[:, :, :1024]), (8, sc[:3]), (8, sc.float()), (8, sc.cpu()),
                    (7, kv.cpu()), (5, b(n, 512).cpu())):
        refused(oa.qwen3_rope_q8, *good[:at], bad, *good[at + 1:])
    plan = oa.decode_plan_q8(n, hq, hk, 16, 200, 64)
    ws = oa.workspace_for(plan)
    good = [b(n, 512), kv, sc, z[:n], z[:n], 1, z[:4], z, 16, b(n, 512), hq, hk, SCALE, plan, ws]
    oa.qwen3_attend_q8(*good)
    for at, bad in ((0, b(2, 512)), (3, z[:2]), (4, z[:2]), (4, None), (6, z[:0]), (9, b(2, 512)), (9, b(512, n).t()), (8, 32),
                    (14, ws[:-1]), (14, None), (14, ws.cpu())):
        refused(oa.qwen3_attend_q8, *good[:at], bad, *good[at + 1:])
    pp = oa.prompt_plan([n], hq, hk)
    good = [pp, b(n, 512), b(n, 256), b(n, 256), b(n, 512), SCALE]
    oa.prompt_run(*good)
    for at, bad in ((1, b(2, 512)), (2, b(n, 512)), (3, b(n, 256).float()), (4, b(n, 256)), (4, b(n, 1024)[:, :512]), (3, b(n, 260)[:, 2:258])):
        refused(oa.prompt_run, *good[:at], bad, *good[at + 1:])
    good = [z[:2], z[:2], z[:2], i32(np.zeros((2, 4))), i32([0] * 9), i32([0, 9]), i32([0] * 4), i32([0] * 4), i32([0] * 4), i32([0] * 3),
            i32([0] * 3), i32([0] * 4), i32([0] * 5)]
    oa.step_tables(*good)
    for at, bad in ((0, z[:2].float()), (1, z[:1]), (2, z[:1]), (3, z), (4, z[:0]), (5, z[:1]), (5, None), (7, z[:3]), (8, z[:3]), (9, z[:2]),
                    (10, z[:2]), (12, z[:4]), (6, z.cpu())):
        refused(oa.step_tables, *good[:at], bad, *good[at + 1:])
    status = i32([0] * 5)
    refused(oa.step_tables, *good[:5], status[3:5], *good[6:12], status)
    torch.cuda.synchronize()
