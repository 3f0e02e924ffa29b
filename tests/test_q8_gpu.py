"""The 8-bit block cache on the GPU: the rotary + quantized write byte for byte
(the cache against a host quantizer fed with the kernel's own bf16 k, the turned
values against 64 bits), and decode attention over it against 64 bits."""
import math

import numpy as np
import pytest
import torch

import omni_attn as oa
import serve_refs as R

pytestmark = pytest.mark.gpu

FORMATS = [torch.float8_e4m3fn, torch.int8]
EPS, THETA = 1e-6, 1e6


def i32(a):
    return torch.from_numpy(np.array(a, dtype=np.int32).copy()).cuda()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def random_cache(g, blocks, hk, fmt):
    kv, sc = oa.q8_cache(blocks, 16, hk, fmt)
    x = torch.randn(kv.shape, device="cuda", generator=g)
    kv.copy_((x * 90).clamp(-448, 448).to(fmt) if fmt == torch.float8_e4m3fn else (x * 40).round().clamp(-127, 127).to(fmt))
    sc.view(torch.uint8).copy_(torch.randint(115, 123, sc.shape, device="cuda", generator=g).to(torch.uint8))
    return kv, sc


def runs_to_slots(rng, runs, blocks):
    """Slots and positions of runs (first token in its block, rows): blocks of their own, anywhere in the pool."""
    ids = list(rng.permutation(blocks))
    slots, pos = [], []
    for t0, m in runs:
        base = None
        for i in range(m):
            t = t0 + i
            if base is None or t % 16 == 0:
                base = int(ids.pop())
            slots.append(base * 16 + t % 16), pos.append(1000 + t)
    return slots, pos


def write(qkv, pos, slots, kv, sc, hq, hk, w, k_out=True, theta=THETA):
    rows = len(slots)
    q = torch.full((rows, hq * 128), 7.0, dtype=torch.bfloat16, device="cuda")
    k = torch.full((rows, hk * 128), 7.0, dtype=torch.bfloat16, device="cuda")
    oa.qwen3_rope_q8(qkv, w[0], w[1], i32(pos), i32(slots), q, k if k_out else None, kv, sc, hq, hk, EPS, theta)
    torch.cuda.synchronize()
    return q, k


def weights(g):
    return [(1 + 0.3 * torch.randn(128, device="cuda", generator=g)).to(torch.bfloat16) for _ in range(2)]


def check_turned(out, x, w, pos, theta=THETA):
    want, bound = R.turned(x, w, torch.tensor(pos), EPS, theta)
    d = (out.double().cpu().view_as(want) - want).abs()
    assert bool((d <= bound).all()), f"turned: {float((d - bound).max()):.3g} past its bound"


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("hq,hk", [(1, 1), (2, 1), (16, 8), (20, 4), (6, 3), (33, 1), (32, 32)])
def test_write_matches_the_host_quantizer(fmt, hq, hk):
    g, rng = gen(hq * 7 + hk), np.random.default_rng(hk)
    runs = [(0, 1), (0, 16), (5, 1), (15, 1), (3, 13), (0, 40), (9, 30), (14, 5), (0, 7), (1, 2)]
    slots, pos = runs_to_slots(rng, runs, 40)
    rows = len(slots)
    qkv = torch.randn(rows, (hq + 2 * hk) * 128, device="cuda", generator=g).to(torch.bfloat16)
    qkv[:, (hq + hk) * 128:] *= torch.pow(2.0, torch.randint(-9, 9, (rows, 1), device="cuda", generator=g)).to(torch.bfloat16)
    w = weights(g)
    kv, sc = random_cache(g, 40, hk, fmt)
    ref = R.Cache(kv, sc, hk)
    q, k = write(qkv, pos, slots, kv, sc, hq, hk, w)
    heads = qkv.view(rows, -1, 128).cpu()
    check_turned(q, heads[:, :hq], w[0].cpu(), pos)
    check_turned(k, heads[:, hq:hq + hk], w[1].cpu(), pos)
    ref.write(slots, k.cpu().double().view(rows, hk, 128), heads[:, hq + hk:].double())
    ref.same_as(kv, sc)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("hq,hk", [(16, 8), (10, 5), (7, 1), (1, 1), (3, 3), (40, 20), (33, 33)])
def test_write_of_many_rows(fmt, hq, hk):
    """Calls of 131,072 heads and more over their rows (other kernels): runs at every place of a block, single rows,
    skipped rows and a slot given twice among them; and the bits of calls of few rows."""
    g, rng = gen(hq + hk), np.random.default_rng(hq)
    runs = [(0, 90), (5, 1), (15, 1), (3, 200), (0, 16), (9, 30), (0, 1), (14, 5), (7, 9), (0, 7)] + [(i % 16, 1) for i in range(40)]
    runs += [(0, 900), (11, 800), (2, 3)]
    runs += [(0, max(0, 131072 // (hq + 2 * hk) - 2000))]
    blocks = 220 + runs[-1][1] // 16
    slots, pos = runs_to_slots(rng, runs, blocks)
    slots[100] = -1
    slots[120] = slots[119]
    rows = len(slots)
    qkv = torch.randn(rows, (hq + 2 * hk) * 128, device="cuda", generator=g).to(torch.bfloat16)
    w = weights(g)
    kv, sc = random_cache(g, blocks, hk, fmt)
    ref, kv1, sc1 = R.Cache(kv, sc, hk), kv.clone(), sc.clone()
    q, k = write(qkv, pos, slots, kv, sc, hq, hk, w)
    heads = qkv.view(rows, -1, 128).cpu()
    there = torch.tensor(slots) >= 0
    check_turned(q.cpu()[there], heads[there, :hq], w[0].cpu(), torch.tensor(pos)[there].tolist())
    check_turned(k.cpu()[there], heads[there, hq:hq + hk], w[1].cpu(), torch.tensor(pos)[there].tolist())
    assert bool((q[~there] == 7).all()) and bool((k[~there] == 7).all())
    ref.write(slots, k.cpu().double().view(rows, hk, 128), heads[:, hq + hk:].double())
    ref.same_as(kv, sc)
    cuts = [0] + [n for n in range(1, rows) if slots[n] // 16 != slots[n - 1] // 16 and slots[n] >= 0 and slots[n - 1] >= 0]
    assert rows * (hq + 2 * hk) >= 131072
    cuts = [n for i, n in enumerate(cuts) if i % 3 == 0] + [rows]
    for a, b in zip(cuts, cuts[1:]):
        q1, k1 = write(qkv[a:b].contiguous(), pos[a:b], slots[a:b], kv1, sc1, hq, hk, w)
        assert torch.equal(q1, q[a:b]) and torch.equal(k1, k[a:b])
    ref.same_as(kv1, sc1)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows", [37, 2100])
@pytest.mark.parametrize("hq,hk", [(1, 1), (4, 2), (3, 3), (10, 5), (16, 8)])
def test_write_of_rows_alone_in_their_blocks(fmt, rows, hq, hk):
    """One token a sequence, at every place of a block, of every size, a few with infinities and NaN, some skipped, two
    pairs of rows next to one another in one block."""
    g, rng = gen(rows + hk), np.random.default_rng(rows)
    slots = [int(b) * 16 + i % 16 for i, b in enumerate(rng.permutation(rows + 9)[:rows])]
    for i in (5, 30):
        slots[i] = slots[i - 1] ^ 1
    for i in (0, 11, rows - 2):
        slots[i] = -1
    pos = rng.integers(0, 60000, rows).tolist()
    qkv = torch.randn(rows, (hq + 2 * hk) * 128, device="cuda", generator=g) * 2.0 ** torch.randint(-9, 9, (rows, 1), device="cuda", generator=g)
    qkv = qkv.to(torch.bfloat16)
    for i, x in enumerate((float("inf"), float("-inf"), float("nan"))):
        qkv[i + 1::17, (hq + hk) * 128 + 3 + 50 * i] = x
        qkv[i + 6::23, hq * 128 + 7 + 40 * i] = x
    qkv[3::11, (hq + hk) * 128:] = 0
    w = weights(g)
    kv, sc = random_cache(g, rows + 9, hk, fmt)
    ref = R.Cache(kv, sc, hk)
    _, k = write(qkv, pos, slots, kv, sc, hq, hk, w)
    ref.write(slots, k.cpu().double().view(rows, hk, 128), qkv.view(rows, -1, 128)[:, hq + hk:].cpu().double())
    ref.same_as(kv, sc)


@pytest.mark.parametrize("fmt", FORMATS)
def test_tokens_appended_one_by_one(fmt):
    """40 steps of five sequences that grow by one token, whose size rises and falls: the cache follows the host's at every step."""
    hq, hk, seqs = 4, 2, 5
    g, rng = gen(3), np.random.default_rng(3)
    kv, sc = random_cache(g, 24, hk, fmt)
    ref = R.Cache(kv, sc, hk)
    blocks = rng.permutation(24)[:20].reshape(seqs, 4)
    start = [0, 3, 16, 9, 1]
    w = weights(g)
    for step in range(40):
        pos = [s + step for s in start]
        slots = [int(blocks[i, p // 16]) * 16 + p % 16 if p < 64 else -1 for i, p in enumerate(pos)]
        qkv = (torch.randn(seqs, (hq + 2 * hk) * 128, device="cuda", generator=g) * 2.0 ** rng.integers(-6, 7)).to(torch.bfloat16)
        _, k = write(qkv, pos, slots, kv, sc, hq, hk, w)
        ref.write(slots, k.cpu().double().view(seqs, hk, 128), qkv.view(seqs, -1, 128)[:, hq + hk:].cpu().double())
        ref.same_as(kv, sc)


@pytest.mark.parametrize("fmt", FORMATS)
def test_write_of_extreme_values(fmt):
    """Infinities, NaN, zeros, the type's largest and smallest values in V; skipped rows write nothing."""
    hq, hk = 2, 2
    g, rng = gen(9), np.random.default_rng(9)
    slots, pos = runs_to_slots(rng, [(0, 16), (4, 3), (0, 2), (7, 1), (0, 1)], 12)
    rows = len(slots)
    qkv = torch.randn(rows, (hq + 2 * hk) * 128, device="cuda", generator=g).to(torch.bfloat16)
    v = qkv[:, (hq + hk) * 128:]
    v[0, 3], v[1, 200], v[2, 5], v[16, 0], v[17, :] = math.inf, -math.inf, math.nan, math.nan, 0
    v[19, :] = 0
    v[20, 1] = 3e38
    v[21] = torch.tensor(1e-39).to(torch.bfloat16)
    v[22, :] = math.inf
    skip = [6, 18]
    for n in skip:
        slots[n] = -1
    w = weights(g)
    kv, sc = random_cache(g, 12, hk, fmt)
    ref = R.Cache(kv, sc, hk)
    q, k = write(qkv, pos, slots, kv, sc, hq, hk, w)
    ref.write(slots, k.cpu().double().view(rows, hk, 128), v.cpu().double().view(rows, hk, 128))
    ref.same_as(kv, sc)
    for n in skip:
        assert bool((q[n] == 7).all()) and bool((k[n] == 7).all())


@pytest.mark.parametrize("fmt", FORMATS)
def test_write_of_rows_in_any_order_and_twice(fmt):
    """The rows of a block in another order, with gaps, among rows of other blocks, a slot given twice."""
    hq, hk = 1, 2
    g = gen(21)
    slots = [5, 37, 4, 33, 7, 7, 160, -1, 46, 2, 161, 80, 5]
    pos = list(range(len(slots)))
    qkv = torch.randn(len(slots), (hq + 2 * hk) * 128, device="cuda", generator=g).to(torch.bfloat16)
    kv, sc = random_cache(g, 11, hk, fmt)
    ref = R.Cache(kv, sc, hk)
    _, k = write(qkv, pos, slots, kv, sc, hq, hk, weights(g))
    there = torch.tensor(slots) >= 0
    k = k.cpu().double().view(len(slots), hk, 128)
    assert bool((k[~there] == 7).all()) and bool((k[there] != 7).any(-1).all())
    ref.write(slots, k, qkv.view(len(slots), -1, 128)[:, hq + hk:].cpu().double())
    ref.same_as(kv, sc)


def test_write_in_place_strided_and_without_k():
    hq, hk, rows = 6, 2, 37
    g, rng = gen(4), np.random.default_rng(4)
    slots, pos = runs_to_slots(rng, [(2, 37)], 8)
    wide = torch.randn(rows, (hq + 2 * hk) * 128 + 72, device="cuda", generator=g).to(torch.bfloat16)
    qkv = wide[:, 64:64 + (hq + 2 * hk) * 128]
    w = weights(g)
    kv, sc = random_cache(g, 8, hk, torch.int8)
    kv0, sc0 = kv.clone(), sc.clone()
    want_q, want_k = write(qkv.contiguous(), pos, slots, kv, sc, hq, hk, w)
    for in_place in (False, True):
        kv1, sc1, rows_in = kv0.clone(), sc0.clone(), wide.clone()
        src = rows_in[:, 64:64 + (hq + 2 * hk) * 128]
        if in_place:
            oa.qwen3_rope_q8(src, w[0], w[1], i32(pos), i32(slots), src[:, :hq * 128], src[:, hq * 128:(hq + hk) * 128], kv1,
                             sc1, hq, hk, EPS, THETA)
            q, k = src[:, :hq * 128], src[:, hq * 128:(hq + hk) * 128]
            assert torch.equal(k, want_k)
            assert torch.equal(src[:, (hq + hk) * 128:], qkv[:, (hq + hk) * 128:])
        else:
            q, _ = write(src, pos, slots, kv1, sc1, hq, hk, w, k_out=False)
            assert torch.equal(rows_in, wide)
        assert torch.equal(q, want_q) and torch.equal(kv1, kv) and torch.equal(sc1.view(torch.uint8), sc.view(torch.uint8))
        assert torch.equal(rows_in[:, :64], wide[:, :64]) and torch.equal(rows_in[:, -8:], wide[:, -8:])


@pytest.mark.parametrize("theta", [0.5, 1.0, 1e4, 1e6, 5e6])
def test_far_positions(theta):
    """2^31 positions of a turn that theta below 1 speeds up leave 2^-20 of the f64 angle."""
    hq, hk = 4, 1
    pos = [0, 1, 40959, 65537, 1 << 20, (1 << 24) + 1, (1 << 30) + 12345, (1 << 31) - 2]
    g = gen(6)
    qkv = torch.randn(8, 6 * 128, device="cuda", generator=g).to(torch.bfloat16)
    w = weights(g)
    kv, sc = random_cache(g, 8, hk, torch.int8)
    q, k = write(qkv, pos, [16 * i for i in range(8)], kv, sc, hq, hk, w, theta=theta)
    heads = qkv.view(8, -1, 128).cpu()
    check_turned(q, heads[:, :hq], w[0].cpu(), pos, theta)
    check_turned(k, heads[:, hq:hq + 1], w[1].cpu(), pos, theta)


def test_heads_of_zeros_and_of_overflowing_squares():
    """A head of zeros stays zero (eps keeps 1 / rms finite); where the f32 sum of squares overflows, 1 / rms is 0 and so is the head."""
    hq, hk = 2, 1
    qkv = torch.randn(3, 4 * 128, device="cuda", generator=gen(2)).to(torch.bfloat16)
    qkv[0, :128], qkv[1, 128:256], qkv[2, 256:384] = 0, 1e30, 3e38
    kv, sc = random_cache(gen(2), 3, hk, torch.float8_e4m3fn)
    q, k = write(qkv, [5, 6, 7], [0, 16, 32], kv, sc, hq, hk, weights(gen(2)))
    assert bool((q[0, :128] == 0).all()) and bool((q[1, 128:] == 0).all()) and bool((k[2] == 0).all())
    assert bool(q.isfinite().all()) and bool(k.isfinite().all())
    assert bool((kv.float()[2, 0] == 0).all()) and int(sc.view(torch.uint8)[2, 0]) == 1


# ------------------------------------------------------------------- decode
class Decode:
    """Sequences of given lengths over a permuted pool; unread tokens of their blocks hold NaN bytes."""

    def __init__(self, lens, hq, hk, page, fmt, seed=0, rows_of=None):
        self.hq, self.hk, self.page, self.fmt = hq, hk, page, fmt
        g, rng = gen(seed), np.random.default_rng(seed)
        per = page // 16
        need = [(n + page - 1) // page for n in lens]
        pool = sum(need) + 3
        self.kv, self.sc = random_cache(g, pool * per, hk, fmt)
        ids = rng.permutation(pool)
        self.indptr = np.concatenate([[0], np.cumsum(need)]).astype(np.int32)
        self.pages = ids[:self.indptr[-1]].astype(np.int32)
        # (sequence, position) of each row; by default one row per sequence at its last token
        self.rows = [(s, n - 1) for s, n in enumerate(lens)] if rows_of is None else rows_of
        if fmt == torch.float8_e4m3fn:
            raw = self.kv.view(torch.uint8)
            for s, n in enumerate(lens):
                last = -1 if n == 0 else n - 1
                for t in range(last + 1, need[s] * page):
                    b = int(self.pages[self.indptr[s] + t // page]) * per + t % page // 16
                    raw[b, :hk].view(hk, 16, 128)[:, t % 16] = 0x7F
                    raw[b, hk:].view(hk, 128, 16)[:, :, t % 16] = 0xFF
        self.q = torch.randn(len(self.rows), hq * 128, device="cuda", generator=g).to(torch.bfloat16)
        self.out = torch.full((len(self.rows), hq * 128), 7.0, dtype=torch.bfloat16, device="cuda")

    def run(self, max_len=None, chunk=0, ragged=True, scale=128 ** -0.5, plan=None, ws=None, stream=None):
        pos = [p for _, p in self.rows]
        plan = plan or oa.decode_plan_q8(len(self.rows), self.hq, self.hk, self.page, max_len or max(1, max(pos) + 1), chunk)
        oa.qwen3_attend_q8(self.q, self.kv, self.sc, i32(pos), i32([s for s, _ in self.rows]) if ragged else None, ragged,
                           i32(self.indptr), i32(self.pages), self.page, self.out, self.hq, self.hk, scale, plan,
                           oa.workspace_for(plan) if ws is None else ws, stream)
        torch.cuda.synchronize()
        return self.out

    def check(self, scale=128 ** -0.5):
        """Half a bf16 step of the result, and 2^-13 of sum p |v| for P in 16 bits, the base-2 exponentials and f32 sums over scores of
        up to some hundreds."""
        per = self.page // 16
        k, v = R.Cache(self.kv, self.sc, self.hk).tokens()
        got = self.out.double().cpu().view(len(self.rows), self.hq, 128)
        for n, (s, p) in enumerate(self.rows):
            t = np.arange(p + 1)
            slots = self.pages[self.indptr[s] + t // self.page].astype(np.int64) * self.page + t % self.page if p >= 0 else t
            want, size = R.attend(self.q[n].cpu().view(self.hq, 128), k[slots], v[slots], scale)
            bound = 2.0 ** -8 * want.abs() + 2.0 ** -13 * size
            d = (got[n] - want).abs()
            assert bool((d <= bound).all()), f"row {n}, {p + 1} keys: {float((d - bound).max()):.3g} past its bound"
        assert per >= 1


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("hq,hk", [(1, 1), (4, 4), (16, 8), (12, 4), (32, 8), (5, 1), (14, 2), (8, 1), (32, 2), (15, 1)])
def test_decode_matches_64_bits(fmt, hq, hk):
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300, 511, 700]
    d = Decode(lens, hq, hk, 16, fmt, seed=hq)
    d.run(ragged=False)
    d.check()


@pytest.mark.parametrize("page", [16, 32, 48, 64, 80, 256])
@pytest.mark.parametrize("chunk", [0, 64, 128, 192, 1024])
def test_decode_pages_and_splits(page, chunk):
    d = Decode([1, 40, 129, 500, 1000, 1025], 8, 2, page, FORMATS[chunk % 3 % 2], seed=page)
    d.run(chunk=chunk)
    d.check()


def test_decode_rows_longer_than_the_plan():
    d = Decode([900, 70, 2000, 1], 16, 8, 16, torch.int8, seed=2)
    d.run(max_len=300, chunk=64)
    d.check()


@pytest.mark.parametrize("fmt", FORMATS)
def test_decode_ragged_rows_and_rows_without_keys(fmt):
    """Several rows of one sequence, out of order, and padding rows (position -1, sequence -1), which store zeros."""
    rows = [(1, 10), (0, 99), (1, 44), (-1, -1), (0, 0), (0, 16), (1, 10), (-1, -1)]
    d = Decode([100, 45], 16, 8, 16, fmt, seed=1, rows_of=rows)
    d.run(chunk=64)
    d.check()
    assert bool((d.out[3] == 0).all()) and bool((d.out[7] == 0).all())


@pytest.mark.parametrize("fmt", FORMATS)
def test_decode_of_large_scores(fmt):
    """Scores of some hundreds: one key takes nearly all the weight."""
    d = Decode([200, 33, 700], 8, 4, 16, fmt, seed=7)
    d.sc.view(torch.uint8)[:, :4] += 4
    d.run(chunk=128)
    d.check()


def test_decode_reads_no_page_past_the_row():
    """Page ids past a row's last key point far outside the cache: they are not followed."""
    d = Decode([17, 16, 100], 4, 2, 16, torch.int8, seed=3)
    d.rows = [(0, 3), (1, 15), (2, 63)]
    used = {int(d.indptr[s]) + t // 16 for s, p in d.rows for t in range(p + 1)}
    for i in range(len(d.pages)):
        if i not in used:
            d.pages[i] = 0
    d.run(chunk=64)
    d.check()


def test_decode_keeps_a_nan_in_its_head():
    """A NaN among the keys of one head is that head's alone."""
    d = Decode([130], 4, 2, 16, torch.float8_e4m3fn, seed=5)
    d.kv.view(torch.uint8)[int(d.pages[3]), 2].view(128, 16)[7, 2] = 0x7F  # V head 0, dim 7
    out = d.run(ragged=False).view(4, 128).float()
    assert bool(out[:2, 7].isnan().all()) and int(out.isnan().sum()) == 2


def test_decode_offsets_past_32_bits():
    hq, hk, page = 4, 8, 16
    blocks = (5 << 30) // (2 * hk * 2048)
    hq = 16
    kv, sc = oa.q8_cache(blocks, page, hk, torch.int8)
    g = gen(8)
    d = Decode([40, 100], hq, hk, page, torch.int8, seed=8)
    far = blocks - d.kv.shape[0]
    kv[far:], sc.view(torch.uint8)[far:] = d.kv, d.sc.view(torch.uint8)
    small = d.run(ragged=False).clone()
    near_kv, near_sc, near = d.kv, d.sc, d.pages.copy()
    d.kv, d.sc, d.pages = kv, sc, d.pages + far
    d.out.zero_()
    assert torch.equal(d.run(ragged=False), small)
    # and the writer: the last block of the large cache
    slot = (blocks - 1) * 16 + 3
    w = weights(g)
    qkv = torch.randn(1, (hq + 2 * hk) * 128, device="cuda", generator=g).to(torch.bfloat16)
    write(qkv, [3], [slot], kv, sc, hq, hk, w)
    write(qkv, [3], [slot - far * 16], near_kv, near_sc, hq, hk, w)
    assert torch.equal(kv[-1], near_kv[-1]) and torch.equal(sc.view(torch.uint8)[-1], near_sc.view(torch.uint8)[-1])
    assert len(near) == len(d.pages)


def test_decode_strided_queries_and_another_stream():
    d = Decode([70, 5, 300], 8, 2, 16, torch.int8, seed=4)
    want = d.run(chunk=128).clone()
    wide = torch.zeros(3, 8 * 128 + 40, dtype=torch.bfloat16, device="cuda")
    wide[:, 8:8 + 8 * 128] = d.q
    d.q = wide[:, 8:8 + 8 * 128]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    d.out.zero_()
    torch.cuda.synchronize()
    assert torch.equal(d.run(chunk=128, stream=s), want)


def test_decode_replays_with_new_lengths():
    """One capture serves every length up to the plan's, and gives the eager bits each time."""
    d = Decode([600] * 5, 16, 8, 16, torch.float8_e4m3fn, seed=6)
    plan = oa.decode_plan_q8(5, 16, 8, 16, 600, 128)
    ws, pos = oa.workspace_for(plan), i32([0] * 5)
    indptr, pages = i32(d.indptr), i32(d.pages)
    call = lambda s=None: oa.qwen3_attend_q8(d.q, d.kv, d.sc, pos, None, 0, indptr, pages, 16, d.out, 16, 8, 0.09, plan, ws, s)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        call()
    for lens in ([599, 0, 63, 64, 300], [-1, 5, 599, 128, 127], [10, 20, 30, 40, 50], [599] * 5):
        pos.copy_(i32(lens))
        call()
        torch.cuda.synchronize()
        want = d.out.clone()
        d.out.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(d.out, want)


@pytest.mark.parametrize("hk", [1, 3, 8, 300])
@pytest.mark.parametrize("rows", [2, 33, 65, 257, 600])
def test_decode_of_many_rows_in_any_order_of_lengths(rows, hk):
    """Rows of lengths in falling, rising and random order, equal, far longer than the plan and without keys, in one split
    each: every row keeps the bits that it has alone."""
    if rows * hk > 20000:
        rows = 20000 // hk
    g, rng = gen(rows + hk), np.random.default_rng(rows)
    kv, sc = random_cache(g, 40, hk, torch.int8)
    q = torch.randn(rows, hk * 128, device="cuda", generator=g).to(torch.bfloat16)
    lens = np.minimum(rng.integers(-1, 600, rows), 500)
    lens[rows // 2:] = np.sort(lens[rows // 2:])
    if rows > 40:
        lens[30:60] = 77
    pages = i32([rng.permutation(40)[:38] for _ in range(rows)])
    indptr = i32(np.arange(rows + 1) * 38)
    out = torch.zeros(rows, hk * 128, dtype=torch.bfloat16, device="cuda")

    def run(lo, hi):
        plan = oa.decode_plan_q8(hi - lo, hk, hk, 16, 128, 128)
        assert plan.splits == 1
        o = torch.full((hi - lo, hk * 128), 3.0, dtype=torch.bfloat16, device="cuda")
        oa.qwen3_attend_q8(q[lo:hi], kv, sc, i32(lens[lo:hi] - 1), None, 0, indptr[lo:], pages.view(-1), 16, o, hk, hk, 0.09,
                           plan, oa.workspace_for(plan))
        return o

    out = run(0, rows)
    few = max(1, 256 // hk)
    alone = torch.cat([run(lo, min(lo + few, rows)) for lo in range(0, rows, few)])
    assert torch.equal(out, alone)
    assert bool((out[torch.from_numpy(lens <= 0).cuda()] == 0).all())


def test_decode_rows_without_keys_may_name_any_sequence():
    d = Decode([40, 20], 4, 2, 16, torch.int8, rows_of=[(0, 39), (2 ** 31 - 1, -1), (1, 19), (-7, -5)])
    d.run(max_len=64)
    assert bool((d.out[[1, 3]] == 0).all())
    d.rows = [(0, 39), (0, -1), (1, 19), (1, -1)]
    want = d.out.clone()
    d.out.fill_(7)
    d.run(max_len=64)
    assert torch.equal(d.out, want)
