"""The operators of a serving step over an 8-bit paged cache, as measurable cases.

A Qwen3 engine's step is four calls: the step's row tables are built on the GPU from the
request lengths; each new row's q and k are normalised and turned, and K and V written to a
cache of 8-bit values with one power-of-two scale per 16 tokens and head; prompts attend to
themselves, packed one behind the other; single new tokens attend to the cache. The kinds:

- ``tables``: positions, slots, sequences, page lists and page allocation of one step.
- ``write``: RMSNorm + rotary of q and k, and the quantized cache write.
- ``decode``: paged attention of one new row per sequence over the 8-bit cache.
- ``prompt``: causal attention of whole prompts, packed.

Lengths follow from the case alone (spread evenly over their range, in a mixed order);
values, page tables and slots follow from the seed.
"""
import math
import os
import random
import sys

import torch

own = False

HEAD = 128
BLOCK = 16  # tokens that share a scale
SCALE = 1.0 / math.sqrt(HEAD)
EPS, THETA = 1e-6, 1e6
FORMATS = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


def _oa():
    at = os.path.join(os.getcwd(), "pega-omni_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import omni_attn

    return omni_attn


def listed():
    return [
        # A decode step of the talker's full batch bucket: one new row each, a page now and then.
        dict(name="tables_64", kind="tables", decode=64, prompts=0, done=0, ctx=2400, new_lo=1, new_hi=1),
        # A busy step: 96 running sequences, 24 prompts of up to 4096 rows admitted, 8 requests done.
        dict(name="tables_mixed", kind="tables", decode=96, prompts=24, done=8, ctx=5120, new_lo=30, new_hi=4096),
        # The cache write of a decode step: 64 rows, each into its own block.
        dict(name="write_64", kind="write", seqs=64, hq=16, hk=8, lo=1, hi=1, cached=2400, fmt="e4m3"),
        # One TTS request's prompt of 187 rows.
        dict(name="write_187", kind="write", seqs=1, hq=16, hk=8, lo=187, hi=187, cached=0, fmt="e4m3"),
        # Chunked prefill of Higgs requests behind what each has cached: the largest write.
        dict(name="write_prefill", kind="write", seqs=12, hq=32, hk=8, lo=512, hi=4096, cached=1024, fmt="e4m3"),
        # A single session late in its context: latency.
        dict(name="decode_1", kind="decode", rows=1, hq=16, hk=8, lo=2400, hi=2400, page=16, fmt="e4m3"),
        # The talker's full batch bucket.
        dict(name="decode_64", kind="decode", rows=64, hq=16, hk=8, lo=200, hi=2400, page=16, fmt="e4m3"),
        # 128 sessions of a 32-head MHA model, integers in the cache: the largest tick.
        dict(name="decode_mha_128", kind="decode", rows=128, hq=32, hk=32, lo=100, hi=3000, page=16, fmt="int8"),
        # Few sessions over very long contexts, in larger pages.
        dict(name="decode_long", kind="decode", rows=4, hq=32, hk=8, lo=100000, hi=130000, page=64, fmt="e4m3"),
        # One TTS request's prompt of 187 rows: latency.
        dict(name="prompt_187", kind="prompt", seqs=1, hq=16, hk=8, lo=187, hi=187),
        # Twelve Higgs prompts of mixed lengths in one call.
        dict(name="prompt_pack", kind="prompt", seqs=12, hq=32, hk=8, lo=300, hi=4000),
        # One long prompt: the largest.
        dict(name="prompt_16k", kind="prompt", seqs=1, hq=32, hk=8, lo=16384, hi=16384),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["tables", "write", "write", "decode", "decode", "prompt", "prompt"])
    if kind == "tables":
        hi = _log(rng, 1, 4096)
        return dict(kind=kind, decode=_log(rng, 1, 512), prompts=_log(rng, 1, max(2, min(25, 48000 // hi))) - 1, done=_log(rng, 1, 17) - 1,
                    ctx=_log(rng, 1, 8192), new_lo=max(1, hi // rng.randint(1, 8)), new_hi=hi)
    hk = rng.choice([1, 2, 4, 8, 8, 8, 16])
    if kind == "write":
        hi = _log(rng, 1, 4096)
        return dict(kind=kind, seqs=_log(rng, 1, max(1, min(128, 192000 // max(8, hk) // hi))),
                    hq=hk * rng.choice([1, 2, 2, 4]), hk=hk,
                    lo=max(1, hi // rng.randint(1, 8)), hi=hi, cached=_log(rng, 1, 4096) - 1, fmt="e4m3")
    if kind == "decode":
        hi = _log(rng, 1, 40000)
        rows = _log(rng, 1, max(1, min(128, 380000 // hi)))
        return dict(kind=kind, rows=rows, hq=hk * rng.choice([1, 2, 2, 4, 4, 5, 7, 8, 16]), hk=hk,
                    lo=max(1, hi // rng.randint(1, 20)), hi=hi, page=rng.choice([16, 16, 32, 64, 256]),
                    fmt=rng.choice(["e4m3", "int8"]))
    hi = _log(rng, 1, 5000)
    return dict(kind=kind, seqs=_log(rng, 1, max(1, min(48, 24000 // hi))),
                hq=hk * rng.choice([1, 2, 2, 4, 4, 8][:3 if hk > 8 else 6]), hk=hk, lo=max(1, hi // rng.randint(1, 8)), hi=hi)


# ------------------------------------------------------------------ inputs
def spread(n, lo, hi):
    """n whole numbers spread evenly over [lo, hi], in a mixed order."""
    return [lo + int((hi - lo + 1) * (((i + 0.5) * 0.6180339887498949) % 1.0)) for i in range(n)]


def _i32(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)


def _normal(gen, *shape):
    return torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(generator=gen)


def _step(case):
    """(first position, new rows) of each sequence of a tables case; -1 rows: the request is done."""
    n, m, d = case["decode"], case["prompts"], case["done"]
    seqs = [(c, 1) for c in spread(n, 0, case["ctx"])]
    seqs += [(0 if i % 3 else case["ctx"] // 5, c) for i, c in enumerate(spread(m, case["new_lo"], case["new_hi"]))]
    return seqs + [(c, -1) for c in spread(d, 1, case["ctx"] + 1)]


def _write_rows(case):
    """(first position, new rows) of each sequence of a write case."""
    new = spread(case["seqs"], case["lo"], case["hi"])
    return list(zip([c for c in spread(case["seqs"], 0, case["cached"])] if case["cached"] else [0] * len(new), new))


def _cache(gen, blocks, hk, fmt):
    """Bytes and scales of a cache in use: values of about unit size."""
    x = _normal(gen, blocks, 2 * hk, HEAD * BLOCK)
    if fmt == "e4m3":
        kv = (x * 100).clamp_(-448, 448).to(torch.float8_e4m3fn)
        mid = 120
    else:
        kv = (x * 36).round_().clamp_(-127, 127).to(torch.int8)
        mid = 122
    exps = torch.randint(mid - 1, mid + 2, (blocks, 2 * hk), dtype=torch.uint8, device="cuda", generator=gen)
    return kv, exps.view(torch.float8_e8m0fnu)


def prepare(case, seed):
    gen, rng, kind = _gen(seed), random.Random(int(seed)), case["kind"]
    st = dict(case)
    if kind == "tables":
        seqs = _step(case)
        page, width = 16, (case["ctx"] + 1 + max(1, case["new_hi"]) + 15) // 16 + 1
        held = [(f + page - 1) // page for f, _ in seqs]
        need = [(f + c + page - 1) // page if c >= 0 else 0 for f, c in seqs]
        new = sum(max(0, b - a) for a, b in zip(held, need))
        pool = sum(held) + new + 64
        ids = list(range(pool))
        rng.shuffle(ids)
        lines = list(range(len(seqs) + 8))
        rng.shuffle(lines)
        table, at = [[-1] * width for _ in lines], 0
        for s, h in enumerate(held):
            table[lines[s]][:h] = ids[at:at + h]
            at += h
        head = rng.randrange(pool)  # the free pages lie from here on, round the end
        free = [-1] * pool
        for i, p in enumerate(ids[at:]):
            free[(head + i) % pool] = p
        rows, npages = sum(max(0, c) for _, c in seqs), sum(need)
        rows = (rows + 63) // 64 * 64  # the batch bucket
        st.update(first=_i32([f for f, _ in seqs]), count=_i32([c for _, c in seqs]), lines=_i32(lines[:len(seqs)]),
                  table=_i32(table), free_pages=_i32(free), free_state=_i32([head, pool - at]))
        for name, n in (("pos", rows), ("slots", rows), ("seq", rows), ("row_indptr", len(seqs) + 1),
                        ("indptr", len(seqs) + 1), ("pages", npages + 16), ("status", 5)):
            st[name] = torch.zeros(n, dtype=torch.int32, device="cuda")
        return st
    hq, hk = case["hq"], case["hk"]
    if kind == "write":
        seqs = _write_rows(case)
        # The sequences' blocks from the one that holds the first new row on, anywhere in the pool.
        need = [(f + c - 1) // BLOCK - f // BLOCK + 1 for f, c in seqs]
        blocks = sum(need) + 16
        ids = list(range(blocks))
        rng.shuffle(ids)
        pos, slots, at = [], [], 0
        for (f, c), n in zip(seqs, need):
            for p in range(f, f + c):
                pos.append(p)
                slots.append(ids[at + p // BLOCK - f // BLOCK] * BLOCK + p % BLOCK)
            at += n
        rows = len(pos)
        st["kv"], st["kv_scale"] = _cache(gen, blocks, hk, case["fmt"])
        st["qkv"] = _normal(gen, rows, (hq + 2 * hk) * HEAD)
        for name in ("q_norm", "k_norm"):
            st[name] = (1.0 + 0.2 * torch.randn(HEAD, device="cuda", generator=gen)).to(torch.bfloat16)
        st["pos"], st["slots"] = _i32(pos), _i32(slots)
        st["q"] = torch.zeros(rows, hq * HEAD, dtype=torch.bfloat16, device="cuda")
        st["k"] = torch.zeros(rows, hk * HEAD, dtype=torch.bfloat16, device="cuda")
        return st
    if kind == "decode":
        lens = spread(case["rows"], case["lo"], case["hi"])
        page = case["page"]
        need = [(n + page - 1) // page for n in lens]
        pool = sum(need) + 16
        ids = torch.randperm(pool, device="cuda", generator=gen).to(torch.int32)
        st["kv"], st["kv_scale"] = _cache(gen, pool * (page // BLOCK), hk, case["fmt"])
        st["qrows"] = _normal(gen, case["rows"], hq * HEAD)
        indptr = [0]
        for n in need:
            indptr.append(indptr[-1] + n)
        st["indptr"], st["pages"] = _i32(indptr), ids[:indptr[-1]].contiguous()
        st["pos"] = _i32([n - 1 for n in lens])
        st["out"] = torch.zeros(case["rows"], hq * HEAD, dtype=torch.bfloat16, device="cuda")
        st["most"] = max(lens)
        if own:
            st["plan"] = _oa().decode_plan_q8(case["rows"], hq, hk, page, max(lens))
            st["ws"] = _oa().workspace_for(st["plan"])
        return st
    lens = spread(case["seqs"], case["lo"], case["hi"])
    rows = sum(lens)
    st["qkv"] = _normal(gen, rows, (hq + 2 * hk) * HEAD)
    st["lens"], st["most"] = _i32(lens), max(lens)
    st["out"] = torch.zeros(rows, hq * HEAD, dtype=torch.bfloat16, device="cuda")
    if own:
        st["plan"] = _oa().prompt_plan(lens, hq, hk)
    return st


# ------------------------------------------------------------------ one pass
def run(st):
    kind = st["kind"]
    if not own:
        return {"tables": _tables, "write": _write, "decode": _decode, "prompt": _prompt}[kind](st)
    oa = _oa()
    if kind == "tables":
        oa.step_tables(st["first"], st["count"], st["lines"], st["table"], st["free_pages"], st["free_state"], st["pos"],
                       st["slots"], st["seq"], st["row_indptr"], st["indptr"], st["pages"], st["status"], 16)
        return {n: st[n] for n in ("pos", "slots", "seq", "row_indptr", "indptr", "pages", "table", "free_pages", "status")}
    hq, hk = st["hq"], st["hk"]
    if kind == "write":
        oa.qwen3_rope_q8(st["qkv"], st["q_norm"], st["k_norm"], st["pos"], st["slots"], st["q"], st["k"], st["kv"],
                         st["kv_scale"], hq, hk, EPS, THETA)
        return {n: st[n] for n in ("q", "k", "kv", "kv_scale")}
    if kind == "decode":
        return oa.qwen3_attend_q8(st["qrows"], st["kv"], st["kv_scale"], st["pos"], None, 0, st["indptr"], st["pages"],
                                  st["page"], st["out"], hq, hk, SCALE, st["plan"], st["ws"])
    q, k, v = st["qkv"].split([hq * HEAD, hk * HEAD, hk * HEAD], dim=1)
    return oa.prompt_run(st["plan"], q, k, v, st["out"], SCALE)


def _owner(ends, x):
    """The sequence whose range [start, end) of a running total holds each x (the last one past the end)."""
    return torch.searchsorted(ends, x, right=True).clamp_(max=ends.numel() - 1)


def _tables(st):
    page = 16
    first, count, lines = st["first"].long(), st["count"].long(), st["lines"].long()
    table, free = st["table"].long(), st["free_pages"].long()
    head, avail, cap = st["free_state"][0].long(), st["free_state"][1].long(), free.numel()
    done = count < 0
    cnt = count.clamp(min=0)
    held = (first + page - 1) // page
    need = torch.where(done, 0, (first + cnt + page - 1) // page)
    new = (need - held).clamp(min=0)
    back = torch.where(done, held, 0)
    row_end, page_end, new_end, back_end = (x.cumsum(0) for x in (cnt, need, new, back))

    def page_of(s, j):
        """Page j of sequence s: one that it holds, or one that this step takes from the free pages."""
        taken = free[(head + (new_end - new)[s] + j - held[s]).clamp(min=0) % cap]
        return torch.where(j < held[s], table[lines[s], j.clamp(0, table.shape[1] - 1)], taken)

    r = torch.arange(st["pos"].numel(), device="cuda")
    s = _owner(row_end, r)
    p = first[s] + r - (row_end - cnt)[s]
    rows = r < row_end[-1]
    st["pos"].copy_(torch.where(rows, p, -1))
    st["slots"].copy_(torch.where(rows, page_of(s, p // page) * page + p % page, -1))
    st["seq"].copy_(torch.where(rows, s, -1))
    st["row_indptr"][1:].copy_(row_end)
    st["indptr"][1:].copy_(page_end)
    i = torch.arange(st["pages"].numel(), device="cuda")
    s = _owner(page_end, i)
    st["pages"].copy_(torch.where(i < page_end[-1], page_of(s, i - (page_end - need)[s]), st["pages"].long()))
    # New pages into the table, done requests' pages behind the free ones; what is neither goes to a spare last place.
    s = _owner(new_end, i)
    j = held[s] + i - (new_end - new)[s]
    spare = torch.where(i < new_end[-1], lines[s] * table.shape[1] + j, table.numel())
    flat = torch.cat([table.reshape(-1), table.new_zeros(1)])
    flat[spare] = page_of(s, j)
    i = torch.arange(cap, device="cuda")
    s = _owner(back_end, i)
    spare = torch.where(i < back_end[-1], (head + avail + i) % cap, cap)
    ring = torch.cat([free, free.new_zeros(1)])
    ring[spare] = table[lines[s], (i - (back_end - back)[s]).clamp(0, table.shape[1] - 1)]
    st["table"].copy_(flat[:-1].view_as(table))
    st["free_pages"].copy_(ring[:-1])
    st["status"].copy_(torch.stack([head * 0, row_end[-1], page_end[-1], (head + new_end[-1]) % cap,
                                    avail - new_end[-1] + back_end[-1]]))
    return {n: st[n] for n in ("pos", "slots", "seq", "row_indptr", "indptr", "pages", "table", "free_pages", "status")}


def _turned(x, weight, pos):
    """RMSNorm (the normalised value rounded to bf16, as the model does) and half-split rotary of heads x [rows, heads, 128]."""
    x = x.float()
    x = (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)).bfloat16().float() * weight.float()
    i = torch.arange(HEAD // 2, device="cuda", dtype=torch.float64)
    angle = pos.double()[:, None] * torch.pow(THETA, -2.0 * i / HEAD)  # far positions need the 64 bits
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    a, b = x[..., :HEAD // 2], x[..., HEAD // 2:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).bfloat16()


def _block_exponent(most, fmt):
    """The biased exponent of the smallest power of two that brings `most` into the format's range."""
    top = 448.0 if fmt == "e4m3" else 127.0
    m, e = torch.frexp(most)  # most = m 2^e, m in [0.5, 1)
    tm, te = math.frexp(top)
    return (e.long() - te + (m > tm).long() + 127).clamp(min=1) * (most > 0) + (most <= 0).long()


def _pow2(biased):
    """2^(biased - 127), exactly."""
    return (biased.int().clamp(min=1) << 23).view(torch.float32)


def _rounded(x, fmt):
    return x.to(torch.float8_e4m3fn) if fmt == "e4m3" else x.round().clamp(-127, 127).to(torch.int8)


def _write(st):
    hq, hk, fmt, rows = st["hq"], st["hk"], st["fmt"], st["pos"].numel()
    q, k, v = st["qkv"].view(rows, -1, HEAD).split([hq, hk, hk], dim=1)
    st["q"].copy_(_turned(q, st["q_norm"], st["pos"]).view(rows, -1))
    k = _turned(k, st["k_norm"], st["pos"])
    st["k"].copy_(k.view(rows, -1))
    slots = st["slots"].long()
    blocks = st["kv"].shape[0]
    written = torch.zeros(blocks * BLOCK, dtype=torch.bool, device="cuda").index_fill_(0, slots, True).view(blocks, BLOCK)
    touched = written.any(1)
    kept = touched & ~written[:, 0]  # tokens before the first new one stay
    raw = st["kv"].float().view(blocks, 2, hk, HEAD * BLOCK)
    old = torch.stack([raw[:, 0].view(blocks, hk, BLOCK, HEAD), raw[:, 1].view(blocks, hk, HEAD, BLOCK).transpose(2, 3)], 1)
    fresh = torch.zeros(blocks * BLOCK, 2, hk, HEAD, device="cuda")
    fresh[slots] = torch.stack([k, v], 1).float()
    fresh = fresh.view(blocks, BLOCK, 2, hk, HEAD).permute(0, 2, 3, 1, 4)
    was = st["kv_scale"].view(torch.uint8).long().view(blocks, 2, hk)
    least = torch.where(kept[:, None, None], was, 1)
    exps = torch.maximum(least, _block_exponent(fresh.abs().amax((3, 4)), fmt))
    shift = _pow2(was - exps + 127)[..., None, None]
    again = torch.where(kept[:, None, None, None, None], _rounded(old * shift, fmt).float(), 0.0)
    new = _rounded(fresh * _pow2(254 - exps)[..., None, None], fmt).float()
    out = torch.where(written[:, None, None, :, None], new, again)
    out = torch.where(touched[:, None, None, None, None], out, old)
    out = torch.stack([out[:, 0].reshape(blocks, hk, -1), out[:, 1].transpose(2, 3).reshape(blocks, hk, -1)], 1)
    st["kv"].copy_(out.view(blocks, 2 * hk, -1).to(st["kv"].dtype))
    st["kv_scale"].view(torch.uint8).copy_(torch.where(touched[:, None, None], exps, was).view(blocks, 2 * hk))
    return {n: st[n] for n in ("q", "k", "kv", "kv_scale")}


def _decode(st):
    rows, hq, hk, page, most = st["rows"], st["hq"], st["hk"], st["page"], st["most"]
    t = torch.arange((most + BLOCK - 1) // BLOCK * BLOCK, device="cuda")
    seen = t[None] <= st["pos"][:, None]
    b = t[::BLOCK]
    at = (st["indptr"][:-1, None] + b[None] // page).clamp(max=st["pages"].numel() - 1)
    block = st["pages"][at.long()].long() * (page // BLOCK) + b[None] % page // BLOCK
    scale = _pow2(st["kv_scale"].view(torch.uint8)[block])
    raw = st["kv"].view(torch.uint8)[block].view(st["kv"].dtype).float() * scale[..., None]  # [rows, blocks, 2 hk, 2048]
    k = raw[:, :, :hk].view(rows, -1, hk, BLOCK, HEAD).permute(0, 2, 4, 1, 3).reshape(rows, hk, HEAD, -1)
    v = raw[:, :, hk:].view(rows, -1, hk, HEAD, BLOCK).permute(0, 2, 1, 4, 3).reshape(rows, hk, -1, HEAD)
    s = torch.matmul(st["qrows"].float().view(rows, hk, hq // hk, HEAD), k) * SCALE
    s = s.masked_fill_(~seen[:, None, None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    return st["out"].copy_(o.view(rows, -1))


def _prompt(st):
    hq, hk, most, lens = st["hq"], st["hk"], st["most"], st["lens"].long()
    n, rows = lens.numel(), st["out"].shape[0]
    r = torch.arange(rows, device="cuda")
    s = _owner(lens.cumsum(0), r)
    p = r - (lens.cumsum(0) - lens)[s]
    padded = torch.zeros(n, most, hq + 2 * hk, HEAD, device="cuda")
    padded[s, p] = st["qkv"].float().view(rows, -1, HEAD)
    q, k, v = padded.transpose(1, 2).split([hq, hk, hk], dim=1)  # [n, heads, most, 128]
    q = q.reshape(n, hk, hq // hk * most, HEAD)
    x = torch.matmul(q, k.transpose(2, 3).contiguous()).view(n, hk, -1, most, most).mul_(SCALE)
    t = torch.arange(most, device="cuda")
    x.masked_fill_(t[None] > t[:, None], -math.inf)
    x.sub_(x.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(x.view(n, hk, -1, most), v.contiguous()).view(n, hk, -1, most, HEAD) / x.sum(-1, keepdim=True)
    return st["out"].copy_(o.view(n, hq, most, HEAD).transpose(1, 2)[s, p].reshape(rows, -1))


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    kind = case["kind"]
    if kind == "tables":
        seqs = _step(case)
        rows = sum(max(0, c) for _, c in seqs)
        need = sum((f + c + 15) // 16 for f, c in seqs if c >= 0)
        moved = sum((f + max(c, 0) + 15) // 16 - (f + 15) // 16 if c >= 0 else (f + 15) // 16 for f, c in seqs)
        return {"bytes": 4 * (3 * len(seqs) + 3 * rows + 2 * len(seqs) + 2 * need + 2 * moved), "flops": 0}
    hq, hk = case["hq"], case["hk"]
    if kind == "write":
        seqs = _write_rows(case)
        rows = sum(c for _, c in seqs)
        row = (2 * hq + 3 * hk) * HEAD * 2 + 2 * hk * HEAD  # the row read; q and k, and 8-bit K and V written
        kept = sum(f % BLOCK for f, _ in seqs)  # read for a scale that may grow
        blocks = sum((f + c - 1) // BLOCK - f // BLOCK + 1 for f, c in seqs)
        return {"bytes": rows * (row + 8) + kept * 2 * hk * HEAD + blocks * 2 * hk, "flops": rows * (hq + hk) * HEAD * 10}
    lens = spread(case.get("rows", case.get("seqs")), case["lo"], case["hi"])
    if kind == "decode":
        keys, blocks = sum(lens), sum((n + BLOCK - 1) // BLOCK for n in lens)
        return {"bytes": keys * 2 * hk * HEAD + blocks * 2 * hk + 4 * len(lens) * hq * HEAD, "flops": 4 * HEAD * hq * keys}
    rows = sum(lens)
    return {"bytes": rows * (2 * hq + 2 * hk) * HEAD * 2, "flops": sum(2 * HEAD * hq * n * (n + 1) for n in lens)}


# ------------------------------------------------------------------ in 64 bits
def _exact_pow2(e):
    return (e.long() + 1023 << 52).view(torch.float64)


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "tables":
        return None  # whole numbers
    hq, hk = case["hq"], case["hk"]
    if kind == "write":
        rows = st["pos"].numel()
        inv = torch.tensor([THETA ** (-2.0 * i / HEAD) for i in range(HEAD // 2)] * 2, dtype=torch.float64, device="cuda")
        angle = st["pos"].double()[:, None, None] * inv
        sign = torch.ones(HEAD, dtype=torch.float64, device="cuda")
        sign[:HEAD // 2] = -1
        heads = st["qkv"].double().view(rows, hq + 2 * hk, HEAD)

        def turned(x, w):
            x = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt()
            x = x.to(torch.bfloat16).double() * w.double()
            return x * angle.cos() + x.roll(HEAD // 2, -1) * sign * angle.sin()

        q, k = turned(heads[:, :hq], st["q_norm"]), turned(heads[:, hq:hq + hk], st["k_norm"])
        kv = st["kv"].double().clone()
        exps = st["kv_scale"].view(torch.uint8).clone()
        slots, step = st["slots"].long(), BLOCK
        new = torch.cat([k.to(torch.bfloat16).double(), heads[:, hq + hk:]], 1)  # [rows, 2 hk, 128]
        # Blocks that take new rows: their first new token's place, and each row's place in its block's list.
        b, inverse = torch.unique(slots // step, return_inverse=True)
        place = slots % step
        start = torch.full((b.numel(),), step, device="cuda").scatter_reduce(0, inverse, place, "amin")
        most = torch.zeros(b.numel(), 2 * hk, dtype=torch.float64, device="cuda")
        most = most.scatter_reduce(0, inverse[:, None].expand(-1, 2 * hk), new.abs().amax(-1), "amax")
        top = 448.0 if case["fmt"] == "e4m3" else 127.0
        e = torch.ceil(torch.log2(most / top)).clamp(min=-126)
        e = torch.where(top * _exact_pow2(e - 1) >= most, e - 1, e)  # log2 rounds
        e = torch.where(most > 0, e, torch.full_like(e, -126.0)).clamp(min=-126)
        old_e = exps[b].double() - 127
        e = torch.where((start > 0)[:, None], torch.maximum(e, old_e), e)
        kv_b = kv[b]
        as_tokens = torch.empty(b.numel(), 2 * hk, step, HEAD, dtype=torch.float64, device="cuda")
        as_tokens[:, :hk] = kv_b[:, :hk].view(-1, hk, step, HEAD)
        as_tokens[:, hk:] = kv_b[:, hk:].view(-1, hk, HEAD, step).transpose(2, 3)
        as_tokens *= (start > 0)[:, None, None, None] * _exact_pow2(old_e - e)[..., None, None]
        as_tokens[inverse, :, place] = new * _exact_pow2(-e)[inverse][..., None]
        as_tokens = as_tokens.float().to(FORMATS[case["fmt"]]).double() if case["fmt"] == "e4m3" else as_tokens.round()
        kv_b[:, :hk] = as_tokens[:, :hk].reshape(-1, hk, step * HEAD)
        kv_b[:, hk:] = as_tokens[:, hk:].transpose(2, 3).reshape(-1, hk, step * HEAD)
        kv[b] = kv_b
        exps[b] = (e + 127).to(torch.uint8)
        return {"q": q.view(rows, -1), "k": k.view(rows, -1), "kv": kv, "kv_scale": _exact_pow2(exps.double() - 127)}
    if kind == "decode":
        out = torch.zeros(case["rows"], hq, HEAD, dtype=torch.float64, device="cuda")
        page, indptr = case["page"], st["indptr"].tolist()
        for n, p in enumerate(st["pos"].tolist()):
            ids = st["pages"][indptr[n]:indptr[n + 1]].long()
            blocks = (ids[:, None] * (page // BLOCK) + torch.arange(page // BLOCK, device="cuda")).reshape(-1)
            factor = _exact_pow2(st["kv_scale"].view(torch.uint8)[blocks].double() - 127)
            raw = st["kv"].view(torch.uint8)[blocks].view(st["kv"].dtype).double() * factor[..., None]
            for h in range(hk):
                k = raw[:, h].reshape(-1, HEAD)[:p + 1]
                v = raw[:, hk + h].view(-1, HEAD, BLOCK).transpose(1, 2).reshape(-1, HEAD)[:p + 1]
                g = slice(h * (hq // hk), (h + 1) * (hq // hk))
                w = torch.softmax(st["qrows"][n].double().view(hq, HEAD)[g] @ k.t() * SCALE, -1)
                out[n, g] = w @ v
        return out.view(case["rows"], -1)
    if sum(n * n for n in st["lens"].tolist()) * hq > 1.2e10:
        return None
    out, at = torch.empty(st["out"].shape, dtype=torch.float64, device="cuda"), 0
    for n in st["lens"].tolist():
        x = st["qkv"][at:at + n].view(n, -1, HEAD)
        later = torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1)
        for h in range(hq):
            g = hq + h // (hq // hk)
            s = (x[:, h].double() @ x[:, g].double().t()) * SCALE
            out[at:at + n, h * HEAD:(h + 1) * HEAD] = torch.softmax(s.masked_fill(later, -math.inf), -1) @ x[:, g + hk].double()
        at += n
    return out
