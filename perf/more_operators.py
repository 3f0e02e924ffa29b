"""Operators around shared prefixes and encoder states, as measurable cases.

Candidates that are forked from one request share its cache pages and its encoder's states;
a prompt behind a shared prefix attends to keys that are in the cache already. The kinds:

- ``fork``: candidates take over their parent's pages (its part-filled page is copied, in every
  layer) and, when they have ended, give them back.
- ``compact``: a pool's pages in use move below a limit, with tables, holders and free queue.
- ``extend``: attention of several new rows per sequence over the 8-bit paged cache, causal.
- ``cross``: attention of packed rows to encoder states of other lengths.

Lengths follow from the case alone (spread evenly over their range, in a mixed order);
values, page tables and free queues follow from the seed.
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


def _oa():
    at = os.path.join(os.getcwd(), "pega-omni_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import omni_attn

    return omni_attn


def listed():
    return [
        # Eight candidates of one TTS prompt of 187 tokens, through the talker's 28 layers.
        dict(name="fork_8", kind="fork", parents=1, each=8, lo=187, hi=187, page=16, hk=8, layers=28),
        # A busy server: 32 requests of up to 4000 tokens, seven candidates each, four layers in a pool.
        dict(name="fork_224", kind="fork", parents=32, each=7, lo=100, hi=4000, page=16, hk=8, layers=4),
        # A small pool, half empty, shrinks to what it holds.
        dict(name="compact_small", kind="compact", lines=24, lo=64, hi=512, page=16, hk=8, layers=4, spare=1.0, keep=1.1),
        # 128 long requests in a pool with a third of its pages free.
        dict(name="compact_pool", kind="compact", lines=128, lo=200, hi=5000, page=16, hk=8, layers=1, spare=0.5, keep=1.02),
        # Five proposed tokens of one session late in its context: latency.
        dict(name="extend_5", kind="extend", seqs=1, lo=5, hi=5, cached_lo=2400, cached_hi=2400, hq=16, hk=8, page=16, fmt="int8"),
        # Four proposed tokens of each session of the talker's full batch bucket.
        dict(name="extend_64x4", kind="extend", seqs=64, lo=4, hi=4, cached_lo=200, cached_hi=2400, hq=16, hk=8, page=16, fmt="e4m3"),
        # Prompts of 30-300 rows behind a shared prefix of thousands of tokens, in larger pages.
        dict(name="extend_prefix", kind="extend", seqs=8, lo=30, hi=300, cached_lo=2000, cached_hi=8000, hq=32, hk=8, page=64, fmt="e4m3"),
        # Chunked prefill behind cached tokens: the largest.
        dict(name="extend_chunks", kind="extend", seqs=12, lo=512, hi=4096, cached_lo=0, cached_hi=1024, hq=32, hk=8, page=16, fmt="e4m3"),
        # One new token of one request over 1500 encoder states, a head of K and V for each of q: latency.
        dict(name="cross_1", kind="cross", groups=1, lo=1, hi=1, src_lo=1500, src_hi=1500, hq=16, hk=16),
        # One new token of each of five candidates of 48 requests.
        dict(name="cross_48x5", kind="cross", groups=48, lo=5, hi=5, src_lo=100, src_hi=1500, hq=16, hk=8),
        # Few rows over long recordings: the states have to be shared out over the GPU.
        dict(name="cross_long", kind="cross", groups=2, lo=20, hi=60, src_lo=30000, src_hi=60000, hq=16, hk=16),
        # Twelve targets known in advance (forced, or scored), packed, over sources of mixed lengths.
        dict(name="cross_pack", kind="cross", groups=12, lo=187, hi=4000, src_lo=300, src_hi=2400, hq=32, hk=8),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        case = _drawn(rng)
        if work(case)["flops"] <= 7e11:  # the largest listed case has 7.9e11
            return case


def _drawn(rng):
    kind = rng.choice(["fork", "compact", "extend", "extend", "extend", "cross", "cross", "cross"])
    if kind == "fork":
        hi = _log(rng, 1, 4000)
        hk = rng.choice([1, 2, 4, 8, 8])
        parents = _log(rng, 1, max(1, min(48, 60000 // hi)))
        page = rng.choice([16, 16, 32, 64])
        layers = _log(rng, 1, max(1, min(28, 500000 // (parents * (hi + 10 * page) * hk // 8 + 1))))
        return dict(kind=kind, parents=parents, each=_log(rng, 1, 8), lo=max(1, hi // rng.randint(1, 20)), hi=hi, page=page, hk=hk, layers=layers)
    if kind == "compact":
        hi = _log(rng, 1, 5000)
        return dict(kind=kind, lines=_log(rng, 1, max(1, min(256, 400000 // hi))), lo=max(1, hi // rng.randint(1, 20)), hi=hi,
                    page=rng.choice([16, 16, 32, 64]), hk=rng.choice([1, 2, 4, 8]), layers=1, spare=rng.choice([0.1, 0.3, 0.5, 1.0]),
                    keep=rng.choice([1.0, 1.02, 1.1]))
    hk = rng.choice([1, 2, 4, 8, 8, 16])
    if kind == "extend":
        cached = _log(rng, 1, 20000) - 1
        hi = _log(rng, 1, 3000)
        seqs = _log(rng, 1, max(1, min(128, 20000 // hi, 300000 // (cached + hi), 400000 // (hk * max(1, hi // 64 * cached // 100 + 1)))))
        g = rng.choice([1, 2, 2, 4, 4, 8] + ([3, 5, 16] if hi <= 64 else []))
        return dict(kind=kind, seqs=seqs, lo=max(1, hi // rng.randint(1, 8)), hi=hi, cached_lo=cached // rng.randint(1, 8), cached_hi=cached,
                    hq=hk * (g if hk * g <= 64 else 2), hk=hk, page=rng.choice([16, 16, 32, 64, 256]), fmt=rng.choice(["e4m3", "e4m3", "int8"]))
    src = _log(rng, 1, 40000)
    hi = _log(rng, 1, 3000)
    groups = _log(rng, 1, max(1, min(128, 20000 // hi, 200000 // src, 400000 // (hk * max(1, hi // 64 * src // 100 + 1)))))
    g = rng.choice([1, 1, 2, 4, 4, 8] + ([3, 5, 16] if hi <= 64 else []))
    return dict(kind=kind, groups=groups, lo=max(1, hi // rng.randint(1, 8)), hi=hi, src_lo=src // rng.randint(1, 8) if rng.random() < 0.8 else 0,
                src_hi=src, hq=hk * (g if hk * g <= 64 else 2), hk=hk)


# ------------------------------------------------------------------ inputs
def spread(n, lo, hi):
    """n whole numbers spread evenly over [lo, hi], in a mixed order."""
    return [lo + int((hi - lo + 1) * (((i + 0.5) * 0.6180339887498949) % 1.0)) for i in range(n)]


def _i32(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


def _zeros(*n):
    return torch.zeros(*n, dtype=torch.int32, device="cuda")


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)


def _normal(gen, *shape):
    return torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(generator=gen)


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


def _layers(gen, layers, pages, case):
    """Cache of all layers: [layers][blocks][2 hk][2048], [layers][blocks][2 hk]."""
    kv, sc = _cache(gen, layers * pages * (case["page"] // BLOCK), case["hk"], "e4m3")
    return kv.view(layers, -1, 2 * case["hk"], HEAD * BLOCK), sc.view(layers, -1, 2 * case["hk"])


def _extend_rows(case):
    """(tokens in the cache before the call, new rows) of each sequence."""
    return list(zip(spread(case["seqs"], case["cached_lo"], case["cached_hi"])[::-1], spread(case["seqs"], case["lo"], case["hi"])))


def _cross_rows(case):
    """(rows, encoder states) of each group."""
    return list(zip(spread(case["groups"], case["lo"], case["hi"]), spread(case["groups"], case["src_lo"], case["src_hi"])[::-1]))


def prepare(case, seed):
    gen, rng, kind = _gen(seed), random.Random(int(seed)), case["kind"]
    st = dict(case)
    if kind in ("fork", "compact"):
        page = case["page"]
        lens = spread(case["parents" if kind == "fork" else "lines"], case["lo"], case["hi"])
        held = [(n + page - 1) // page for n in lens]
        if kind == "fork":
            pool = sum(held) + 2 * len(lens) * case["each"] + 16
        else:
            pool = int(sum(held) * (1 + case["spare"])) + 8
        ids = list(range(pool))
        rng.shuffle(ids)
        width, nlines = max(held) + 2, len(lens) * (1 + case.get("each", 0)) + 4
        order = list(range(nlines))
        rng.shuffle(order)
        table, at = [[-1] * width for _ in range(nlines)], 0
        for line, h in zip(order, held):
            table[line][:h] = ids[at:at + h]
            at += h
        head = rng.randrange(pool)  # the free pages lie from here on, round the end
        free = [-1] * pool
        for i, p in enumerate(ids[at:]):
            free[(head + i) % pool] = p
        shares = [0] * pool
        if kind == "compact":
            for p in ids[:at:7]:  # some pages are shared with lines of another pool's table
                shares[p] = rng.randrange(3)
        st.update(table=_i32(table), free_pages=_i32(free), shares=_i32(shares))
        st["kv"], st["kv_scale"] = _layers(gen, case["layers"], pool, case)
        if kind == "fork":
            n = len(lens) * case["each"]
            st.update(parents_of=_i32([order[i // case["each"]] for i in range(n)]), children=_i32(order[len(lens):len(lens) + n]),
                      tokens=_i32([lens[i // case["each"]] for i in range(n)]), src=_zeros(n), dst=_zeros(n),
                      forked=_zeros(5), freed=_i32([0, 0, 0, head, pool - at]))
            return st
        st["limit"] = min(pool, int(math.ceil(sum(held) * case["keep"])))
        st["state"] = _i32([head, pool - at])
        for name, like in (("table_out", "table"), ("free_out", "free_pages"), ("shares_out", "shares"), ("new_ids", "shares")):
            st[name] = torch.zeros_like(st[like])
        st["src"], st["dst"], st["status"] = _zeros(pool), _zeros(pool), _zeros(5)
        return st
    hq, hk = case["hq"], case["hk"]
    if kind == "extend":
        seqs, page = _extend_rows(case), case["page"]
        need = [(f + c + page - 1) // page for f, c in seqs]
        pool = sum(need) + 16
        st["kv"], st["kv_scale"] = _cache(gen, pool * (page // BLOCK), hk, case["fmt"])
        ids = torch.randperm(pool, device="cuda", generator=gen).to(torch.int32)
        indptr = [0]
        for n in need:
            indptr.append(indptr[-1] + n)
        st["indptr"], st["pages"] = _i32(indptr), ids[:indptr[-1]].contiguous()
        st["pos"] = torch.cat([torch.arange(f, f + c, dtype=torch.int32) for f, c in seqs]).cuda()
        rows = [c for _, c in seqs]
        st["qkv"] = _normal(gen, sum(rows), (hq + 2 * hk) * HEAD)
        st["most"] = max(f + c for f, c in seqs)
    else:
        pairs = _cross_rows(case)
        rows, lens = [c for c, _ in pairs], [n for _, n in pairs]
        order = list(range(len(lens)))
        rng.shuffle(order)
        first, at = [0] * len(lens), 0
        for i in order:
            first[i] = at
            at += lens[i]
        # Source e is what the group at its place in another order attends to.
        named = [0] * len(lens)
        for e, i in enumerate(order):
            named[i] = e
        st["of"], st["first"], st["len"] = _i32(named), _i32([first[i] for i in order]), _i32([lens[i] for i in order])
        st["kv"] = _normal(gen, max(1, at), 2 * hk * HEAD)
        st["qrows"] = _normal(gen, sum(rows), hq * HEAD)
        st["most"] = max(1, max(lens))
    st["counts"], st["mostq"] = _i32(rows), max(rows)
    st["out"] = torch.zeros(sum(rows), hq * HEAD, dtype=torch.bfloat16, device="cuda")
    if own:
        oa = _oa()
        keys = [f + c for f, c in seqs] if kind == "extend" else lens
        st["plan"] = (oa.extend_plan if kind == "extend" else oa.cross_plan)(rows, hq, hk, st["most"], keys)
        st["ws"] = oa.workspace_for(st["plan"].plan)
    return st


# ------------------------------------------------------------------ one pass
def run(st):
    kind = st["kind"]
    if not own:
        return {"fork": _fork, "compact": _compact, "extend": _extend, "cross": _cross}[kind](st)
    oa = _oa()
    if kind == "fork":
        page = st["page"]
        oa.pages_fork(st["parents_of"], st["children"], st["tokens"], st["table"], st["free_pages"], st["freed"][3:5], st["shares"],
                      st["src"], st["dst"], st["forked"], page)
        oa.pages_copy(st["kv"], st["kv_scale"], st["src"], st["dst"], page)
        oa.pages_free(st["children"], st["tokens"], st["table"], st["free_pages"], st["forked"][3:5], st["shares"], st["freed"], page)
        return {n: st[n] for n in ("table", "free_pages", "shares", "src", "dst", "forked", "freed", "kv", "kv_scale")}
    if kind == "compact":
        oa.pages_compact(st["table"], st["free_pages"], st["state"], st["shares"], st["limit"], st["table_out"], st["free_out"],
                         st["shares_out"], st["new_ids"], st["src"], st["dst"], st["status"])
        oa.pages_copy(st["kv"], st["kv_scale"], st["src"], st["dst"], st["page"], st["status"][1:2])
        return {n: st[n] for n in ("table_out", "free_out", "shares_out", "new_ids", "src", "dst", "status", "kv", "kv_scale")}
    hq, hk = st["hq"], st["hk"]
    if kind == "extend":
        return oa.qwen3_extend_q8(st["plan"], st["qkv"][:, :hq * HEAD], st["kv"], st["kv_scale"], st["pos"], st["indptr"], st["pages"],
                                  st["page"], st["out"], SCALE, st["ws"])
    k, v = st["kv"].split([hk * HEAD, hk * HEAD], dim=1)
    return oa.cross_run(st["plan"], st["qrows"], k, v, st["of"], st["first"], st["len"], st["out"], SCALE, st["ws"])


def _owner(ends, x):
    """The sequence whose range [start, end) of a running total holds each x (the last one past the end)."""
    return torch.searchsorted(ends, x, right=True).clamp_(max=ends.numel() - 1)


def _put(to, at, what, where):
    """`to` with `what` at `at`, where `where` is true."""
    flat = torch.cat([to.reshape(-1), to.new_zeros(1)])
    flat[torch.where(where, at, to.numel())] = what.to(to.dtype)
    return flat[:-1].view_as(to)


def _copied(st):
    """Pages src to dst, in every layer; pairs of -1 are none."""
    pairs = torch.stack([st["src"], st["dst"]])[:, st["src"] >= 0].long()
    kv = st["kv"].view(torch.uint8).view(st["layers"], -1, st["page"] // BLOCK * 2 * st["hk"] * HEAD * BLOCK)
    scale = st["kv_scale"].view(torch.uint8).view(st["layers"], -1, st["page"] // BLOCK * 2 * st["hk"])
    kv[:, pairs[1]] = kv[:, pairs[0]]
    scale[:, pairs[1]] = scale[:, pairs[0]]


def _fork(st):
    page, table, cap = st["page"], st["table"].long(), st["free_pages"].numel()
    parent, child, tokens = st["parents_of"].long(), st["children"].long(), st["tokens"].long()
    head, avail = st["freed"][3].long(), st["freed"][4].long()
    j = torch.arange(table.shape[1], device="cuda")
    full = tokens // page
    part = (tokens % page > 0).long()
    taken = st["free_pages"].long()[(head + part.cumsum(0) - part) % cap]
    lines = table[parent]
    mine = torch.where(j < full[:, None], lines, torch.where((j == full[:, None]) & (part[:, None] > 0), taken[:, None], table[child]))
    st["table"][child] = mine.int()
    shared = j < full[:, None]
    st["shares"].copy_(torch.cat([st["shares"], st["shares"].new_zeros(1)]).index_add_(
        0, torch.where(shared, lines, cap).reshape(-1), shared.int().reshape(-1))[:-1])
    last = lines.gather(1, full.clamp(max=table.shape[1] - 1)[:, None])[:, 0]
    st["src"].copy_(torch.where(part > 0, last, -1))
    st["dst"].copy_(torch.where(part > 0, taken, -1))
    n = part.sum()
    head, avail = (head + n) % cap, avail - n
    st["forked"].copy_(torch.stack([n * 0, n, full.sum(), head, avail]))
    _copied(st)
    # And back: every page of the children loses a holder; pages without one join the queue in ascending order.
    held = j < (full + part)[:, None]
    shares = torch.cat([st["shares"], st["shares"].new_zeros(1)]).index_add_(
        0, torch.where(held, mine, cap).reshape(-1), -held.int().reshape(-1))[:-1]
    free = shares < 0
    rank = free.long().cumsum(0) - 1
    st["free_pages"].copy_(_put(st["free_pages"], (head + avail + rank) % cap, torch.arange(cap, device="cuda"), free))
    st["shares"].copy_(shares.clamp(min=0))
    back = free.sum()
    st["freed"].copy_(torch.stack([n * 0, back, held.sum(), head, avail + back]))
    return {n: st[n] for n in ("table", "free_pages", "shares", "src", "dst", "forked", "freed", "kv", "kv_scale")}


def _compact(st):
    limit, cap = st["limit"], st["free_pages"].numel()
    i = torch.arange(cap, device="cuda")
    head, avail = st["state"][0].long(), st["state"][1].long()
    listed_ids = st["free_pages"].long()[(head + i) % cap]
    free = _put(torch.zeros(cap, dtype=torch.bool, device="cuda"), listed_ids.clamp(min=0), torch.ones_like(i, dtype=torch.bool), i < avail)
    moving, hole = ~free & (i >= limit), free & (i < limit)
    nth, hole_nth = moving.long().cumsum(0) - 1, hole.long().cumsum(0) - 1
    n, holes = moving.sum(), hole.sum()
    none = torch.full_like(i, -1)
    src, holes_at = _put(none, nth, i, moving), _put(none, hole_nth, i, hole)
    dst = torch.where(i < n, holes_at, -1)
    new_ids = torch.where(moving, dst[nth.clamp(min=0)], i)
    table = st["table"].long()
    inside = (table >= 0) & (table < cap)
    st["table_out"].copy_(torch.where(inside, new_ids[table.clamp(0, cap - 1)], table))
    st["shares_out"].copy_(_put(torch.where(moving, 0, st["shares"].long()), new_ids, st["shares"].long(), moving))
    # The queue afterwards: holes that stay, then everything from the limit on.
    left = (hole & (hole_nth >= n)) | (i >= limit)
    st["free_out"].copy_(_put(none, left.long().cumsum(0) - 1, i, left))
    st["src"].copy_(src), st["dst"].copy_(dst), st["new_ids"].copy_(new_ids)
    st["status"].copy_(torch.stack([n * 0, n, holes - n, n * 0, avail]))
    _copied(st)
    return {n: st[n] for n in ("table_out", "free_out", "shares_out", "new_ids", "src", "dst", "status", "kv", "kv_scale")}


def _pow2(biased):
    """2^(biased - 127), exactly."""
    return (biased.int().clamp(min=1) << 23).view(torch.float32)


def _padded(rows, counts, most):
    """Packed rows as [sequences][most][..], and where they came from."""
    n, counts = counts.numel(), counts.long()
    r = torch.arange(rows.shape[0], device="cuda")
    s = _owner(counts.cumsum(0), r)
    p = r - (counts.cumsum(0) - counts)[s]
    out = torch.zeros(n, most, *rows.shape[1:], device="cuda", dtype=rows.dtype)
    out[s, p] = rows
    return out, s, p


def _weighted(q, k, v, seen, hk):
    """softmax over the keys that `seen` [n][most q][keys] lets through; q [n][most q][hq][128], k and v [n][keys][hk][128]."""
    n, most, hq = q.shape[:3]
    t = k.shape[1]
    k, v = k.permute(0, 2, 3, 1).contiguous(), v.permute(0, 2, 1, 3).contiguous()
    x = torch.matmul(q.transpose(1, 2).reshape(n, hk, hq // hk * most, HEAD), k).view(n, hk, -1, most, t).mul_(SCALE)
    x.masked_fill_(~seen[:, None, None], -math.inf)
    x.sub_(x.amax(-1, keepdim=True).clamp_(min=-3e38)).exp_()
    o = torch.matmul(x.view(n, hk, -1, t), v).view(n, hk, -1, most, HEAD)
    total = x.sum(-1, keepdim=True)
    return (o / torch.where(total > 0, total, 1.0)).view(n, hq, most, HEAD).transpose(1, 2)


def _extend(st):
    hq, hk, page, most = st["hq"], st["hk"], st["page"], st["most"]
    rows = st["out"].shape[0]
    b = torch.arange((most + BLOCK - 1) // BLOCK, device="cuda") * BLOCK
    at = (st["indptr"][:-1, None] + b[None] // page).clamp(max=st["pages"].numel() - 1)
    block = st["pages"][at.long()].long() * (page // BLOCK) + b[None] % page // BLOCK
    n, keys = block.shape[0], b.numel() * BLOCK
    scale = _pow2(st["kv_scale"].view(torch.uint8)[block])
    raw = st["kv"].view(torch.uint8)[block].view(st["kv"].dtype).float() * scale[..., None]  # [n, blocks, 2 hk, 2048]
    k = raw[:, :, :hk].view(n, -1, hk, BLOCK, HEAD).transpose(2, 3).reshape(n, keys, hk, HEAD)
    v = raw[:, :, hk:].view(n, -1, hk, HEAD, BLOCK).permute(0, 1, 4, 2, 3).reshape(n, keys, hk, HEAD)
    q, s, p = _padded(st["qkv"][:, :hq * HEAD].float().view(rows, hq, HEAD), st["counts"], st["mostq"])
    pos = _padded(st["pos"] + 1, st["counts"], st["mostq"])[0]
    o = _weighted(q, k, v, torch.arange(keys, device="cuda") < pos[..., None], hk)
    return st["out"].copy_(o[s, p].reshape(rows, -1))


def _cross(st):
    hq, hk, most, rows = st["hq"], st["hk"], st["most"], st["out"].shape[0]
    of = st["of"].long()
    t = torch.arange(most, device="cuda")
    seen = t < st["len"][of][:, None]
    at = (st["first"][of].long()[:, None] + t).clamp(max=st["kv"].shape[0] - 1)
    kv = st["kv"].float().view(-1, 2 * hk, HEAD)[at]
    q, s, p = _padded(st["qrows"].float().view(rows, hq, HEAD), st["counts"], st["mostq"])
    o = _weighted(q, kv[:, :, :hk], kv[:, :, hk:], seen[:, None].expand(-1, st["mostq"], -1), hk)
    return st["out"].copy_(o[s, p].reshape(rows, -1))


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    kind = case["kind"]
    if kind in ("fork", "compact"):
        page = case["page"]
        page_bytes = case["layers"] * page // BLOCK * 2 * case["hk"] * (HEAD * BLOCK + 1)
        lens = spread(case["parents" if kind == "fork" else "lines"], case["lo"], case["hi"])
        held = [(n + page - 1) // page for n in lens]
        if kind == "fork":
            copies = sum(case["each"] for n in lens if n % page)
            full = sum(n // page * case["each"] for n in lens)
            # Lines read and written, holders counted up and down, queue entries taken and given back.
            return {"bytes": copies * (2 * page_bytes + 24) + full * 24 + len(lens) * case["each"] * 12, "flops": 0}
        pool = int(sum(held) * (1 + case["spare"])) + 8
        limit = min(pool, int(math.ceil(sum(held) * case["keep"])))
        moves = int(sum(held) * (pool - limit) / pool)  # of pages anywhere in the pool, as many as lie past the limit
        cells = len(lens) * (max(held) + 2) + 4 * (max(held) + 2)
        return {"bytes": moves * 2 * page_bytes + cells * 8 + pool * 28, "flops": 0}
    hq, hk = case["hq"], case["hk"]
    if kind == "extend":
        seqs = _extend_rows(case)
        keys, blocks = sum(f + c for f, c in seqs), sum((f + c + BLOCK - 1) // BLOCK for f, c in seqs)
        rows = sum(c for _, c in seqs)
        pairs = sum(c * f + c * (c + 1) // 2 for f, c in seqs)
        return {"bytes": keys * 2 * hk * HEAD + blocks * 2 * hk + rows * 4 * hq * HEAD, "flops": 4 * HEAD * hq * pairs}
    pairs = _cross_rows(case)
    return {"bytes": sum(n for _, n in pairs) * 4 * hk * HEAD + sum(c for c, _ in pairs) * 4 * hq * HEAD,
            "flops": 4 * HEAD * hq * sum(c * n for c, n in pairs)}


# ------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    kind = case["kind"]
    if kind in ("fork", "compact"):
        return None  # whole numbers and bytes that are moved
    hq, hk = case["hq"], case["hk"]
    g = hq // hk
    pairs = _extend_rows(case) if kind == "extend" else _cross_rows(case)
    if hq * sum((c * (f + c) if kind == "extend" else f * c) for f, c in pairs) > 3e10:
        return None
    st = prepare(case, seed)
    out = torch.zeros(st["out"].shape[0], hq, HEAD, dtype=torch.float64, device="cuda")
    at = 0
    for i, pair in enumerate(pairs):
        if kind == "extend":
            f, c = pair
            per = case["page"] // BLOCK
            ids = st["pages"][int(st["indptr"][i]):int(st["indptr"][i + 1])].long()
            blocks = (ids[:, None] * per + torch.arange(per, device="cuda")).reshape(-1)
            factor = (st["kv_scale"].view(torch.uint8)[blocks].long() + 1023 - 127 << 52).view(torch.float64)
            raw = st["kv"].view(torch.uint8)[blocks].view(st["kv"].dtype).double() * factor[..., None]
            hidden = torch.arange(f + c, device="cuda") > (f + torch.arange(c, device="cuda"))[:, None]
        else:
            c, f = pair
            e = int(st["of"][i])
            kv = st["kv"][int(st["first"][e]):int(st["first"][e]) + f].double().view(f, 2 * hk, HEAD)
        for h in range(hk if kind == "extend" or f > 0 else 0):
            if kind == "extend":
                k = raw[:, h].reshape(-1, HEAD)[:f + c]
                v = raw[:, hk + h].view(-1, HEAD, BLOCK).transpose(1, 2).reshape(-1, HEAD)[:f + c]
            else:
                k, v = kv[:, h], kv[:, hk + h]
            for j in range(h * g, h * g + g):
                q = (st["qkv"] if kind == "extend" else st["qrows"])[at:at + c, j * HEAD:(j + 1) * HEAD].double()
                s = q @ k.t() * SCALE
                if kind == "extend":
                    s.masked_fill_(hidden, -math.inf)
                out[at:at + c, j] = torch.softmax(s, -1) @ v
        at += c
    return out.view(-1, hq * HEAD)
