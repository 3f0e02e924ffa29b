"""Plain references for the serving calls over the 8-bit block cache: the step's
row tables in host loops, the block quantizer byte for byte, the rotary and the
attentions in 64 bits."""
from __future__ import annotations

import math

import numpy as np
import torch

BLOCK, HEAD = 16, 128
TOP = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


# ------------------------------------------------------------------ tables
def tables(first, count, lines, table, free, state, row_cap, page_cap, page=16, ring=0):
    """Dict of what step_tables leaves behind. free None: the table holds every page."""
    n = len(first)
    lines = list(range(n)) if lines is None else list(lines)
    table, free = table.copy(), None if free is None else free.copy()
    width, total = table.shape[1], 0 if free is None else len(free)
    head, avail = (0, 0) if free is None else (int(state[0]), int(state[1]))
    reach = lambda t: min(t, ring) if ring else t
    pages_of = lambda t: (reach(t) + page - 1) // page
    codes, rows, pages, taken, back = set(), 0, 0, 0, 0
    for f, c, line in zip(first, count, lines):
        f, c = int(f), int(c)
        if f < 0 or (c > 0 and f + c > 2**31 - 1) or not 0 <= line < table.shape[0]:
            codes.add(1)
            continue
        held, need = pages_of(f), 0 if c < 0 else pages_of(f + max(c, 0))
        if max(held, need) > width:
            codes.add(4)
            continue
        rows, pages = rows + max(c, 0), pages + need
        taken, back = taken + (0 if c < 0 else need - held), back + (held if c < 0 else 0)
    if free is not None:
        if not 0 <= head < total or not 0 <= avail <= total or avail + back > total:
            codes.add(1)
        if taken > max(avail, 0):
            codes.add(5)
    if rows > row_cap:
        codes.add(2)
    if pages > page_cap:
        codes.add(3)
    out = dict(pos=[], slots=[], seq=[], row_indptr=[0], indptr=[0], pages=[], table=table, free=free)
    code = min(codes) if codes else 0
    if code:
        out["row_indptr"] = out["indptr"] = [0] * (n + 1)
        out["status"] = [code, 0, 0, head if free is not None else 0, avail if free is not None else 0]
        return out
    at, end = head, (head + avail)
    for s, (f, c, line) in enumerate(zip(first, count, lines)):
        f, c = int(f), int(c)
        if c < 0:
            if free is not None:
                for j in range(pages_of(f)):
                    free[end % total] = table[line, j]
                    end += 1
        else:
            if free is not None:
                for j in range(pages_of(f), pages_of(f + c)):
                    table[line, j] = free[at % total]
                    at += 1
            ids = [int(x) for x in table[line, :pages_of(f + c)]]
            for p in range(f, f + c):
                q = p % ring if ring else p
                out["pos"].append(p), out["seq"].append(s), out["slots"].append(ids[q // page] * page + q % page)
            out["pages"] += ids
        out["row_indptr"].append(len(out["pos"])), out["indptr"].append(len(out["pages"]))
    left = [0, 0] if free is None else [at % total, end - at]
    out["status"] = [0, len(out["pos"]), len(out["pages"])] + left
    return out


# ------------------------------------------------------------------ quantizer
def rounded(x, fmt):
    """f64 values, already divided by the scale, as stored values (f64)."""
    x = x.clone()
    if fmt == torch.float8_e4m3fn:
        x[~torch.isfinite(x)] = math.nan
        return x.float().to(fmt).double()  # exact in f32: bf16 inputs times a power of two
    x[torch.isnan(x)] = 0
    return torch.round(x).clamp(-127, 127)


def exponent(most, fmt):
    """Biased exponent of the smallest power of two that brings `most` (> 0) to at most the top."""
    e = -126
    while TOP[fmt] * 2.0 ** e < most:
        e += 1
    return e + 127


class Cache:
    """The cache as values: [blocks][2 hk][16][128] stored numbers and exponents."""

    def __init__(self, kv, kv_scale, hk):
        self.hk, self.fmt = hk, kv.dtype
        raw = kv.cpu().float().double()
        n = raw.shape[0]
        self.val = torch.cat([raw[:, :hk].reshape(n, hk, BLOCK, HEAD),
                              raw[:, hk:].reshape(n, hk, HEAD, BLOCK).transpose(2, 3)], 1).clone()
        self.exp = kv_scale.cpu().view(torch.uint8).int().clone()

    def write(self, slots, k, v):
        """Rows in call order: k, v [rows][hk][128] f64 (bf16 values)."""
        new = torch.cat([k, v], 1)
        of = [int(x) // BLOCK if int(x) >= 0 else -1 for x in slots]
        for n, b in enumerate(of):
            if b < 0 or b in of[max(0, n - 15):n]:
                continue
            at = {int(slots[i]) % BLOCK: i for i in range(n, min(n + 16, len(of))) if of[i] == b}  # the last of a slot counts
            tokens, rows = list(at), list(at.values())
            for h in range(2 * self.hk):
                x = new[rows, h]
                fin = x[torch.isfinite(x)].abs()
                e = exponent(float(fin.max()) if fin.numel() else 0.0, self.fmt)
                if 0 not in at:
                    old = int(self.exp[b, h])
                    e = max(e, old)
                    if e > old:
                        self.val[b, h] = rounded(self.val[b, h] * 2.0 ** (old - e), self.fmt)
                else:
                    self.val[b, h] = 0
                self.val[b, h, tokens] = rounded(x * 2.0 ** (127 - e), self.fmt)
                self.exp[b, h] = e

    def tokens(self):
        """(K, V) values [slots][hk][128] in f64."""
        x = self.val * torch.pow(2.0, (self.exp - 127).double())[..., None, None]
        x = x.transpose(1, 2).reshape(-1, 2 * self.hk, HEAD)
        return x[:, :self.hk], x[:, self.hk:]

    def same_as(self, kv, kv_scale):
        """Equal values (any NaN equals any NaN) and equal exponents."""
        other = Cache(kv, kv_scale, self.hk)
        assert torch.equal(self.exp, other.exp), "exponents differ"
        assert torch.equal(torch.nan_to_num(self.val, 1e30), torch.nan_to_num(other.val, 1e30)), "values differ"


# ------------------------------------------------------------------ rotary
def turned(x, w, pos, eps, theta):
    """RMSNorm and half-split rotary in f64, and the bound on a bf16 kernel that rounds the normalised value and the result:
    half a step (2^-8) of either, and 2^-18 of the pair for f32 arithmetic between them. x [rows][heads][128]."""
    x, w = x.double(), w.double()
    y = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w
    i = torch.arange(HEAD // 2, dtype=torch.float64)
    ang = pos.double()[:, None] * torch.pow(torch.tensor(float(theta), dtype=torch.float64), -2 * i / HEAD)
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    a, b = y[..., :HEAD // 2], y[..., HEAD // 2:]
    out = torch.cat([a * c - b * s, b * c + a * s], -1)
    pair = torch.cat([(a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()], -1)
    amp = (a.abs() + b.abs()).repeat(1, 1, 2)
    return out, 2.0 ** -8 * (out.abs() + pair) * (1 + 2.0 ** -7) + 2.0 ** -18 * amp


# ------------------------------------------------------------------ attention
def attend(q, k, v, scale):
    """One row's attention in f64: q [hq][128], k and v [keys][hk][128]. (out, sum p |v| / sum p)."""
    hq, hk = q.shape[0], k.shape[1]
    g = hq // hk
    if k.shape[0] == 0:
        return torch.zeros(hq, HEAD, dtype=torch.float64), torch.zeros(hq, HEAD, dtype=torch.float64)
    qq = q.double().view(hk, g, HEAD)
    p = torch.softmax(torch.einsum("hgd,khd->hgk", qq, k.double()) * scale, -1)
    o = torch.einsum("hgk,khd->hgd", p, v.double()).reshape(hq, HEAD)
    return o, torch.einsum("hgk,khd->hgd", p, v.double().abs()).reshape(hq, HEAD)
