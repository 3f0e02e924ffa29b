"""Plain references for the pages that requests share: fork, free, compact and copy
in host loops over numpy arrays, which they change in place like the calls do."""
from __future__ import annotations

import numpy as np


def _state_bad(head, avail, total):
    return not 0 <= head < total or not 0 <= avail <= total


def fork(parents, children, tokens, page, table, free, state, shares):
    """(src, dst, status). Nothing changes where status[0] is not 0."""
    lines, width, total = table.shape[0], table.shape[1], len(free)
    head, avail = int(state[0]), int(state[1])
    live = [i for i in range(len(tokens)) if tokens[i] >= 0]
    codes = {1} if _state_bad(head, avail, total) else set()
    seen = set()
    need = 0
    for i in live:
        if not 0 <= parents[i] < lines or not 0 <= children[i] < lines:
            codes.add(1)
            continue
        if children[i] in seen:
            codes.add(1)
        seen.add(children[i])
        if -(-int(tokens[i]) // page) > width:
            codes.add(4)
        need += tokens[i] % page > 0
    if any(parents[i] in seen for i in live):
        codes.add(1)
    if need > avail:
        codes.add(5)
    src, dst = [-1] * len(tokens), [-1] * len(tokens)
    if codes:
        return src, dst, [min(codes), 0, 0, head, avail]
    shared = taken = 0
    for i in live:
        full = int(tokens[i]) // page
        for j in range(full):
            p = table[parents[i], j]
            table[children[i], j] = p
            if 0 <= p < total:
                shares[p] += 1
        shared += full
        if tokens[i] % page:
            src[i] = int(table[parents[i], full])
            dst[i] = table[children[i], full] = int(free[(head + taken) % total])
            taken += 1
    return src, dst, [0, taken, shared, (head + taken) % total, avail - taken]


def give_back(lines_of, tokens, page, table, free, state, shares):
    """status."""
    lines, width, total = table.shape[0], table.shape[1], len(free)
    head, avail = int(state[0]), int(state[1])
    codes = {1} if _state_bad(head, avail, total) else set()
    live = [i for i in range(len(tokens)) if tokens[i] >= 0]
    seen = set()
    for i in live:
        if not 0 <= lines_of[i] < lines:
            codes.add(1)
            continue
        if lines_of[i] in seen:
            codes.add(1)
        seen.add(lines_of[i])
        if -(-int(tokens[i]) // page) > width:
            codes.add(4)
    if codes:
        return [min(codes), 0, 0, head, avail]
    held = 0
    for i in live:
        for j in range(-(-int(tokens[i]) // page)):
            held += 1
            p = table[lines_of[i], j]
            if 0 <= p < total:
                shares[p] -= 1
    back = [p for p in range(total) if shares[p] < 0]
    shares[back] = 0
    if len(back) > total - avail:
        return [6, 0, held, head, avail]
    for k, p in enumerate(back):
        free[(head + avail + k) % total] = p
    return [0, len(back), held, head, avail + len(back)]


def compact(table, free, state, shares, limit, cap):
    """None where nothing is written, or dict of outputs; and status."""
    total = len(free)
    head, avail = int(state[0]), int(state[1])
    queue = [] if _state_bad(head, avail, total) else [int(free[(head + k) % total]) for k in range(avail)]
    if _state_bad(head, avail, total) or len(set(queue)) != len(queue) or any(not 0 <= p < total for p in queue):
        return None, [1, 0, 0, head, avail]
    is_free = np.zeros(total, bool)
    is_free[queue] = True
    moving = [p for p in range(limit, total) if not is_free[p]]
    holes = [p for p in range(limit) if is_free[p]]
    if len(moving) > cap:
        return None, [3, 0, 0, head, avail]
    if len(moving) > len(holes):
        return None, [5, 0, 0, head, avail]
    new_ids, held = np.arange(total), shares.copy()
    held[is_free] = 0
    for s, d in zip(moving, holes):
        new_ids[s] = d
        held[d], held[s] = shares[s], 0
    inside = (table >= 0) & (table < total)
    left = holes[len(moving):] + list(range(limit, total))
    pad = lambda a, n: np.array(list(a) + [-1] * (n - len(a)))
    out = dict(table=np.where(inside, new_ids[np.clip(table, 0, total - 1)], table), free=pad(left, total), shares=held, new_ids=new_ids,
               src=pad(moving, cap), dst=pad(holes[:len(moving)], cap))
    return out, [0, len(moving), len(holes) - len(moving), 0, avail]
