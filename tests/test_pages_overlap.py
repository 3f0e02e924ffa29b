"""Buffers that may not overlap: the calls on shared pages read some of theirs in every workgroup while others write, so what a call
writes lies apart from all else that it is given. Refused before any launch (CPU)."""
import itertools

import pytest

import omni_attn as oa

# Buffers of a call, far apart: name -> (address, int32 entries), in the order of the call's pointers.
AT = {name: (1 << 20) * (i + 1) for i, name in enumerate(
    ["parents", "lines", "tokens", "table", "free", "state", "shares", "src", "dst", "status", "table_out", "free_out", "shares_out", "new_ids"])}
SIZES = dict(parents=6, lines=6, tokens=6, table=40, free=9, state=2, shares=9, src=6, dst=6, status=5, table_out=40, free_out=9, shares_out=9,
             new_ids=9)


def fork(**at):
    p = {**AT, **at}
    return oa.load().omni_attn_pages_fork(p["parents"], p["lines"], p["tokens"], 6, 16, p["table"], 5, 8, p["free"], 9, p["state"], p["shares"],
                                          p["src"], p["dst"], p["status"], None)


def free(**at):
    p = {**AT, **at}
    return oa.load().omni_attn_pages_free(p["lines"], p["tokens"], 6, 16, p["table"], 5, 8, p["free"], 9, p["state"], p["shares"], p["status"], None)


def compact(**at):
    p = {**AT, **at}
    return oa.load().omni_attn_pages_compact(p["table"], 5, 8, p["free"], 9, p["state"], p["shares"], 5, p["table_out"], p["free_out"],
                                             p["shares_out"], p["new_ids"], p["src"], p["dst"], 6, p["status"], None)


CALLS = {
    "pages_fork": (fork, ["parents", "lines", "tokens", "free", "state"], ["table", "shares", "src", "dst", "status"]),
    "pages_free": (free, ["lines", "tokens", "table", "state"], ["free", "shares", "status"]),
    "pages_compact": (compact, ["table", "free", "state", "shares"], ["table_out", "free_out", "shares_out", "new_ids", "src", "dst", "status"]),
}
CASES = [(call, a, b) for call, (_, reads, writes) in CALLS.items()
         for a, b in [*itertools.combinations(writes, 2), *itertools.product(reads, writes)]]


@pytest.mark.parametrize("call,a,b", CASES)
def test_refused(call, a, b):
    """Each pair of which one is written: the last entry of one on the first of the other, and the other way round; and one inside the
    other. (A table compacted in place is no overlap: equal addresses of those two are left out.)"""
    f = CALLS[call][0]
    for x, y in ((a, b), (b, a)):
        places = [AT[x] + 4 * (SIZES[x] - 1)]
        if {x, y} != {"table", "table_out"}:
            places.append(AT[x])
        for at in places:
            assert f(**{y: at}) == oa.EINVAL, (x, y)
            assert call.encode() in oa.load().omni_attn_last_error()


@pytest.mark.gpu
def test_neighbours_are_taken():
    """Buffers that touch, in one tensor; the compacted table in place; the same read-only list twice."""
    import torch

    def one(*sizes):
        at, out = 0, []
        all_ = torch.zeros(sum(sizes), dtype=torch.int32, device="cuda")
        for n in sizes:
            out.append(all_[at:at + n])
            at += n
        return out

    table, free_, shares, status, state, src, dst, par, chi, tok = one(40, 9, 9, 5, 2, 6, 6, 6, 6, 6)
    table = table.view(8, 5)
    free_.copy_(torch.arange(9, dtype=torch.int32))
    state.copy_(torch.tensor([0, 9], dtype=torch.int32))
    tok.fill_(-1)
    oa.pages_fork(par, chi, tok, table, free_, state, shares, src, dst, status)
    oa.pages_free(chi, tok, table, free_, state, shares, status)
    oa.pages_free(tok, tok, table, free_, state, shares, status)
    fout, sout, ids, st2 = one(9, 9, 9, 5)
    oa.pages_compact(table, free_, status[3:5], shares, 5, table, fout, sout, ids, src, dst, st2)
    torch.cuda.synchronize()
    assert status.tolist() == [0, 0, 0, 0, 9] and st2.tolist() == [0, 0, 5, 0, 9] and fout.tolist() == list(range(9))
