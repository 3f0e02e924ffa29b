"""What lines that share pages must not do, by the host loops of the tables and of fork: come back to a page that others hold, by a
ring or by going back to fewer tokens. The header, the mirror and the guide say so where a caller reads of fork and of rings."""
import os

import numpy as np
import pytest

import omni_attn as oa
import pages_refs as P
import serve_refs as S

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def forked(tokens):
    """A parent of 40 tokens and its child of `tokens` in pages of 16; table, queue, state and counts."""
    table = np.array([[3, 1, 5, -1], [-1, -1, -1, -1]])
    free, shares = np.array([0, 2, 4, 6, 7, -1, -1, -1]), np.zeros(8, np.int64)
    st = P.fork([0], [1], [tokens], 16, table, free, [0, 5], shares)[2]
    assert st[0] == 0
    return table, free, st[3:], shares


def slots(first, ring):
    table, free, state, shares = forked(40)
    out = S.tables([first, first], [1, 1], [0, 1], table, free, state, 8, 16, 16, ring)
    return out["status"][0], out["slots"], [int(shares[s // 16]) for s in out["slots"]]


def test_without_a_ring_no_line_writes_where_another_reads():
    for first in (40, 47, 48):
        code, (a, b), shares = slots(first, 0)
        assert code == 0 and a != b and shares == [0, 0]


def test_behind_a_ring_both_write_one_slot_of_a_shared_page():
    code, (a, b), shares = slots(64, 64)
    assert code == 0 and a == b == 3 * 16 and shares == [1, 1]
    for first in (40, 48):  # before it comes round a ring changes nothing
        assert slots(first, 64) == slots(first, 0)


def test_a_line_of_more_tokens_than_its_ring_is_given_back_by_the_ring():
    table, free, state, shares = forked(40)
    assert P.give_back([0], [100], 16, table, free, state, shares)[0] == 4
    table[0, 3] = 2  # a line of a ring of 64 that came round: four pages, whatever its position
    assert P.give_back([0], [64], 16, table, free, [int(state[0]) + 1, int(state[1]) - 1], shares)[:2] == [0, 2]


def test_a_line_that_goes_back_behind_a_fork_writes_to_shared_pages():
    table, free, state, shares = forked(40)
    out = S.tables([30], [1], [0], table, free, state, 8, 16, 16, 0)
    assert out["slots"] == [1 * 16 + 14] and shares[1] == 1


def section(path, begin, end):
    text = " ".join(open(os.path.join(ROOT, path)).read().replace("\n *", " ").split())
    return text[text.index(begin):text.index(end, text.index(begin))]


@pytest.mark.parametrize("text", [
    lambda: section("include/omni_attn.h", "Candidates forked from one request", "int omni_attn_pages_fork"),
    lambda: section("include/omni_attn.h", "A ring's tables are for the calls", "int omni_attn_step_tables"),
    lambda: section("INTEGRATION.md", "Requests that share prefixes", "Preconditions the calls check"),
    lambda: oa.pages_fork.__doc__], ids=["pages", "tables", "guide", "mirror"])
def test_it_is_said(text):
    assert "ring" in text() and "share" in text() and ("fork" in text())
