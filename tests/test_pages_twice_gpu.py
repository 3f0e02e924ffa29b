"""Lines that are given back twice while others hold pages: pages_free says so (code 6) before the queue lists a page twice."""
import numpy as np
import pytest
import torch

import omni_attn as oa
from test_pages_gpu import Pool, fork, give_back, host, i32

pytestmark = pytest.mark.gpu


def again(pool, lines, tokens):
    """A call that gives pages back which nobody holds: code 6, the queue and its state as they were, no count below zero."""
    d, status = pool.d, i32([9] * 5)
    held = sum(-(-t // pool.page) for t in tokens)
    oa.pages_free(i32(lines), i32(tokens), d["table"], d["free"], d["state"], d["shares"], status, pool.page)
    torch.cuda.synchronize()
    assert status.tolist() == [6, 0, held, *[int(x) for x in pool.state]]
    assert np.array_equal(host(d["free"]), pool.free) and bool((d["shares"] >= 0).all())
    pool.shares = host(d["shares"])
    d["state"] = status[3:5]


def fill(pool):
    """Whether every page is in the queue once or in a line."""
    head, avail = (int(x) for x in pool.state)
    queue = [int(pool.free[(head + k) % pool.total]) for k in range(avail)]
    return len(set(queue)) == avail


@pytest.mark.parametrize("width", [12, 5000])  # all in one launch; the lines' entries too many for that
@pytest.mark.parametrize("first", [0, 1])
def test_a_line_twice_beside_another_request(first, width):
    pool = Pool(np.random.default_rng(3 + first), [70, 90], 16, 3, 0, width=width)
    pool.upload()
    line, other = pool.lines[first], pool.lines[1 - first]
    tokens, rest = pool.lens[first], pool.lens[1 - first]
    assert give_back(pool, [line], [tokens])[0] == 0
    again(pool, [line], [tokens])
    again(pool, [line], [1])
    assert fill(pool) and give_back(pool, [other], [rest])[0] == 0
    assert sorted(pool.free.tolist()) == list(range(pool.total))


def test_a_line_twice_beside_one_that_ends():
    """The call is taken as a whole: the other line's pages stay out of the queue too, and the code says why."""
    pool = Pool(np.random.default_rng(5), [70, 90, 40], 16, 3, 0)
    pool.upload()
    a, b, c = pool.lines
    assert give_back(pool, [a], [70])[0] == 0
    again(pool, [b, a], [90, 70])
    assert fill(pool) and give_back(pool, [c], [40])[0] == 0


def test_a_child_twice():
    """Its shared pages lose a holder too many, unseen while others hold them; its own page is in the queue."""
    pool = Pool(np.random.default_rng(6), [70], 16, 6, 3)
    pool.upload()
    a, b, c, _ = pool.lines
    fork(pool, [a, a], [b, c], [70, 70])
    assert give_back(pool, [b], [70])[0] == 0
    again(pool, [b], [70])


@pytest.mark.parametrize("total,at", [(70_001, 40_000), (70_001, 8191), (70_001, 8192), (1 << 19, 300_000), ((1 << 19) + 77, 11), ((1 << 19) + 77, 500_000)])
@pytest.mark.parametrize("width", [None, 5000])
def test_anywhere_in_the_queue_of_a_large_pool(total, at, width):
    """One page of a free line in a long queue, which runs round the end of its array."""
    pool = Pool(np.random.default_rng(total + at), [20, 3], 1, total - 23, 0, width=width)
    pool.upload()
    line, other = pool.lines
    pool.table[line, 0] = pool.free[(pool.head + at) % pool.total]
    pool.d["table"] = i32(pool.table)
    again(pool, [line], [1])
    assert give_back(pool, [other], [3])[0] == 0
