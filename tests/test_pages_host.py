"""Refusals of the calls on shared pages, before any launch (CPU), and the host
references that the GPU tests compare with."""
import numpy as np
import pytest
import torch

import omni_attn as oa
import pages_refs as R

P = 4096  # stands for a device pointer: nothing is launched


def fork(**k):
    a = dict(parents=P, children=P, tokens=P, n=2, page=16, table=P, ld=4, num_lines=2, free=P, num_pages=9, state=P + 64, shares=P,
             src=P, dst=P, status=P)
    a.update(k)
    return oa.load().omni_attn_pages_fork(*a.values(), None)


@pytest.mark.parametrize("bad", [
    dict(n=-1), dict(page=0), dict(page=-16), dict(ld=-1), dict(num_lines=-1), dict(num_pages=0), dict(parents=None),
    dict(children=None), dict(tokens=None), dict(table=None), dict(free=None), dict(state=None), dict(shares=None), dict(src=None),
    dict(dst=None), dict(status=None), dict(state=P), dict(state=P + 16), dict(state=P - 4)])
def test_fork_refusals(bad):
    assert fork(**bad) == oa.EINVAL
    assert b"pages_fork" in oa.load().omni_attn_last_error()


def test_fork_limits():
    assert fork(num_lines=(1 << 18) + 1) == oa.EUNSUPPORTED
    assert fork(n=2**24) == oa.EUNSUPPORTED


def free(**k):
    a = dict(lines=P, tokens=P, n=2, page=16, table=P, ld=4, num_lines=2, free=P, num_pages=9, state=P + 64, shares=P, status=P)
    a.update(k)
    return oa.load().omni_attn_pages_free(*a.values(), None)


@pytest.mark.parametrize("bad", [
    dict(n=-1), dict(page=0), dict(ld=-1), dict(num_lines=-1), dict(num_pages=0), dict(lines=None), dict(tokens=None), dict(table=None),
    dict(free=None), dict(state=None), dict(shares=None), dict(status=None), dict(state=P + 16)])
def test_free_refusals(bad):
    assert free(**bad) == oa.EINVAL
    assert b"pages_free" in oa.load().omni_attn_last_error()


def compact(**k):
    a = dict(table=P, ld=4, num_lines=2, free=P, num_pages=9, state=P + 64, shares=P + 4096, limit=5, table_out=P, free_out=P + 8192,
             shares_out=P + 12288, ids=P, src=P, dst=P, cap=3, status=P)
    a.update(k)
    return oa.load().omni_attn_pages_compact(*a.values(), None)


@pytest.mark.parametrize("bad", [
    dict(ld=-1), dict(ld=2**31), dict(num_lines=-1), dict(num_pages=0), dict(limit=-1), dict(limit=10), dict(cap=-1), dict(table=None),
    dict(table_out=None), dict(free=None), dict(state=None), dict(shares=None), dict(free_out=None), dict(shares_out=None), dict(ids=None),
    dict(src=None), dict(dst=None), dict(status=None), dict(state=P + 16), dict(free_out=P), dict(free_out=P + 32), dict(shares_out=P + 4096),
    dict(table_out=P + 4), dict(table=P + 28)])
def test_compact_refusals(bad):
    assert compact(**bad) == oa.EINVAL
    assert b"pages_compact" in oa.load().omni_attn_last_error()


def test_compact_limits():
    assert compact(num_pages=(1 << 19) + 1) == oa.EUNSUPPORTED


def copy(**k):
    a = dict(kv=P, page_bytes=4096, stride=40960, scale=P, scale_bytes=2, scale_stride=20, layers=3, num_pages=10, src=P, dst=P, n=2, count=None)
    a.update(k)
    return oa.load().omni_attn_pages_copy(*a.values(), None)


@pytest.mark.parametrize("bad", [
    dict(n=-1), dict(layers=-1), dict(num_pages=-1), dict(page_bytes=0), dict(page_bytes=24), dict(page_bytes=2**40 + 16), dict(stride=-16),
    dict(stride=40968), dict(stride=40944), dict(scale_bytes=-1), dict(scale_stride=-1), dict(scale_stride=19), dict(kv=None), dict(src=None),
    dict(dst=None), dict(kv=P + 8)])
def test_copy_refusals(bad):
    assert copy(**bad) == oa.EINVAL
    assert b"pages_copy" in oa.load().omni_attn_last_error()


def test_copies_of_nothing():
    assert copy(n=0, src=None, dst=None) == oa.OK
    assert copy(layers=0, kv=None) == oa.OK
    assert copy(num_pages=0) == oa.OK


def test_the_mirror_refuses_host_tensors_and_other_shapes():
    z = torch.zeros(8, dtype=torch.int32)
    t = torch.zeros(2, 4, dtype=torch.int32)
    kv, sc = oa.q8_cache(4, 16, 2, device="cpu")
    for call in (lambda: oa.pages_fork(z, z, z, t, z, z, z, z, z, z), lambda: oa.pages_free(z, z, t, z, z, z, z),
                 lambda: oa.pages_compact(t, z, z, z, 3, t, z, z, z, z, z, z), lambda: oa.pages_copy(kv, sc, z, z),
                 lambda: oa.pages_fork(z, z, z, z, z, z, z, z, z, z), lambda: oa.pages_free(z, z, z, z, z, z, z),
                 lambda: oa.pages_compact(z, z, z, z, 3, t, z, z, z, z, z, z)):
        with pytest.raises(oa.OmniAttnError) as e:
            call()
        assert e.value.code == oa.EINVAL


@pytest.mark.parametrize("kv,sc,page", [
    ((4, 4, 2048), (4, 4), 24), ((4, 4, 2048), (4, 4), 0), ((4, 4, 2048), (4, 4), -16), ((5, 4, 2048), (5, 4), 32), ((4, 3, 2048), (4, 3), 16),
    ((4, 4, 1024), (4, 4), 16), ((4, 4, 2048), (4, 2), 16), ((4, 4, 2048), (3, 4), 16), ((2, 4, 4, 2048), (4, 4), 16), ((1, 2, 4, 4, 2048), (4, 4), 16),
    ((4, 2048), (4, 4), 16), ((2, 4, 4, 2048), (3, 4, 4), 16)])
def test_caches_that_are_none(kv, sc, page):
    kv = torch.zeros(kv, dtype=torch.int8)
    sc = torch.zeros(sc, dtype=torch.uint8)
    with pytest.raises(oa.OmniAttnError) as e:
        oa._take("p", "kv", -1, kv, sc, page)
    assert "kv" in str(e.value)
    with pytest.raises(oa.OmniAttnError):
        oa._take("p", "kv", -1, kv, None, page)  # not bf16


def test_the_references_on_a_case_by_hand():
    table = np.array([[3, 1, 5], [-1, -1, -1], [-1, -1, -1]])
    free, shares = np.array([0, 2, 4, 6, 7, -1, -1, -1]), np.zeros(8, np.int64)
    src, dst, st = R.fork([0, 0], [1, 2], [40, 32], 16, table, free, [0, 5], shares)
    assert (src, dst, st) == ([5, -1], [0, -1], [0, 1, 4, 1, 4])
    assert table.tolist() == [[3, 1, 5], [3, 1, 0], [3, 1, -1]] and shares.tolist() == [0, 2, 0, 2, 0, 0, 0, 0]
    assert R.give_back([0, 1], [40, 40], 16, table, free, [1, 4], shares) == [0, 2, 6, 1, 6]
    assert free.tolist() == [0, 2, 4, 6, 7, 0, 5, -1] and shares.tolist() == [0] * 8
    out, st = R.compact(table[2:], free, [1, 6], shares, 3, 4)
    assert st == [0, 1, 1, 0, 6] and out["table"].tolist() == [[0, 1, -1]]
    assert out["src"].tolist() == [3, -1, -1, -1] and out["dst"].tolist() == [0, -1, -1, -1]
    assert out["free"].tolist() == [2, 3, 4, 5, 6, 7, -1, -1]
