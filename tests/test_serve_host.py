"""The 8-bit serving calls without a GPU: plans, work lists and refusals. Nothing
is launched: every C call here is refused or has nothing to do (pointers are made
up), and the Python mirror is given host tensors."""
import ctypes

import numpy as np
import pytest
import torch

import omni_attn as oa
import serve_refs as R

P = 0x10000  # a made-up, aligned address


# ------------------------------------------------------------------ plans
@pytest.mark.parametrize("rows,hk,max_len,chunk,splits", [
    (1, 8, 1, 64, 1), (1, 8, 300, 320, 1), (1, 8, 2400, 128, 19), (1, 8, 8000, 256, 32), (1, 1, 40000, 768, 53),
    (4, 8, 512, 512, 1), (16, 8, 2400, 256, 10), (32, 8, 1000, 1024, 1), (64, 8, 2400, 2432, 1), (21, 8, 5120, 512, 10),
    (128, 32, 3000, 3008, 1), (4, 8, 130000, 4096, 32),
])
def test_decode_plan_q8(rows, hk, max_len, chunk, splits):
    p = oa.decode_plan_q8(rows, 2 * hk, hk, 16, max_len)
    assert (p.chunk, p.splits, p.group_heads) == (chunk, splits, 0)
    assert p.workspace_bytes == (rows * 2 * hk * splits * 129 * 4 if splits > 1 else 0)


def test_decode_plan_q8_bounds():
    for rows, hk, max_len in ((0, 8, 5), (65535, 1, 100000), (1, 1, 2**31 - 1), (65535, 8, 2**31 - 1)):
        p = oa.decode_plan_q8(rows, hk, hk, 16, max_len)
        assert p.chunk % 64 == 0 and p.splits == -(-max_len // p.chunk)
    assert oa.decode_plan_q8(2, 32, 2, 256, 700, chunk=192).splits == 4
    for args in ((-1, 8, 8, 16, 9), (65536, 8, 8, 16, 9), (1, 9, 8, 16, 9), (1, 0, 8, 16, 9), (1, 8, 0, 16, 9),
                 (1, 8, 8, 0, 9), (1, 8, 8, 16, 0), (1, 8, 8, 16, 9, 100)):
        with pytest.raises(oa.OmniAttnError) as e:
            oa.decode_plan_q8(*args)
        assert e.value.code == oa.EINVAL
    for args in ((1, 17, 1, 16, 9), (1, 8, 8, 24, 9), (65535, 65536, 65536, 16, 9)):
        with pytest.raises(oa.OmniAttnError) as e:
            oa.decode_plan_q8(*args)
        assert e.value.code == oa.EUNSUPPORTED


def prompt_items(lens, hq, hk):
    pp = oa.prompt_plan(lens, hq, hk, device="cpu")
    work = pp.work.numpy()
    items = work[16:16 + 4 * pp.plan.tiles * hk].reshape(-1, 4)
    return pp.plan, work[:9], items


@pytest.mark.parametrize("hq,hk", [(1, 1), (16, 8), (32, 8), (8, 1), (3, 3)])
def test_prompt_plan_covers_every_row_once(hq, hk):
    lens = [0, 1, 31, 32, 33, 0, 128, 500, 64, 0]
    plan, ranges, items = prompt_items(lens, hq, hk)
    per = 256 // (hq // hk)
    starts = np.concatenate([[0], np.cumsum(lens)])
    seen = np.zeros((sum(lens), hk), int)
    for begin, first, rows, head in items:
        s = int(np.searchsorted(starts, first, side="right")) - 1
        while lens[s] == 0:
            s -= 1
        assert begin == starts[s] and (first - begin) % per == 0 and 1 <= rows <= per and first + rows <= starts[s + 1]
        seen[first:first + rows, head] += 1
    assert (seen == 1).all() and plan.rows == sum(lens) and plan.nseq == len(lens)
    assert plan.tiles == sum(-(-n // per) for n in lens)
    assert ranges[0] == 0 and ranges[8] == plan.tiles * hk and (np.diff(ranges) >= 0).all() and np.ptp(np.diff(ranges)) <= 1
    assert plan.workgroups == -(-plan.tiles * hk // 8) * 8


def test_prompt_plan_bounds():
    plan, _, _ = prompt_items([], 4, 2)
    assert plan.tiles == 0 and plan.rows == 0
    for lens, hq, hk, code in (([-1], 4, 2, oa.EINVAL), ([5], 5, 2, oa.EINVAL), ([5], 0, 2, oa.EINVAL), ([5], 6, 2, oa.EUNSUPPORTED),
                               ([5], 32, 2, oa.EUNSUPPORTED), ([2**31 - 1, 2**31 - 1], 4, 4, oa.EUNSUPPORTED)):
        with pytest.raises(oa.OmniAttnError) as e:
            oa.prompt_plan(lens, hq, hk, device="cpu")
        assert e.value.code == code
    L, plan = oa.load(), oa.PromptPlan()
    lens = np.array([300], np.int32)
    work = np.zeros(20, np.int32)
    rc = L.omni_attn_prompt_plan_init(1, lens.ctypes.data_as(ctypes.c_void_p), 8, 8, work.ctypes.data_as(ctypes.c_void_p), 20,
                                      ctypes.byref(plan))
    assert rc == oa.EWORKSPACE and plan.work_bytes == (16 + 4 * 2 * 8) * 4
    assert L.omni_attn_prompt_plan_init(1, None, 8, 8, None, 0, ctypes.byref(plan)) == oa.EINVAL
    assert L.omni_attn_prompt_plan_init(1, None, 8, 8, None, 0, None) == oa.EINVAL


# ------------------------------------------------------------------ refusals of the C calls
def tables(**k):
    a = dict(first=P, count=P, lines=P, nseq=2, page=16, ring=0, table=P, ld=4, num_lines=2, free=P, num_pages=9, state=P + 64,
             row_cap=4, page_cap=4, pos=P, slots=P, seq=P, row_indptr=P, indptr=P, pages=P, status=P)
    a.update(k)
    return oa.load().omni_attn_step_tables(*a.values(), None)


@pytest.mark.parametrize("bad", [
    dict(nseq=-1), dict(page=0), dict(ring=-1), dict(ld=-1), dict(num_lines=-1), dict(row_cap=-1), dict(page_cap=-1),
    dict(row_cap=2**31 - 1), dict(page_cap=2**31 - 1), dict(first=None), dict(count=None), dict(table=None), dict(pos=None),
    dict(slots=None), dict(seq=None), dict(row_indptr=None), dict(indptr=None), dict(pages=None), dict(status=None),
    dict(state=None), dict(num_pages=0), dict(num_pages=2**28), dict(state=P), dict(state=P + 16), dict(state=P - 4),
])
def test_step_tables_refusals(bad):
    assert tables(**bad) == oa.EINVAL
    assert b"step_tables" in oa.load().omni_attn_last_error()


def write(**k):
    a = dict(qkv=P, ld=1024, qn=P, kn=P, pos=P, slots=P, q=P, q_ld=512, k=P, k_ld=256, kv=P, scale=P, fmt=0, rows=3, hq=4, hk=2,
             eps=1e-6, theta=1e6)
    a.update(k)
    return oa.load().omni_qwen3_rope_q8(*a.values(), None)


@pytest.mark.parametrize("bad", [
    dict(rows=-1), dict(hq=0), dict(hk=0), dict(fmt=2), dict(fmt=-1), dict(qkv=None), dict(qn=None), dict(kn=None), dict(pos=None),
    dict(slots=None), dict(q=None), dict(kv=None), dict(scale=None), dict(qkv=P + 8), dict(q=P + 2), dict(k=P + 4), dict(kv=P + 8),
    dict(qn=P + 8), dict(ld=1016), dict(ld=1028), dict(q_ld=504), dict(q_ld=515), dict(k_ld=248), dict(k_ld=257), dict(eps=-1.0),
    dict(eps=float("nan")), dict(theta=0.0), dict(theta=float("inf")),
])
def test_rope_q8_refusals(bad):
    assert write(**bad) == oa.EINVAL


def test_rope_q8_of_no_rows_and_too_many_heads():
    assert write(rows=0, qkv=None, q=None, kv=None) == oa.OK
    assert write(hk=70000, ld=(4 + 140000) * 128, k_ld=70000 * 128) == oa.EUNSUPPORTED


def attend(plan=None, **k):
    plan = plan or oa.decode_plan_q8(3, 4, 2, 16, 100)
    a = dict(q=P, stride=512, kv=P, scale=P, fmt=0, pos=P, seq=P, ragged=0, indptr=P, pages=P, page=16, out=P, hq=4, hk=2,
             scale_=0.1, plan=ctypes.byref(plan), ws=None)
    a.update(k)
    return oa.load().omni_qwen3_attend_q8(*a.values(), None)


@pytest.mark.parametrize("bad", [
    dict(plan=None), dict(fmt=3), dict(page=32), dict(page=0), dict(hq=8), dict(hk=4), dict(hk=0), dict(q=None), dict(kv=None),
    dict(scale=None), dict(pos=None), dict(indptr=None), dict(pages=None), dict(out=None), dict(ragged=1, seq=None), dict(q=P + 8),
    dict(kv=P + 8), dict(out=P + 8), dict(stride=504), dict(stride=516), dict(scale_=float("nan")), dict(ws=P + 8),
])
def test_attend_q8_refusals(bad):
    if bad.get("plan", 1) is None:
        assert oa.load().omni_qwen3_attend_q8(P, 512, P, P, 0, P, P, 0, P, P, 16, P, 4, 2, 0.1, None, None, None) == oa.EINVAL
    else:
        assert attend(**bad) == oa.EINVAL


def test_attend_q8_plans_that_do_not_agree():
    for field, value in (("rows", -1), ("rows", 70000), ("max_len", 0), ("chunk", 32), ("chunk", 0), ("splits", 2), ("group_heads", 1)):
        plan = oa.decode_plan_q8(3, 4, 2, 16, 100)
        setattr(plan, field, value)
        assert attend(plan) == oa.EINVAL, field
    plan = oa.decode_plan_q8(3, 4, 2, 16, 1000, chunk=64)
    assert attend(plan) == oa.EWORKSPACE
    plan.workspace_bytes -= 1
    assert attend(plan, ws=P) == oa.EINVAL
    assert attend(oa.decode_plan_q8(0, 4, 2, 16, 100), q=None, kv=None) == oa.OK
    assert attend(page=24) == oa.EUNSUPPORTED


def prompt(plan=None, **k):
    if plan is None:
        plan = oa.prompt_plan([10], 4, 2, device="cpu").plan
    a = dict(plan=ctypes.byref(plan), q=P, qs=512, k=P, ks=256, v=P, vs=256, out=P, scale=0.1, work=P)
    a.update(k)
    return oa.load().omni_attn_prompt_run(*a.values(), None)


@pytest.mark.parametrize("bad", [
    dict(plan=None), dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(work=None), dict(q=P + 8), dict(k=P + 8),
    dict(v=P + 8), dict(out=P + 8), dict(qs=504), dict(qs=513), dict(ks=128), dict(ks=260), dict(vs=128), dict(vs=262),
    dict(ks=(1 << 22) + 8), dict(vs=(1 << 22) + 8), dict(scale=float("inf")),
])
def test_prompt_run_refusals(bad):
    if "plan" in bad:
        assert oa.load().omni_attn_prompt_run(None, P, 512, P, 256, P, 256, P, 0.1, P, None) == oa.EINVAL
    else:
        assert prompt(**bad) == oa.EINVAL


def test_prompt_run_plans_that_do_not_agree():
    for field, value in (("tiles", 2), ("tiles", -1), ("hq", 6), ("hk", 0), ("tile_rows", 128), ("workgroups", 16), ("work_bytes", 4),
                         ("exact_p", 2), ("rows", -1)):
        plan = oa.prompt_plan([10], 4, 2, device="cpu").plan
        setattr(plan, field, value)
        assert prompt(plan) == oa.EINVAL, field
    assert prompt(oa.prompt_plan([0], 4, 2, device="cpu").plan, q=None, k=None) == oa.OK


# ------------------------------------------------------------------ the mirror
def refused(f, *a, **k):
    with pytest.raises(oa.OmniAttnError) as e:
        f(*a, **k)
    assert e.value.code == oa.EINVAL


def test_the_mirror_refuses_host_tensors():
    i = lambda n: torch.zeros(n, dtype=torch.int32)
    b = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)
    kv, sc = oa.q8_cache(2, 16, 2, device="cpu")
    refused(oa.step_tables, i(2), i(2), i(2), i(8).view(2, 4), i(9), i(2), i(4), i(4), i(4), i(3), i(3), i(4), i(5))
    refused(oa.qwen3_rope_q8, b(3, 1024), b(128), b(128), i(3), i(3), b(3, 512), b(3, 256), kv, sc, 4, 2, 1e-6, 1e6)
    plan = oa.decode_plan_q8(3, 4, 2, 16, 100)
    refused(oa.qwen3_attend_q8, b(3, 512), kv, sc, i(3), None, 0, i(4), i(4), 16, b(3, 512), 4, 2, 0.1, plan)
    refused(oa.prompt_run, oa.prompt_plan([3], 4, 2, device="cpu"), b(3, 512), b(3, 256), b(3, 256), b(3, 512), 0.1)


def test_q8_cache():
    kv, sc = oa.q8_cache(3, 64, 2, torch.int8, device="cpu")
    assert kv.shape == (12, 4, 2048) and kv.dtype == torch.int8 and not kv.any()
    assert sc.shape == (12, 4) and sc.dtype == torch.float8_e8m0fnu
    for a in ((3, 24, 2), (3, 0, 2), (-1, 16, 2), (1, 16, 0)):
        refused(oa.q8_cache, *a, device="cpu")
    refused(oa.q8_cache, 1, 16, 1, torch.float16, device="cpu")


# ------------------------------------------------------------------ the references themselves
def test_the_quantizer_reference_rounds_like_the_definition():
    """Every value of a block within half a step of what is stored (e4m3: relative 2^-4 of normals, 2^-10 of the scale below;
    integers: half a scale), the largest in range, and the exponent the smallest that does it."""
    g = torch.Generator().manual_seed(0)
    for fmt in R.TOP:
        x = (torch.randn(64, 128, generator=g, dtype=torch.float64) * torch.pow(2.0, torch.randint(-20, 20, (64, 1), generator=g))).bfloat16().double()
        for row in x:
            most = float(row.abs().max())
            e = R.exponent(most, fmt)
            scale = 2.0 ** (e - 127)
            assert most <= R.TOP[fmt] * scale and (e == 1 or most > R.TOP[fmt] * scale / 2)
            d = (R.rounded(row / scale, fmt) * scale - row).abs()
            bound = torch.maximum(row.abs() * 2.0 ** -4, torch.tensor(2.0 ** -10 * scale)) if fmt == torch.float8_e4m3fn else 0.5 * scale
            assert bool((d <= bound).all())


def test_the_tables_reference_agrees_with_the_row_builder():
    first, count = [3, 16, 0], [20, 1, 5]
    table = np.arange(12, dtype=np.int32).reshape(3, 4)
    want = R.tables(first, count, None, table, None, None, 30, 30)
    rows = oa.Rows(16)
    for s in range(3):
        rows.push(table[s, :(first[s] + count[s] + 15) // 16], first[s], count[s], s)
    for mine, theirs in (("pos", rows.pos), ("slots", rows.slot), ("seq", rows.seq), ("indptr", rows.indptr), ("pages", rows.pages)):
        assert np.array_equal(want[mine], theirs), mine


def test_the_checks_of_tensors_name_the_one_at_fault():
    i, b = torch.zeros(6, dtype=torch.int32), torch.zeros(3, 8, dtype=torch.bfloat16)
    kv, sc = torch.zeros(2, 4, 2048, dtype=torch.int8), torch.zeros(2, 4, dtype=torch.uint8)

    def said(*a):
        with pytest.raises(oa.OmniAttnError) as e:
            oa._take(*a)
        assert e.value.args
        return str(e.value)

    assert "x must lie on the current device" in said("i", "x", 0, i, 6)
    assert "y must be a contiguous int32 tensor of at least 7" in said("Ii", "x y", 0, None, 0, i, 7)
    assert "y must be a contiguous bf16" in said("Ib", "x y", 0, None, 0, i, 1)
    assert "contiguous" in said("i", "x", 0, i[::2], 1)
    assert "rows must be bf16 rows [4][8]" in said("r", "rows", 0, b, 4, 8)
    assert "rows must be bf16 rows [3][9]" in said("r", "rows", 0, b, 3, 9)
    assert "adjacent" in said("r", "rows", 0, b.t(), 8, 3)
    assert "kv must be float8_e4m3fn or int8 [blocks][6][2048]" in said("c", "kv", 0, kv, sc, 6)
    assert "kv_scale" in said("c", "kv", 0, kv, sc[:1], 4)
    assert "x must be a tensor" in said("i", "x", 0, 5, 0)
    assert "x must be a tensor" in said("i", "x", 0, None, 0)
    assert "too few" in said("i", "x", 0, i) and "too many" in said("I", "x", 0, None, 0, 0)
    assert "integer" in said("i", "x", 0, i, "6") and "no such kind" in said("z", "x", 0, i, 0, 0)
    assert oa._take("IRI", "x y z", 0, None, 0, None, 1, 1, None, 0) == (None, None, 0, None)
