"""Causal attention of packed prompts on the GPU against 64 bits, and bit for bit
against itself in other packings, orders and strides."""
import numpy as np
import pytest
import torch

import omni_attn as oa

pytestmark = pytest.mark.gpu


def make(lens, hq, hk, seed=0, extra=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows = sum(lens) + extra
    return torch.randn(rows, (hq + 2 * hk) * 128, device="cuda", generator=g).to(torch.bfloat16)


def parts(qkv, hq, hk):
    return qkv.split([hq * 128, hk * 128, hk * 128], dim=1)


def run(qkv, lens, hq, hk, exact_p=False, scale=128 ** -0.5, fill=7.0, stream=None):
    out = torch.full((qkv.shape[0], hq * 128), fill, dtype=torch.bfloat16, device="cuda")
    oa.prompt_run(oa.prompt_plan(lens, hq, hk, exact_p=exact_p), *parts(qkv, hq, hk), out, scale, stream)
    torch.cuda.synchronize()
    return out


def check(out, qkv, lens, hq, hk, exact_p=False, scale=128 ** -0.5):
    """Half a bf16 step (2^-8) of the result; P rounded to bf16 adds 2^-8 of sum p |v| (16 bits with exact_p: 2^-16), and
    2^-13 of it stands for the exponentials and f32 sums."""
    at = 0
    for n in lens:
        x = qkv[at:at + n].double().view(n, qkv.shape[1] // 128, 128)
        later = torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1)
        for h in range(hq):
            kh = hq + h // (hq // hk)
            p = torch.softmax((x[:, h] @ x[:, kh].t() * scale).masked_fill(later, -float("inf")), -1)
            want, size = p @ x[:, kh + hk], p @ x[:, kh + hk].abs()
            bound = 2.0 ** -8 * want.abs() + (2.0 ** -13 if exact_p else 2.0 ** -8 + 2.0 ** -13) * size
            d = (out[at:at + n, h * 128:(h + 1) * 128].double() - want).abs()
            assert bool((d <= bound).all()), f"prompt of {n} at {at}, head {h}: {float((d - bound).max()):.3g} past its bound"
        at += n


@pytest.mark.parametrize("hq,hk", [(1, 1), (4, 4), (16, 8), (8, 2), (8, 1), (3, 3), (32, 8)])
@pytest.mark.parametrize("exact_p", [False, True])
def test_matches_64_bits(hq, hk, exact_p):
    lens = [1, 2, 0, 31, 33, 127, 128, 129, 0, 257, 500, 7]
    qkv = make(lens, hq, hk, seed=hq, extra=3)
    out = run(qkv, lens, hq, hk, exact_p)
    check(out, qkv, lens, hq, hk, exact_p)
    assert bool((out[sum(lens):] == 7).all())  # rows behind the last prompt stay


@pytest.mark.parametrize("lens,hq,hk", [([1], 16, 8), ([187], 16, 8), ([2000], 16, 8), ([4100], 4, 1), ([1500, 1300, 90], 32, 8),
                                        ([64] * 40, 32, 8), ([1] * 300, 8, 8), ([700, 650], 16, 16)])
def test_forms_of_few_and_many_tiles(lens, hq, hk):
    qkv = make(lens, hq, hk, seed=len(lens))
    check(run(qkv, lens, hq, hk), qkv, lens, hq, hk)


@pytest.mark.parametrize("exact_p", [False, True])
def test_a_prompt_has_the_same_bits_in_any_packing(exact_p):
    hq, hk = 8, 2
    lens = [300, 77, 1, 1030, 0, 260]
    qkv = make(lens, hq, hk, seed=5)
    whole = run(qkv, lens, hq, hk, exact_p)
    at = 0
    for n in lens:
        if n:
            alone = run(qkv[at:at + n].contiguous(), [n], hq, hk, exact_p)
            assert torch.equal(alone, whole[at:at + n])
        at += n


def test_no_prompts_and_empty_prompts():
    qkv = make([], 4, 2, extra=2)
    for lens in ([], [0], [0, 0]):
        assert bool((run(qkv, lens, 4, 2) == 7).all())


def test_separate_and_strided_rows():
    hq, hk, lens = 8, 4, [130, 40, 300]
    qkv = make(lens, hq, hk, seed=2)
    want = run(qkv, lens, hq, hk)
    q, k, v = (t.contiguous() for t in parts(qkv, hq, hk))
    wide = torch.full((sum(lens), 2 * hk * 128 + 24), float("nan"), dtype=torch.bfloat16, device="cuda")
    wide[:, 16:16 + hk * 128], wide[:, 16 + hk * 128:16 + 2 * hk * 128] = v, k  # v before k, a stride of its own
    out = torch.zeros_like(want)
    oa.prompt_run(oa.prompt_plan(lens, hq, hk), q, wide[:, 16 + hk * 128:16 + 2 * hk * 128], wide[:, 16:16 + hk * 128], out,
                  128 ** -0.5)
    assert torch.equal(out, want)


def test_rows_of_other_prompts_do_not_matter():
    """NaN and infinities in one prompt stay there, and so does what lies before and behind the packed rows."""
    hq, hk, lens = 8, 2, [200, 150, 90]
    qkv = make(lens, hq, hk, seed=3)
    want = run(qkv, lens, hq, hk)
    bad = qkv.clone()
    bad[200:350] = float("nan")
    bad[210] = float("inf")
    out = run(bad, lens, hq, hk)
    assert torch.equal(out[:200], want[:200]) and torch.equal(out[350:], want[350:])
    assert bool(out[200:350].isnan().all())


def test_later_rows_of_a_prompt_do_not_matter():
    hq, hk, n = 4, 2, 300
    qkv = make([n], hq, hk, seed=4)
    want = run(qkv, [n], hq, hk)
    bad = qkv.clone()
    bad[201:, hq * 128:(hq + hk) * 128] = 1e30
    out = run(bad, [n], hq, hk)
    assert torch.equal(out[:201], want[:201])


def test_another_stream_and_replays():
    hq, hk, lens = 16, 8, [100, 300]
    qkv = make(lens, hq, hk, seed=6)
    plan = oa.prompt_plan(lens, hq, hk)
    out = torch.zeros(sum(lens), hq * 128, dtype=torch.bfloat16, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        oa.prompt_run(plan, *parts(qkv, hq, hk), out, 0.1)
    torch.cuda.synchronize()
    assert torch.equal(out, run(qkv, lens, hq, hk, scale=0.1))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        oa.prompt_run(plan, *parts(qkv, hq, hk), out, 0.1)
    for rep in range(3):
        qkv.copy_(make(lens, hq, hk, seed=20 + rep))
        want = run(qkv, lens, hq, hk, scale=0.1)
        out.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    assert np.isfinite(float(out.float().sum()))
