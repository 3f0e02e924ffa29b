"""The tiled attention calls (packed prompts, paged prefill, DiT) at scales of
zero and below: every finite scale weighs the keys that a row sees and no other."""
import numpy as np
import pytest
import torch

import omni_attn as oa
import workloads as W
from gpu_util import dev_bits, dev_i32
from test_prompt_gpu import check, make, run
from test_tiled_gpu import dit_path

pytestmark = pytest.mark.gpu

SCALES = [0.0, -128 ** -0.5, -0.3]


@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("exact_p", [False, True])
@pytest.mark.parametrize("lens,hq,hk", [([1, 2, 33, 127, 128, 129, 0, 300], 8, 2), ([187], 16, 8), ([900, 700, 90], 32, 8), ([1500], 16, 16)])
def test_prompts(lens, hq, hk, exact_p, scale):
    qkv = make(lens, hq, hk, seed=hq)
    check(run(qkv, lens, hq, hk, exact_p, scale), qkv, lens, hq, hk, exact_p, scale)


def within(got, q, k, v, lims, scale):
    """got and q [rows][128], k and v [keys][128] (f64); row n sees lims[n] keys. The bound of test_prompt_gpu's check."""
    hidden = torch.arange(k.shape[0], device=q.device)[None] >= lims[:, None]
    p = torch.softmax((q @ k.t() * scale).masked_fill(hidden, -float("inf")), -1)
    want, size = p @ v, p @ v.abs()
    bound = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -13) * size
    assert bool(((got - want).abs() <= bound).all())


@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("page", [16, 12])
def test_paged_prefill(page, scale):
    c = W.ragged_prefill_case(3, 8, 2, 1, 300, 0, 200, page=page, seed=page)
    pf = oa.prefill_plan(c.rows, c.hq, c.hk, c.page, c.seq, c.pos)
    out = torch.zeros(c.rows, c.hq * 128, dtype=torch.bfloat16, device="cuda")
    qkv, kv = dev_bits(c.qkv), dev_bits(c.kv)
    oa.prefill_run(pf, qkv, kv, dev_i32(c.pos), dev_i32(c.seq), dev_i32(c.indptr), dev_i32(c.pages), out, scale)
    torch.cuda.synchronize()
    for s in range(3):
        rows = torch.from_numpy(np.flatnonzero(c.seq == s)).cuda()
        lims = torch.from_numpy(c.pos[c.seq == s].astype(np.int64) + 1).cuda()
        t = np.arange(int(lims.max()))
        slots = torch.from_numpy(c.pages[c.indptr[s] + t // page].astype(np.int64) * page + t % page).cuda()
        keys = kv[slots].double().view(len(t), 2 * c.hk, 128)
        x = qkv[rows].double().view(len(rows), -1, 128)
        o = out[rows].double().view(len(rows), c.hq, 128)
        for h in range(c.hq):
            kh = h // (c.hq // c.hk)
            within(o[:, h], x[:, h], keys[:, kh], keys[:, c.hk + kh], lims, scale)


@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("causal", [0, 1])
@pytest.mark.parametrize("q_len,paths", [(65, ("quarters", "quarters")), (300, ("halves", "halves")), (1100, ("halves", "2 chunks"))])
def test_dit(q_len, paths, causal, scale):
    hq, hk, kv_len = 32, 8, 300
    assert (dit_path(hq, hk, q_len, 2), dit_path(hq, hk, q_len, 2, ws=True)) == paths
    c = W.dense_case(hq, hk, q_len, kv_len, causal, batch=2, seed=q_len)
    q, k, v = dev_bits(c.q), dev_bits(c.k), dev_bits(c.v)
    bs = (q_len * c.q_stride, kv_len * hk * 128, q_len * hq * 128)
    lims = torch.full((q_len,), kv_len, device="cuda")
    if causal:
        lims = torch.minimum(lims, torch.arange(1, q_len + 1, device="cuda"))
    for ws in (None, oa.hidream_workspace()):
        out = torch.zeros(2, q_len, hq * 128, dtype=torch.bfloat16, device="cuda")
        oa.hidream_attend_ws(q, k, v, out, q_len, dev_i32(np.array([kv_len], np.int32)), c.q_stride, causal,
                             scale * 1.4426950408889634, hq, hk, 2, *bs, ws)
        torch.cuda.synchronize()
        for b in range(2):
            kk, vv = (t[b].double().view(kv_len, hk, 128) for t in (k, v))
            for h in range(0, hq, 5):
                x = q[b].view(q_len, -1)[:, h * 128:(h + 1) * 128].double()
                within(out[b, :, h * 128:(h + 1) * 128].double(), x, kk[:, h // 4], vv[:, h // 4], lims, scale)
