"""Plans of many short sequences beside a long one: the long one's keys are split however many tiles the others are."""
import numpy as np
import pytest
import torch

import omni_attn as oa
from test_multi_host import check_tiles, tile_items

PLANS = [oa.extend_plan, oa.cross_plan]


@pytest.mark.parametrize("make", PLANS)
@pytest.mark.parametrize("hq,hk,short,longest", [(16, 8, 47, 60000), (16, 8, 48, 60000), (16, 8, 400, 60000), (32, 8, 61, 20000), (4, 4, 2000, 200000),
                                                 (2, 1, 600, 100000), (3, 1, 600, 100000)])
def test_a_long_sequence_beside_short_ones_is_split(make, hq, hk, short, longest):
    g = hq // hk
    counts = [40 * 2 // g] * short + [120 * 2 // g]
    keys = [200] * short + [longest]
    mp = make(counts, hq, hk, longest, keys, device="cpu")
    check_tiles(mp, counts, keys, make is oa.extend_plan)
    p, machines = mp.plan, 256 // hk
    tiles = p.tiles
    assert tiles * 2 > 3 * machines or short == 47
    assert p.split_tiles >= 1 and p.tile_units - tiles <= 4 * machines
    # No workgroup walks much longer than the others keep the GPU busy.
    steps = -(-longest // 128)
    share = (2 * tiles + steps) / machines
    assert p.tile_chunk // 128 <= max(24, 3 * share), (p.tile_chunk // 128, share)


@pytest.mark.parametrize("make", PLANS)
def test_evenly_spread_lengths_stay_whole(make):
    rng = np.random.default_rng(3)
    for hq, hk, n, lo, hi in ((32, 8, 12, 512, 4096), (16, 8, 200, 40, 120), (16, 16, 80, 22, 157)):
        counts = [int(x) for x in rng.integers(lo, hi, n)]
        keys = [c + int(x) for c, x in zip(counts, rng.integers(0, 1024, n))]
        p = make(counts, hq, hk, max(keys), keys, device="cpu").plan
        assert p.split_tiles == 0 and p.tile_units == p.tiles


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [torch.float8_e4m3fn, torch.int8])
def test_against_64_bits(fmt):
    import test_multi_gpu as T

    counts, lens = [40] * 34 + [90], [60 + 3 * i for i in range(34)] + [9000]
    e, _ = T.extend(T.Cache(3, lens, 8, 16, fmt), counts, 16)
    assert e.plan.tiles == 35 and e.plan.split_tiles == 1
    counts, lens = [40] * 50 + [90], [60 + 3 * i for i in range(50)] + [30000]
    e, _ = T.cross(3, counts, lens, 16, 8)
    assert e.plan.tiles == 51 and e.plan.split_tiles >= 1
