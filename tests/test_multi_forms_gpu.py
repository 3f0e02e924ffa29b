"""Extend and cross attention in each form of a tile, with the sizes that choose the form pinned: quarters and halves where the items
(tiles times K/V heads) leave CUs over, whole tiles where they do not, where a split stands among them, and where a position's query
heads do not divide a tile."""
import numpy as np
import pytest
import torch

import test_multi_gpu as T

pytestmark = pytest.mark.gpu


def sequences(seqs, seed):
    rng = np.random.default_rng(seed)
    counts = [int(x) for x in rng.integers(34, 130, seqs)]
    return counts, [c + int(x) for c, x in zip(counts, rng.integers(0, 260, seqs))]


def form_of(plan):
    """By the rule of the launch: quarters if four workgroups an item fit the CUs, halves if two do."""
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    items, g = plan.tile_units * plan.hk, plan.hq // plan.hk
    if plan.split_tiles or 256 % g:
        return "whole"
    return "quarters" if 4 * items <= cus else "halves" if 2 * items <= cus else "whole"


# sequences, K/V heads, query heads of one: the form
CASES = [(1, 2, 2, "quarters"), (4, 8, 2, "quarters"), (12, 8, 2, "halves"), (20, 16, 2, "whole"), (34, 8, 2, "whole"),
         (1, 1, 16, "quarters"), (4, 4, 16, "halves"), (12, 8, 16, "whole"), (3, 4, 1, "quarters"), (3, 4, 8, "quarters"), (10, 4, 8, "halves"),
         (1, 1, 3, "whole"), (2, 2, 7, "whole")]


@pytest.mark.parametrize("fmt", T.FORMATS)
@pytest.mark.parametrize("seqs,hk,g,form", CASES)
def test_extend(seqs, hk, g, form, fmt):
    counts, lens = sequences(seqs, seqs + g)
    mp, _ = T.extend(T.Cache(seqs, lens, hk, 16, fmt), counts, g * hk, chunk=T.APART)
    assert mp.plan.tiles >= seqs and form_of(mp.plan) == form


@pytest.mark.parametrize("seqs,hk,g,form", CASES)
def test_cross(seqs, hk, g, form):
    counts, lens = sequences(seqs, seqs + g)
    lens[0] = 0 if seqs > 2 else lens[0]
    mp, _ = T.cross(seqs, counts, lens, g * hk, hk, chunk=T.APART)
    assert mp.plan.tiles > 0 and form_of(mp.plan) == form


@pytest.mark.parametrize("fmt", T.FORMATS)
def test_few_tiles_in_splits_are_whole(fmt):
    mp, _ = T.extend(T.Cache(2, [1500], 2, 16, fmt), [70], 4, chunk=T.APART)
    assert mp.plan.split_tiles > 0 and form_of(mp.plan) == "whole"
