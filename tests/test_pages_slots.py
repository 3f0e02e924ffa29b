"""pages_copy through the mirror over uint8 slots, as the FP8 calls take them: the header's call takes a cache of any format."""
import numpy as np
import pytest
import torch

import omni_attn as oa

HEADS = 3
SLOT = 2 * HEADS * 128 + 2 * HEADS * 4  # an FP8 slot: E4M3 bytes and their scales


def test_what_the_mirror_makes_of_them():
    kv = torch.zeros(2, 32, SLOT, dtype=torch.uint8)
    for good in (kv, kv[0]):  # but for lying on the host
        with pytest.raises(oa.OmniAttnError) as e:
            oa._take("p", "kv", -1, good, None, 16)
        assert "device" in str(e.value)
    for bad, page in ((kv[0, 0], 16), (kv[None], 16), (kv, 0), (kv, -16), (kv, 24), (kv[:, :, :16], 16), (kv.view(torch.int8), 16)):
        with pytest.raises(oa.OmniAttnError) as e:
            oa._take("p", "kv", -1, bad, None, page)
        assert e.value.code == oa.EINVAL and "device" not in str(e.value)


@pytest.mark.gpu
@pytest.mark.parametrize("layers,page", [(0, 16), (3, 4), (2, 2)])
def test_copy(layers, page):
    pages = 11
    g = torch.Generator(device="cuda").manual_seed(page)
    shape = (pages * page, SLOT) if layers == 0 else (layers, pages * page, SLOT)
    kv = torch.randint(0, 256, shape, dtype=torch.uint8, device="cuda", generator=g)
    want = kv.clone().view(max(layers, 1), pages, page * SLOT)
    ids = np.random.default_rng(page).permutation(pages)
    src, dst = ids[:4], ids[4:8]
    want[:, dst.tolist()] = want[:, src.tolist()]
    i32 = lambda a: torch.tensor(a.astype(np.int32), device="cuda")
    oa.pages_copy(kv, None, i32(src), i32(dst), page)
    torch.cuda.synchronize()
    assert torch.equal(kv.view(want.shape), want)
    if page == 2:  # a page of 2 x 792 bytes is a multiple of 16, one of 792 is not
        with pytest.raises(oa.OmniAttnError) as e:
            oa.pages_copy(kv, None, i32(src), i32(dst), 1)
        assert e.value.code == oa.EINVAL
