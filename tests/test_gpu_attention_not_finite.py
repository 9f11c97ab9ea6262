"""Values of V that are not finite, in keys that whole row tiles see: every query
that sees such a key gets them, whatever unit of 32 keys it lies in and wherever the
first key that some row of the tile does not see lies."""
import math

import pytest
import torch

from test_gpu_prefix_attention import BF, F8, HF, make, reference, run

pytestmark = pytest.mark.gpu


def plant(c, b, pos, kind, pool, gpu):
    """V of request b's key `pos`, the second K/V head's value 5."""
    raw = torch.uint8 if pool == F8 else torch.int16
    value = torch.tensor([kind], dtype=torch.float32).to(pool).view(raw)[0].to(gpu)
    page = int(c["table"][b, pos // c["P"]])
    c["pool"].view(raw)[1, page, pos % c["P"], 1, 1, 5] = value


def same_kind(got, kind):
    return torch.isnan(got).all() if math.isnan(kind) else (got == kind).all()


def compare(got, clean, hit, kind):
    assert hit.any()
    assert same_kind(got[hit], kind), f"{int(torch.isfinite(got[hit]).sum())} of {int(hit.sum())} finite"
    off = (got.double() - clean[0]).abs()[~hit]
    assert torch.isfinite(got[~hit]).all() and (off <= clean[1][~hit]).all()


KINDS = [float("nan"), float("inf"), -float("inf")]


@pytest.mark.parametrize("dtype,pool,D", [(BF, BF, 64), (HF, HF, 64), (BF, BF, 128), (HF, HF, 200), (BF, F8, 64)])
@pytest.mark.parametrize("cached", [0, 20, 70, 3000])
def test_seen_by_whole_tiles(pkg, gpu, dtype, pool, D, cached):
    """Own keys: the tiles' first unseen keys lie 32 keys apart, so in odd and even
    units; the value in each unit before them and several earlier.  3000: in splits."""
    new = [150, 70]
    lens = [n + cached for n in new]
    c = make(gpu, 31, lens, new, 8, 2, D, dtype, pool, 16, 0)
    clean, keep = reference(c), c["pool"].clone()
    for i, pos in enumerate(p for p in (0, 3, 31, 32, 40, 70, 100, cached - 300, cached - 90, cached - 2, cached + 75)
                            if 0 <= p < lens[0]):
        kind = KINDS[0 if pool == F8 else i % 3]
        c["pool"].copy_(keep)
        plant(c, 0, pos, kind, pool, gpu)
        got = run(pkg, c, cu_q=c["cu"], max_q=max(new))
        hit = torch.zeros(got.shape, dtype=torch.bool, device=gpu)
        hit[max(0, pos - cached):new[0], 4:8, 5] = True
        compare(got, clean, hit, kind)


@pytest.mark.parametrize("dtype,pool,D", [(BF, BF, 64), (HF, HF, 128), (BF, F8, 64)])
@pytest.mark.parametrize("prefix", [33, 48, 80, 112, 128, 2000])
@pytest.mark.parametrize("B", [6, 20])
def test_in_the_prefix(pkg, gpu, dtype, pool, D, prefix, B):
    """Shared keys, by stream and tile blocks: the first key that a row does not see
    lies right behind the prefix's end, in odd and even units."""
    lens = [prefix + 1 + (i * 7) % 40 for i in range(B)]
    c = make(gpu, 32, lens, [1] * B, 8, 2, D, dtype, pool, 16, prefix)
    clean, keep = reference(c), c["pool"].clone()
    for i, pos in enumerate(p for p in (0, 3, 32, 40, 70, prefix - 70, prefix - 40, prefix - 1) if 0 <= p < prefix):
        kind = KINDS[0 if pool == F8 else i % 3]
        c["pool"].copy_(keep)
        plant(c, 0, pos, kind, pool, gpu)
        got = run(pkg, c)
        hit = torch.zeros(got.shape, dtype=torch.bool, device=gpu)
        hit[:, 4:8, 5] = True
        compare(got, clean, hit, kind)
