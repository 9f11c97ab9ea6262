"""Attention over a cache with block scales, values that are not finite in the waves' second pass:
one and two K/V heads a wave, own keys and a prefix that stream blocks take."""
import pytest
import torch

from test_gpu_block_attention import BF, HF, case, run
from test_gpu_block_infinite import fill
from test_gpu_prefix_attention import reference

pytestmark = pytest.mark.gpu

BITS = pytest.mark.parametrize("bits", [8, 4])


def place(c, where):
    """(slot, which queries see it): request 0's last key, or the prefix's fourth (all see it)."""
    N = c["q"].shape[0]
    see = torch.zeros(N, dtype=torch.bool, device=c["q"].device)
    pos = int(c["lens"][0]) - 1 if where == "own" else 3
    see[:N if where == "prefix" else c["new"][0]] = True
    if where == "own":
        see[:c["new"][0] - 1] = False                        # the request's last query alone
    return int(c["table"][0, pos // c["P"]]) * c["P"] + pos % c["P"], see


def beside(got, clean, hit):
    """What is not hit is as it was."""
    off = (got.double() - clean[0]).abs()[~hit]
    assert torch.isfinite(got[~hit]).all() and (off <= clean[1][~hit]).all()


# by rows: 4 or 8 of a head (two heads of 4 bits a wave), 12 (one)
@pytest.mark.parametrize("new", [[1, 1], [2, 1], [3, 1]], ids=["1", "2", "3"])
@pytest.mark.parametrize("where,prefix", [("own", 0), ("own", 40), ("prefix", 40)])
@pytest.mark.parametrize("Hk", [1, 2, 5, 8])
@pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "fp16"])
@BITS
def test_nan_in_one_head(pkg, gpu, bits, dtype, Hk, where, prefix, new):
    """A NaN in V of one head reaches that head's queries that see the key, in its block's 32 values; a NaN
    in K all their values; the pair's other head, the other rows and values stay."""
    lens = [prefix + n + 20 for n in new]
    c = case(pkg, gpu, 8 + Hk, lens, new, 4 * Hk, Hk, 64, dtype, bits, 16, prefix)
    clean = reference(c)
    slot, see = place(c, where)
    was = c["data"].clone()
    for head in {0, min(1, Hk - 1), Hk - 1}:
        for half in (1, 0):
            c["data"].copy_(was)
            fill(c, slot, half, head, 1, 1, 255, bits)
            got = run(pkg, c, cu_q=c["cu"], max_q=max(new))
            hit = torch.zeros(got.shape, dtype=torch.bool, device=gpu)
            hit[see, 4 * head:4 * head + 4, 32 if half else 0:] = True
            assert torch.isnan(got[hit]).all()
            beside(got, clean, hit)


@pytest.mark.parametrize("new", [[1, 1], [2, 1], [3, 1], [150, 70]], ids=["1", "2", "3", "150"])
@pytest.mark.parametrize("where,prefix", [("own", 0), ("own", 40), ("prefix", 40)])
@pytest.mark.parametrize("D", [64, 128, 256])
@BITS
def test_values_that_float16_makes_infinite(pkg, gpu, bits, D, where, prefix, new):
    """A block of V past 65504 in head 0, under -65504 in head 1: infinite for the queries that see it."""
    lens = [prefix + n + 20 for n in new]
    c = case(pkg, gpu, D, lens, new, 8, 2, D, HF, bits, 16, prefix)
    clean = reference(c)
    slot, see = place(c, where)
    code, scale = (0x7E, 127 + 10) if bits == 8 else (0x7, 127 + 14)    # 448 * 2^10, 6 * 2^14
    block = D // 32 - 1
    fill(c, slot, 1, 0, block, code, scale, bits)
    fill(c, slot, 1, 1, block, code | (0x80 if bits == 8 else 8), scale, bits)
    got = run(pkg, c, cu_q=c["cu"], max_q=max(new))
    hit = torch.zeros(got.shape, dtype=torch.bool, device=gpu)
    hit[see, :, block * 32:] = True
    assert (got[see, :4, block * 32:] == float("inf")).all() and (got[see, 4:, block * 32:] == float("-inf")).all()
    beside(got, clean, hit)
