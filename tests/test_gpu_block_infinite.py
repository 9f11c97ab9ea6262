"""Attention over a cache with block scales whose values pass the queries' type: float16 makes
those past 65504 infinite, as reading them back does."""
import pytest
import torch

from test_gpu_block_attention import again, case, check, run
from test_gpu_prefix_attention import reference

pytestmark = pytest.mark.gpu

HF = torch.float16


def fill(c, slot, half, head, block, code, scale, bits, layer=1):
    """The 32 values of a block of one key: one code, one scale."""
    Hk, D = c["pool"].shape[4:]
    flat = c["data"].view(c["data"].shape[0], -1, 2, c["data"].shape[-1])
    rec = flat[layer, slot, half]
    at = head * D + block * 32
    rec[at * bits // 8:(at + 32) * bits // 8] = code if bits == 8 else code * 17
    rec[Hk * D * bits // 8 + at // 32] = scale


@pytest.mark.parametrize("new,prefix", [([1, 1], 0), ([1, 1, 1], 40), ([70, 3], 0), ([40, 40, 40], 25)])
@pytest.mark.parametrize("D", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("bits", [8, 4])
def test_keys_of_minus_infinity(pkg, gpu, D, bits, new, prefix):
    """A key whose product with every query is -infinity has weight 0: the definition without that key.
    Pages of one token, so that leaving a key out is a hole in the table."""
    lens = [prefix + n + 30 for n in new]
    c = case(pkg, gpu, D, lens, new, 4, 2, D, HF, bits, 1, prefix)
    c["q"].copy_(c["q"].abs().clamp_min(2.0 ** -8))
    code, scale = (0xFE, 127 + 10) if bits == 8 else (0xF, 127 + 14)    # -448 * 2^10, -6 * 2^14
    gone = c["table"].clone()
    places = [(0, prefix + 3)] + ([(0, 7)] if prefix else [])
    for block in {0, D // 32 - 1}:
        again(pkg, c)
        for b, pos in places:
            for head in range(2):
                fill(c, int(c["table"][b, pos]), 0, head, block, code, scale, bits)
            gone[b, pos] = -1
        got = run(pkg, c, cu_q=c["cu"], max_q=max(new))
        again(pkg, c)
        check(got, reference(dict(c, table=gone)))
