"""The cache write's form for many tokens (four query rows a group, K and V by one wave) over a cache with
block scales, in 16-bit types with heads of two rows a group and more; and types and heads that do not take it."""
import pytest
import torch

from test_gpu_block_scale import BF, HF, FF, case, check, go

pytestmark = pytest.mark.gpu


def among_many(pkg, gpu, c, n, **kw):
    """The case's tokens among n, the others without a slot; queries of all, bytes of the whole pool."""
    g = torch.Generator().manual_seed(n)
    x = torch.randn(n, c["x"].shape[1], generator=g).to(c["dtype"])
    at = torch.randperm(n, generator=g)[:c["N"]].sort().values
    at[-1] = n - 1
    x[at] = c["x"]
    slots = torch.full((n,), -1, dtype=torch.int32)
    slots[at] = c["slots"]
    pos = torch.zeros(n, dtype=torch.int32)
    pos[at] = c["pos"]
    got, data = go(pkg, gpu, dict(c, x=x, slots=slots, pos=pos, N=n), **kw)
    check(c, got[at], data)
    return x, got


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "fp16"])
@pytest.mark.parametrize("D", [32, 64, 96, 128, 160, 192, 224, 256])
def test_every_head_size(pkg, gpu, D, dtype, bits):
    """Two rows a group at least (heads of 32 values: 32 groups), whole and not, turned in both ways, in part
    and not at all; tokens on either side of the form's border."""
    lanes = 1 << (D // 16 - 1).bit_length()
    groups = 64 // lanes
    for Hq, Hk, rot, inter in ((groups + 1, 2, D, False), (4 * groups + 3, groups + 2, D // 2 // 16 * 16, True), (2 * groups, 1, 0, False)):
        c = case(D + Hq, 24, Hq, Hk, D, rot, dtype, bits, interleaved=inter)
        waves = -(-Hq // groups) + 2 * -(-Hk // groups)
        border = -(-2 * 256 * 32 // waves)
        for n in (border - 1, border):
            among_many(pkg, gpu, c, n)


@pytest.mark.parametrize("bits", [8, 4])
def test_on_either_side(pkg, gpu, bits):
    """A token's bytes and queries are the same in both forms, and in place as apart."""
    c = case(7, 30, 40, 8, 128, 128, BF, bits)
    few, _ = go(pkg, gpu, c)
    x, got = among_many(pkg, gpu, c, 4096)
    at = [int((x == row).all(1).nonzero()[0]) for row in c["x"][:5]]
    assert torch.equal(got[at], few[:5])
    among_many(pkg, gpu, c, 4096, in_place=True)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype,Hq,Hk,D", [(FF, 32, 8, 128), (FF, 12, 4, 256), (BF, 8, 2, 64), (HF, 4, 4, 128)])
def test_many_tokens_one_row_a_group(pkg, gpu, dtype, Hq, Hk, D, bits):
    c = case(Hq + D, 24, Hq, Hk, D, D, dtype, bits)
    among_many(pkg, gpu, c, 9000)
