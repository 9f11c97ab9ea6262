"""Caches with block scales: every head size at the write's many-token form and its few-token
one, and records past 4 GiB."""
import pytest
import torch

from test_gpu_block_scale import BF, HF, case, check, go

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("D", [32, 64, 96, 128, 160, 192, 224, 256])
def test_every_head_size(pkg, gpu, D, bits):
    """Rows of two to sixteen lanes, turned whole, in part and not at all; of one head (lanes
    without a row) and more than a wave's rows."""
    for Hq, Hk, rot, inter in ((4, 2, D, False), (70, 67, D, True), (1, 1, D // 2 // 16 * 16, False), (9, 5, 0, False)):
        c = case(D + Hk, 11, Hq, Hk, D, rot, BF, bits, interleaved=inter)
        check(c, *go(pkg, gpu, c))


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("D", [32, 64, 96, 128, 160, 192, 224, 256])
def test_every_head_size_many_tokens(pkg, gpu, D, bits):
    """The same where tokens are many: K and V by one wave, four query rows a group."""
    n = 32768                                            # 4 + 2 x 2 heads: three waves a token at least
    c = case(D + bits, 40, 4, 2, D, D, HF, bits, interleaved=D % 64 == 0)
    g = torch.Generator().manual_seed(D)
    x = torch.randn(n, c["x"].shape[1], generator=g).to(HF)
    at = torch.randperm(n, generator=g)[:40].sort().values
    x[at] = c["x"]
    slots = torch.full((n,), -1, dtype=torch.int32)
    slots[at] = c["slots"]
    pos = torch.zeros(n, dtype=torch.int32)
    pos[at] = c["pos"]
    got, data = go(pkg, gpu, dict(c, x=x, slots=slots, pos=pos, N=n))
    check(c, got[at], data)


@pytest.mark.parametrize("bits", [8, 4])
def test_records_past_4_gib(pkg, gpu, bits):
    """Written, read and attended to at the end of a cache of more than 4 GiB as at its start."""
    Hq, Hk, D, P, own = 16, 8, 128, 16, 600
    half = pkg.blockscale.half_bytes(Hk, D, bits)
    pages = (1 << 32) // (2 * half * P) + 200
    pool = pkg.blockscale.BlockPool.zeros(1, pages, P, Hk, D, bits, device=gpu)
    assert pool.data.numel() > 1 << 32
    n = 2 * own
    g = torch.Generator().manual_seed(bits)
    x = torch.randn(n, Hq + 2 * Hk, D, generator=g).to(BF).to(gpu)
    per = -(-own // P)
    # two requests, pages in an order of their own; the same at the cache's end
    low = (torch.randperm(2 * per, generator=g)).view(2, per).to(torch.int32).to(gpu)
    i = torch.arange(own, device=gpu)
    outs = []
    for table in (low, low + (pages - 2 * per)):
        slots = (table[:, i // P] * P + i % P).reshape(-1).to(torch.int32)
        pkg.attention.norm_rotate_write(x[:, :Hq], x[:, Hq:Hq + Hk], x[:, Hq + Hk:], None, None, pool, slots)
        k, v = pkg.blockscale.read(pool, slots, BF)
        lens = torch.tensor([own, own - 37], dtype=torch.int32, device=gpu)
        few = pkg.attention.prefix_attention(x[:2, :Hq], pool, table, lens)
        cu = torch.tensor([0, 200, 400], dtype=torch.int32, device=gpu)
        many = pkg.attention.prefix_attention(x[:400, :Hq], pool, table, lens, cu_q=cu, max_q=200)
        outs.append((k, v, few, many))
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    assert all(t.float().abs().max() > 0.1 for t in outs[0])
