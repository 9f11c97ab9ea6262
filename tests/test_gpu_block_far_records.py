"""Records of a cache of more than 4 GiB, byte by byte: a token written to a far slot lies there, and
nowhere else.  (An address that lost its upper bits in the write, the read and the attention alike would
find its own token again.)"""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("tokens", [64, 32768], ids=["few", "many"])
def test_bytes_of_far_records(pkg, gpu, bits, tokens):
    Hq, Hk, D, P = 4, 8, 128, 16
    half = pkg.blockscale.half_bytes(Hk, D, bits)
    pages = (1 << 32) // (2 * half * P) + 2 * tokens // P + 100
    pool = pkg.blockscale.BlockPool.zeros(1, pages, P, Hk, D, bits, device=gpu)
    flat = pool.data.view(-1, 2, half)
    n = flat.shape[0]
    assert (n - tokens) * 2 * half > 1 << 32
    g = torch.Generator().manual_seed(bits)
    x = torch.randn(tokens, Hq + 2 * Hk, D, generator=g).to(torch.bfloat16).to(gpu)
    order = torch.randperm(tokens, generator=g).to(torch.int32).to(gpu)
    for first in (0, n - tokens):
        pkg.attention.norm_rotate_write(x[:, :Hq], x[:, Hq:Hq + Hk], x[:, Hq + Hk:], None, None, pool, order + first)
    near, far = flat[:tokens], flat[n - tokens:]
    assert torch.equal(near, far)
    assert near.view(tokens, -1).any(1).all()
    for at in range(tokens, n - tokens, 1 << 20):           # nothing else was written
        assert not flat[at:min(at + (1 << 20), n - tokens)].any()
    # read there and here: and not from where an address of 32 bits would lie
    k, v = pkg.blockscale.read(pool, order, torch.bfloat16)
    flat[:tokens] = 0
    k2, v2 = pkg.blockscale.read(pool, order + (n - tokens), torch.bfloat16)
    assert torch.equal(k, k2) and torch.equal(v, v2) and k.any() and v.any()
    table = torch.arange(n // P - tokens // P, n // P, dtype=torch.int32, device=gpu).view(1, -1)
    lens = torch.tensor([tokens], dtype=torch.int32, device=gpu)
    got = pkg.attention.prefix_attention(x[:1, :Hq * 2].contiguous(), pool, table, lens)
    flat[:tokens] = far
    here = pkg.attention.prefix_attention(x[:1, :Hq * 2].contiguous(), pool, table - table[0, 0], lens)
    assert torch.equal(got, here) and got.any()
