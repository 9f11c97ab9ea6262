"""Chunked coding of a cache with block scales: its records (codes, scales and the bytes that fill them up)
against the oracle, and rebuilt into the pool."""
import numpy as np
import pytest
import torch

from test_gpu_chunked import PATTERNS, erase

pytestmark = pytest.mark.gpu

# layers, sequences, pages a sequence, tokens a page, K/V heads, dim, k, p, m, tokens a chunk
CONFIGS = [(2, 3, 4, 16, 8, 128, 5, 7, 3, 16), (2, 2, 8, 8, 1, 32, 4, 5, 2, 16), (1, 2, 6, 16, 5, 96, 6, 7, 2, 32),
           (2, 1, 4, 4, 10, 128, 5, 7, 3, 4)]


def setup(pkg, gpu, cfg, bits, keep_data):
    """A pool written by the package, coded chunk by chunk."""
    L, B, pps, pt, H, D, k, p, m, ct = cfg
    pages = B * pps + 3
    pool = pkg.blockscale.BlockPool.zeros(L, pages, pt, H, D, bits, device=gpu)
    g = torch.Generator().manual_seed(sum(cfg))
    table = torch.randperm(pages, generator=g)[:B * pps].to(torch.int32).view(B, pps)
    slots = (table.view(-1, 1).long() * pt + torch.arange(pt)).reshape(-1).to(torch.int32).to(gpu)
    N = slots.numel()
    for layer in range(L):
        x = torch.randn(N, 3 * H, D, generator=g).to(torch.bfloat16).to(gpu)
        pkg.attention.norm_rotate_write(x[:, :H], x[:, H:2 * H], x[:, 2 * H:], None, None, pool, slots, layer=layer)
    table_d = table.to(gpu)
    kv = pkg.chunked.chunk_kv(pool, table_d, 0, ct)
    assert kv.token_bytes == pkg.blockscale.half_bytes(H, D, bits)
    st = pkg.chunked.ChunkedStripes(kv.stream_bytes(), 2 * kv.token_bytes, pps * pt // ct, gpu, k=k, p=p, m=m,
                                    keep_data=keep_data)
    for c in range(st.n_chunks):
        st.encode(pkg.chunked.chunk_kv(pool, table_d, c, ct), c)
    torch.cuda.synchronize()
    return pool, table, table_d, st


@pytest.mark.parametrize("cfg", CONFIGS)
@pytest.mark.parametrize("bits", [8, 4])
def test_encode_matches_oracle(pkg, ora, gpu, cfg, bits):
    L, B, pps, pt, H, D, k, p, m, ct = cfg
    pool, table, _, st = setup(pkg, gpu, cfg, bits, True)
    W, data, P, Q, rs = ora.chunked_encode(pool.data.cpu().numpy(), table.numpy(), pt, ct, st.n_chunks, k, p, m, st.unit_bytes)
    assert st.width == W
    for i, (got, want) in enumerate(zip(st.shards(), data + [P, Q] + rs)):
        assert np.array_equal(got.cpu().numpy(), want), i


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("keep_data", [True, False])
def test_lost_records_rebuilt(pkg, gpu, bits, keep_data):
    """Every pattern of lost shards: the pool's bytes and the parity as they were, tokens read back as before."""
    cfg = CONFIGS[0]
    pool, table, table_d, st = setup(pkg, gpu, cfg, bits, keep_data)
    ct = cfg[-1]
    was, shards = pool.data.clone(), [t.clone() for t in st.shards()]
    slots = torch.arange(pool.shape[1] * pool.shape[2], dtype=torch.int32, device=gpu)
    before = pkg.blockscale.read(pool, slots, torch.float32, layer=1)
    gen = torch.Generator().manual_seed(9)
    for i, er in enumerate(PATTERNS):
        c = i % st.n_chunks
        kv = pkg.chunked.chunk_kv(pool, table_d, c, ct)
        touched = erase(pkg, st, kv, c, er, gen)
        assert torch.equal(pool.data, was) != touched
        st.decode(kv, c, er)
        assert torch.equal(pool.data, was), er
        assert all(torch.equal(a, b) for a, b in zip(st.shards(), shards)), er
    assert all(torch.equal(a, b) for a, b in zip(before, pkg.blockscale.read(pool, slots, torch.float32, layer=1)))
