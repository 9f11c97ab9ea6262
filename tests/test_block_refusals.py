"""What a cache with block scales refuses, on the host, before anything is launched."""
import ctypes as C

import pytest
import torch

BF = torch.bfloat16


@pytest.fixture
def no_gpu():
    """Made-up addresses and CPU tensors must not reach a launch."""
    if torch.cuda.is_available():
        pytest.skip("CPU-only test")


def data(bs, heads=2, dim=64, bits=8, layers=1, pages=3, pt=4):
    return torch.zeros(layers, pages, pt, 2, bs.half_bytes(heads, dim, bits), dtype=torch.uint8)


def test_sizes(pkg):
    bs = pkg.blockscale
    assert bs.half_bytes(8, 128, 8) == 1056 and bs.half_bytes(8, 128, 4) == 544
    assert bs.half_bytes(1, 32, 4) == 32 and bs.half_bytes(3, 96, 4) == 160
    for bad in ((0, 64, 8), (2, 16, 8), (2, 80, 8), (2, 288, 8), (2, 64, 6), (2, 0, 4)):
        with pytest.raises(ValueError):
            bs.half_bytes(*bad)


def test_pool(pkg):
    bs = pkg.blockscale
    p = bs.BlockPool(data(bs), 2, 64, 8)
    assert p.shape == (1, 3, 4, 2, 2, 64) and p.records.shape == (1, 3, 4, 2, 1, 144) and p.code == 4
    assert p.layer(0) == (p.data.data_ptr(), 12)
    with pytest.raises(ValueError):
        p.layer(1)
    with pytest.raises(ValueError):
        bs.BlockPool(data(bs), 2, 64, 4)                     # of other records
    with pytest.raises(ValueError):
        bs.BlockPool(data(bs).to(torch.int16), 2, 64, 8)
    with pytest.raises(ValueError):
        bs.BlockPool(data(bs)[0], 2, 64, 8)
    with pytest.raises(ValueError):
        bs.BlockPool(data(bs, pages=6)[:, ::2], 2, 64, 8)    # not contiguous
    z = bs.BlockPool.zeros(2, 3, 4, 2, 64, 4, device="cpu")
    assert z.bits == 4 and not z.data.any()


def test_read_refuses(pkg, no_gpu):
    bs = pkg.blockscale
    p = bs.BlockPool(data(bs), 2, 64, 8)
    slots = torch.zeros(3, dtype=torch.int32)
    for args, kw in (((data(bs), slots), {}), ((p, slots.long()), {}), ((p, slots.view(1, 3)), {}),
                     ((p, torch.zeros(6, dtype=torch.int32)[::2]), {}), ((p, slots, torch.float64), {}),
                     ((p, slots), {"layer": 1}), ((p, slots), {"layer": -1}), ((p, slots), {})):   # the last: not on a GPU
        with pytest.raises(ValueError):
            bs.read(*args, **kw)


def test_write_and_attention_refuse(pkg, no_gpu):
    bs, at = pkg.blockscale, pkg.attention
    p = bs.BlockPool(data(bs), 2, 64, 8)
    q, k = torch.zeros(2, 4, 64, dtype=BF), torch.zeros(2, 2, 64, dtype=BF)
    slots = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        at.norm_rotate_write(q, k, k, None, None, p, slots)  # not on a GPU
    with pytest.raises(ValueError):
        at.prefix_attention(q, p, torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError):
        pkg.serving.PagedBackend(p, torch.zeros(1, 1, dtype=torch.int32), layer=1)


def norm_rotate(pkg, **kw):
    s = pkg._lib.NormRotate(tokens=2, heads=4, kv_heads=2, dim=64, dtype=1, q=4096, k=8192, v=12288, q_stride=256,
                            q_head_stride=64, k_stride=128, k_head_stride=64, v_stride=128, v_head_stride=64, q_out=16384,
                            o_stride=256, o_head_stride=64, norm=1, eps=1e-6, rot=0, axes=1, factor=1.0, pool=1 << 20,
                            pool_dtype=4, n_slots=8, slots=1 << 16)
    for name, x in kw.items():
        setattr(s, name, x)
    return pkg._lib.lib().kvec_norm_rotate_write(C.byref(s), None)


def test_write_checks_of_the_library(pkg, no_gpu):
    E, U = -1, -2
    assert norm_rotate(pkg, k_scale=64) == E                 # scales are an fp8 pool's
    assert norm_rotate(pkg, dim=80, q_head_stride=80, k_head_stride=80, v_head_stride=80) == U
    assert norm_rotate(pkg, dim=288) == U
    assert norm_rotate(pkg, pool_dtype=6) == E
    assert norm_rotate(pkg, pool=(1 << 20) + 8) == E         # not 16-byte aligned
    assert norm_rotate(pkg, pool=4096 - 64) == E             # over q
    assert norm_rotate(pkg, tokens=1 << 33) == E             # so many rows of q lie over the pool
    assert norm_rotate(pkg, tokens=1 << 33, k=1 << 45, v=1 << 46, q_out=1 << 47, slots=1 << 48, pool=1 << 49) == U
    assert norm_rotate(pkg, tokens=0) == 0


def block_read(pkg, **kw):
    s = pkg._lib.BlockRead(tokens=4, kv_heads=2, dim=64, pool_dtype=4, pool=1 << 20, n_slots=8, slots=4096, dtype=1, k=8192,
                           v=16384)
    for name, x in kw.items():
        setattr(s, name, x)
    return pkg._lib.lib().kvec_block_read_kv(C.byref(s), None)


def test_read_checks_of_the_library(pkg, no_gpu):
    E, U = -1, -2
    L = pkg._lib.lib()
    assert L.kvec_block_read_kv(None, None) == E
    for bad in (dict(tokens=-1), dict(kv_heads=0), dict(dim=0), dict(n_slots=-1), dict(pool_dtype=3), dict(pool_dtype=1),
                dict(dtype=3), dict(dtype=4), dict(slots=None), dict(k=None), dict(v=None), dict(pool=None), dict(k=8200),
                dict(pool=(1 << 20) + 4), dict(v=8192), dict(v=8192 + 512), dict(k=(1 << 20) + 16), dict(slots=8192)):
        assert block_read(pkg, **bad) == E, bad
    assert block_read(pkg, dim=48) == U and block_read(pkg, dim=288) == U
    assert block_read(pkg, tokens=1 << 40) == U and block_read(pkg, kv_heads=1 << 30) == U
    assert block_read(pkg, tokens=0) == 0


def attention(pkg, **kw):
    s = pkg._lib.Attention(tokens=2, batch=2, heads=4, kv_heads=2, dim=64, dtype=1, q=4096, q_stride=256, q_head_stride=64,
                           out=8192, o_stride=256, o_head_stride=64, pool=1 << 20, pool_dtype=5, pool_pages=2, page_tokens=4,
                           page_table=16384, pages_per_seq=2, seq_lens=20480, max_q=1, max_len=0, prefix=0, scale=0.1)
    for name, x in kw.items():
        setattr(s, name, x)
    need = pkg._lib.lib().kvec_prefix_attention_workspace(C.byref(s))
    return need if need < 0 else pkg._lib.lib().kvec_prefix_attention(C.byref(s), None, 0, None)


def test_attention_checks_of_the_library(pkg, no_gpu):
    assert attention(pkg, k_scale=64) < 0 and attention(pkg, v_scale=64) < 0
    assert attention(pkg, dim=80) < 0 and attention(pkg, dim=16) < 0
    assert attention(pkg, pool_dtype=7) < 0 and attention(pkg, pool=(1 << 20) + 8) < 0
    assert attention(pkg, out=(1 << 20) + 64) < 0            # inside the pool
    assert attention(pkg, tokens=0, batch=0) == 0


@pytest.mark.parametrize("bits", [4, 5])
def test_workspace_over_sizes(pkg, bits):
    """The plan for every batch and length up to the largest: a size that its launch can have, or a refusal."""
    L = pkg._lib.lib()
    for B in (1, 2, 7, 64, 1000, 60000):
        for heads, kv in ((1, 1), (4, 4), (7, 1), (12, 3), (32, 8), (71, 1), (64, 64)):
            for dim in (32, 96, 128, 256):
                for cap, prefix in ((1, 0), (100, 0), (100000, 0), (1 << 20, 70000), (1000, 1000)):
                    for new in (1, 3, 40):
                        s = pkg._lib.Attention(tokens=B * new, batch=B, heads=heads, kv_heads=kv, dim=dim, dtype=1, pool_dtype=bits,
                                               pool_pages=1 << 20, page_tokens=16, pages_per_seq=-(-cap // 16) if cap < 1 << 19 else 1 << 16,
                                               prefix=prefix if prefix < cap else 0, max_q=new, cu_q=64 if new > 1 else None, scale=1.0)
                        n = L.kvec_prefix_attention_workspace(C.byref(s))
                        assert n >= -1
                        if n > 0:                        # 512 parts of each row at most, of the prefix and of the own keys
                            assert n <= B * new * heads * 1024 * (4 * dim + 8) + 16


def test_packed_read(pkg):
    """The descriptor as the wrapper packs it is the structure that the library reads."""
    L = pkg._lib
    fmt, cls = L.BLOCK_READ_FORMAT, L.BlockRead
    values = [(i * 7919 + 3) % 1000 + 1 for i in range(len(cls._fields_))]
    assert fmt.size == C.sizeof(cls)
    s = cls.from_buffer_copy(fmt.pack(*values))
    assert [getattr(s, name) for name, _ in cls._fields_] == values


@pytest.mark.parametrize("code, heads", [(4, 1 << 19), (5, 1 << 20)])
def test_records_that_count_past_32_bits(pkg, no_gpu, code, heads):
    """A token's K of 128 MiB and more: its codes' bits would not count in 32."""
    far = {n: (i + 1) << 40 for i, n in enumerate(("q", "k", "v", "q_out", "slots", "pool"))}
    assert norm_rotate(pkg, tokens=1, heads=1, kv_heads=heads, dim=256, q_head_stride=256, k_head_stride=256,
                       v_head_stride=256, o_head_stride=256, pool_dtype=code, n_slots=1, **far) == -2
    assert block_read(pkg, tokens=1, kv_heads=heads, dim=256, pool_dtype=code, n_slots=1, k=1 << 40, v=1 << 41, pool=1 << 42) == -2
    s = dict(tokens=1, batch=1, heads=heads, kv_heads=heads, dim=256, pool_dtype=code, pool_pages=1, q_head_stride=256,
             o_head_stride=256, q=1 << 40, out=1 << 41, pool=1 << 42)
    assert attention(pkg, **s) == -2
