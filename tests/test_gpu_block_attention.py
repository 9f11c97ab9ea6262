"""Attention over a cache with block scales against the definition in 64 bits.

K and V are what the records stand for, exactly (16-bit types hold them), so the
tolerance is that of the attention over plain pools (test_gpu_prefix_attention).
"""
import math

import numpy as np
import pytest
import torch

import blockref as ref
from test_gpu_prefix_attention import check, make, reference

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
JUNK = 0xFF                                              # NaN: every code of e4m3, every scale


def blocks(pkg, c, bits):
    """The case's pool as records: c["records"] (a BlockPool), c["pool"] what they stand for."""
    pool, dtype = c["pool"], c["q"].dtype
    L, pages, P, _, Hk, D = pool.shape
    x = pool.float().cpu()
    dead = ~torch.isfinite(x).flatten(4).all(-1)            # places that no request holds
    g = torch.Generator().manual_seed(bits)
    x = torch.where(dead[..., None, None], 0.0, x)
    x = x * torch.exp2(torch.randint(-2, 2, (*x.shape[:-1], D // 32, 1), generator=g).float()).expand(*x.shape[:-1], D // 32, 32).flatten(-2)
    code, scale = ref.quantise(x.flatten(4), bits, dtype)
    half = torch.cat([ref.pack(code, bits), scale], -1)
    half = torch.nn.functional.pad(half, (0, ref.half_bytes(Hk, D, bits) - half.shape[-1]), value=JUNK)
    half[dead] = JUNK
    c["data"] = half.contiguous().to(c["q"].device)
    c["bits"] = bits
    return again(pkg, c)


def again(pkg, c):
    """The case after its records changed."""
    Hk, D = c["pool"].shape[4:]
    c["records"] = pkg.blockscale.BlockPool(c["data"], Hk, D, c["bits"])
    c["pool"] = ref.values(c["data"].cpu(), Hk, D, c["bits"]).to(c["q"].device)
    return c


def run(pkg, c, layer=1, **kw):
    one = all(n == 1 for n in c["new"])
    kw.setdefault("cu_q", None if one else c["cu"])
    return pkg.attention.prefix_attention(c["q"], c["records"], c["table"], c["lens"], c["prefix"], layer=layer, **kw)


def case(pkg, gpu, seed, lens, new, Hq, Hk, D, dtype, bits, P, prefix=0, **kw):
    return blocks(pkg, make(gpu, seed, lens, new, Hq, Hk, D, dtype, dtype, P, prefix, **kw), bits)


BITS = pytest.mark.parametrize("bits", [8, 4])


@pytest.mark.parametrize("D", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "fp16"])
@pytest.mark.parametrize("prefix", [0, 70])
@BITS
def test_decode(pkg, gpu, D, dtype, bits, prefix):
    """One token a request: lengths of one, of whole pages, idle rows."""
    lens = [prefix + n for n in (1, 16, 33, 200, 15, 64, 129)] + [0, 0]
    c = case(pkg, gpu, D, lens, [1] * 9, 8, 2, D, dtype, bits, 16, prefix)
    check(run(pkg, c), reference(c))


@pytest.mark.parametrize("Hq,Hk", [(1, 1), (4, 4), (14, 2), (3, 3), (10, 5), (12, 6), (7, 7), (32, 8), (17, 1), (36, 9), (64, 1), (130, 1)])
@pytest.mark.parametrize("prefix,B", [(0, 3), (160, 3), (300, 30)])
@BITS
def test_heads(pkg, gpu, Hq, Hk, prefix, B, bits):
    """K/V heads of one to three blocks, query heads to one from one to more than a tile's rows."""
    rng = np.random.default_rng(Hq)
    lens = [prefix + int(n) for n in rng.integers(1, 90, B)]
    c = case(pkg, gpu, Hq, lens, [1] * B, Hq, Hk, 64, BF, bits, 16, prefix)
    check(run(pkg, c), reference(c))


@pytest.mark.parametrize("P", [1, 2, 8, 64, 256])
@BITS
def test_page_sizes(pkg, gpu, P, bits):
    for prefix in (0, 77, 256):
        lens = [prefix + n for n in (3, 40, 150, 1, 300)]
        c = case(pkg, gpu, P + prefix, lens, [1, 1, 2, 1, 5], 8, 4, 64, HF, bits, P, prefix)
        check(run(pkg, c, max_q=5), reference(c))


@pytest.mark.parametrize("dtype,D", [(BF, 128), (HF, 64), (HF, 256), (BF, 96), (BF, 192)])
@pytest.mark.parametrize("new,prefix", [
    ([3, 1, 0, 5, 2], 0), ([3, 1, 0, 5, 2], 100), ([1, 130, 64, 0, 17], 0), ([1, 130, 64, 0, 17], 333),
    ([200, 65, 1, 128, 129], 64), ([33], 500), ([1], 2999), ([40, 40, 40], 5),
])
@BITS
def test_extend(pkg, gpu, dtype, D, new, prefix, bits):
    """Several new tokens a request, none at all, more than a tile's rows."""
    rng = np.random.default_rng(len(new) + prefix)
    lens = [prefix + n + int(rng.integers(0, 150)) if n else prefix + 9 for n in new]
    c = case(pkg, gpu, prefix + D, lens, new, 8, 2, D, dtype, bits, 16, prefix)
    check(run(pkg, c, cu_q=c["cu"], max_q=max(new)), reference(c))


@pytest.mark.parametrize("prefix,own", [(0, 90), (40, 300), (500, 30), (500, 0)])
@pytest.mark.parametrize("n", [4, 8, 16, 33, 64])
@BITS
def test_rows_of_a_request(pkg, gpu, n, prefix, own, bits):
    """A request's rows from one stream block's to two tiles', the hints right and wrong."""
    new = [n, 1, n - 3]
    lens = [prefix + own + m for m in new]
    c = case(pkg, gpu, n + prefix, lens, new, 8, 2, 64, BF, bits, 16, prefix)
    want = reference(c)
    for max_len in (None, max(lens), prefix + 1, 1):
        check(run(pkg, c, max_q=n, max_len=max_len), want)
    check(run(pkg, c, max_q=(1 << 31) - 1), want)


@pytest.mark.parametrize("Hk", [1, 2, 8])
@BITS
def test_many_runs(pkg, gpu, Hk, bits):
    """Long requests beside short ones: runs that are full, short, empty, whatever max_len says."""
    lens = [6000, 1, 0, 129, 2047, 3333]
    c = case(pkg, gpu, Hk, lens, [1] * 6, 4 * Hk, Hk, 64, BF, bits, 16, layers=2, qscale=2.0)
    want = reference(c)
    for max_len in (None, 6000, 100, 3000):
        check(run(pkg, c, max_len=max_len), want)
    c = case(pkg, gpu, Hk, [20000], [1], 2 * Hk, Hk, 128, HF, bits, 16)
    check(run(pkg, c), reference(c))


@BITS
def test_pages_outside_the_pool(pkg, gpu, bits):
    """Keys on pages that are not there are left out, whoever sees them."""
    for new, prefix in (([1] * 5, 0), ([1] * 5, 64), ([40] * 5, 64), ([3] * 5, 64)):
        lens = [prefix + n for n in (300, 41, 90, 47, 64)]
        c = case(pkg, gpu, 17, lens, new, 8, 2, 64, BF, bits, 16, prefix)
        shared = prefix // 16
        c["table"][0, shared + 2] = -1
        c["table"][0, shared + 7] = c["pool_pages"]
        c["table"][1, shared:] = 2**31 - 1
        if prefix:
            c["table"][0, 1] = -7                          # of the prefix: for all
        check(run(pkg, c, cu_q=c["cu"], max_q=max(new)), reference(c))
    # no page in the pool: nothing is seen
    c = case(pkg, gpu, 17, [70, 3], [1, 1], 8, 2, 64, BF, bits, 16)
    empty = pkg.blockscale.BlockPool(c["data"][:, :0].contiguous(), 2, 64, bits)
    got = pkg.attention.prefix_attention(c["q"], empty, c["table"], c["lens"], 0, layer=1)
    assert not got.any()


@BITS
def test_longer_than_the_row(pkg, gpu, bits):
    for n in (100, 112):
        c = case(pkg, gpu, 5, [n, 64], [1, 1], 8, 2, 64, BF, bits, 16)
        c["lens"] = torch.tensor([2**31 - 1, 5000], dtype=torch.int32, device=gpu)
        check(run(pkg, c), reference(c))
    c["lens"] = torch.tensor([-5, 64], dtype=torch.int32, device=gpu)
    check(run(pkg, c), reference(c))


@pytest.mark.parametrize("new,prefix,dtype", [([6, 3], 0, BF), ([6, 3], 40, HF), ([150, 70], 0, BF), ([150, 70], 40, HF)])
@BITS
def test_nan_behind_a_query(pkg, gpu, new, prefix, dtype, bits):
    """A block of V that is NaN reaches the queries that see it, in its 32 values, and no other; a key that
    is takes the queries that see it, and no other."""
    lens = [prefix + n + 20 for n in new]
    c = case(pkg, gpu, 8, lens, new, 8, 2, 64, dtype, bits, 16, prefix)
    clean = reference(c)
    b, back = 0, 3                                          # three keys before the end of request 0
    pos = lens[b] - back
    page, place = int(c["table"][b, pos // 16]), pos % 16
    at = 2 * 64 * bits // 8 + 1 * 2 + 1                     # the scale of the second head's second block
    was = c["data"].clone()
    for half in (1, 0):
        c["data"].copy_(was)
        c["data"][1, page, place, half, at] = 255
        got = run(pkg, c, cu_q=c["cu"], max_q=max(new))
        hit = torch.zeros(got.shape, dtype=torch.bool, device=gpu)
        hit[new[0] - back:new[0], 4:8, 32 if half else 0:] = True
        assert torch.isnan(got[hit]).all()
        off = (got.double() - clean[0]).abs()[~hit]
        assert torch.isfinite(got[~hit]).all() and (off <= clean[1][~hit]).all()


@BITS
def test_large_scores_and_a_long_tail(pkg, gpu, bits):
    """Scores of hundreds, and of 2^16 in either sign; a row whose keys are all alike."""
    for qscale in (50.0, 3e4):
        for new in ([1, 1, 1], [40, 2, 30]):
            c = case(pkg, gpu, 9, [n + 300 for n in new], new, 8, 2, 128, BF, bits, 16, qscale=qscale)
            check(run(pkg, c, cu_q=c["cu"], max_q=max(new)), reference(c))
    c = case(pkg, gpu, 10, [4000, 700], [1, 1], 8, 2, 64, HF, bits, 16)
    half = c["data"].shape[-1]
    c["data"][..., 0, :] = 0                                # K: all scores are equal
    c["data"].view(2, -1, 2, half)[:, :, 1] = c["data"].view(2, -1, 2, half)[:, int(c["table"][0, 0]) * 16, 1][:, None]
    again(pkg, c)
    check(run(pkg, c), reference(c))


@BITS
def test_strided_queries_and_max_q(pkg, gpu, bits):
    new, prefix = [5, 2, 9], 40
    lens = [prefix + n + 33 for n in new]
    c = case(pkg, gpu, 21, lens, new, 8, 2, 64, BF, bits, 16, prefix, packed=True)
    want = reference(c)
    assert not c["q"].is_contiguous()
    check(run(pkg, c, max_q=9), want)
    out = torch.full_like(want[0], 7.0, dtype=BF)
    run(pkg, c, max_q=5, out=out)                           # the last request's rows past five stay
    assert (out[12:] == 7.0).all()
    check(out[:12], (want[0][:12], want[1][:12]))
    # rows before the first request and behind the last stay
    c["cu"] = torch.tensor([2, 5, 7, 14], dtype=torch.int32, device=gpu)
    c["lens"] = torch.tensor([40, 45, 60], dtype=torch.int32, device=gpu)
    for max_q in (7, 16):
        out = torch.full_like(want[0], 7.0, dtype=BF)
        run(pkg, c, max_q=max_q, out=out)
        assert (out[:2] == 7.0).all() and (out[14:] == 7.0).all()
        o, tol = reference(c)
        check(out[2:14], (o[2:14], tol[2:14]))


@BITS
def test_in_a_graph(pkg, gpu, bits):
    """Captured on a stream of its own and replayed on new lengths, tables and records."""
    lens, new = [300, 17, 2000, 64], [1] * 4
    c = case(pkg, gpu, 31, lens, new, 16, 4, 128, BF, bits, 16)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run(pkg, c, max_len=2000)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = run(pkg, c, max_len=2000)
    torch.cuda.current_stream().wait_stream(s)
    for seed in (1, 2, 3):
        c["lens"].copy_(torch.tensor([int(x) for x in np.random.default_rng(seed).permutation([300, 17, 1999, 1])][:4]).to(gpu).minimum(
            torch.tensor(lens, device=gpu)))
        c["q"].copy_(torch.randn(c["q"].shape, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        got = out.clone()
        eager = run(pkg, c, max_len=2000)
        assert torch.equal(got, eager)
        check(got, reference(c))


@BITS
def test_same_result_twice(pkg, gpu, bits):
    c = case(pkg, gpu, 41, [5000, 100, 777], [1] * 3, 32, 8, 128, BF, bits, 16)
    first = run(pkg, c)
    for _ in range(3):
        assert torch.equal(run(pkg, c), first)
