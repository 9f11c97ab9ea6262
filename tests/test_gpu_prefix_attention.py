"""Shared-prefix attention over the paged pool against the definition in 64 bits.

Tolerance of a value, with u = eps/2 of the type (half a step), n keys, A = sum
p |v| / sum p, s the largest |q| |k| sum of a score (scaled), x the largest
score in powers of two: a score is a 32-bit sum of dim products, off by at most
dim * 2^-24 * s, and its power's argument by 2^-23 * x more; each p is rounded to
the type (u) and its power is off by 2^-23; the sums of n terms, of p and of p v,
are off by at most n * 2^-24 of A each; the result is rounded once (u):
  u |o| + A (u + 2 (dim 2^-24 s + 2^-23 x + 2^-23 + n 2^-24))
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, HF, F8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def make(gpu, seed, lens, new, Hq, Hk, D, dtype, pool_dtype, P, prefix=0, width=None, junk=True, layers=2, qscale=1.0,
         packed=False):
    """Requests of `lens` keys of which the last `new` are queried; pages of the
    pool that no request holds, and places behind a request's last token, are NaN."""
    g = torch.Generator(device="cpu").manual_seed(seed)
    B = len(lens)
    need = [-(-n // P) for n in lens]
    shared = prefix // P
    width = width or max([1] + need)
    total = sum(max(n - shared, 0) for n in need) + shared + 4
    ids = (torch.randperm(total, generator=g) + 1).tolist()
    pool = torch.randn(layers, total + 1, P, 2, Hk, D, generator=g)
    if pool_dtype == F8:
        pool = pool * 40
    pool = pool.to(pool_dtype)
    table = torch.full((B, width), -1, dtype=torch.int32)
    front = [ids.pop() for _ in range(shared)]
    used = torch.zeros(total + 1, P, dtype=torch.bool)
    for b, n in enumerate(lens):
        for j in range(need[b]):
            table[b, j] = front[j] if j < shared else ids.pop()
            used[table[b, j], : max(0, min(P, n - j * P))] = True
    if prefix % P:                                    # each request's own copy of the page it ends in
        raw = pool.view(torch.uint8)
        rows = [b for b, n in enumerate(lens) if n > shared * P]
        for b in rows[1:]:
            raw[:, table[b, shared], : prefix % P] = raw[:, table[rows[0], shared], : prefix % P]
    if junk:
        pool.view(torch.uint8)[:, ~used] = 0x7F if pool_dtype == F8 else 0xFF       # NaN in every type
    N = sum(new)
    q = (torch.randn(N, Hq + 3, D, generator=g) * qscale).to(dtype)
    cu = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32)
    c = dict(pool=pool.to(gpu), table=table.to(gpu), lens=torch.tensor(lens, dtype=torch.int32).to(gpu), cu=cu.to(gpu),
             q=q.to(gpu)[:, 1:Hq + 1] if packed else q[:, :Hq].contiguous().to(gpu), prefix=prefix, new=new,
             pool_pages=total + 1, P=P)
    return c


def reference(c, layer=1, scale=None, ks=1.0, vs=1.0, prefix_pages=None):
    """(o, tolerance) in 64 bits, one request at a time."""
    q, pool = c["q"].double(), c["pool"][layer]
    N, Hq, D = q.shape
    P, Hk = pool.shape[1], pool.shape[3]
    G = Hq // Hk
    scale = D ** -0.5 if scale is None else scale
    flat = pool.reshape(-1, 2, Hk, D)
    table, cu, lens = c["table"].cpu().numpy(), c["cu"].tolist(), c["lens"].tolist()
    front = table[0] if prefix_pages is None else prefix_pages.cpu().numpy()
    u = torch.finfo(c["q"].dtype).eps / 2
    o = torch.zeros(N, Hq, D, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(o)
    for b in range(len(lens)):
        n_q = cu[b + 1] - cu[b]
        keys, pos = [], []
        for j in range(min(lens[b], table.shape[1] * P)):
            page = (front if j < c["prefix"] else table[b])[j // P]
            if 0 <= page < pool.shape[0]:
                keys.append(page * P + j % P)
                pos.append(j)
        if n_q == 0 or not keys:
            continue
        kv = flat[torch.tensor(keys, device=q.device)].double()
        pos = torch.tensor(pos, device=q.device)
        see = pos[None] <= lens[b] - n_q + torch.arange(n_q, device=q.device)[:, None]
        for h in range(Hk):
            K, V = kv[:, 0, h] * ks, kv[:, 1, h] * vs
            for x in range(h * G, (h + 1) * G):
                qq = q[cu[b]:cu[b + 1], x]
                s = (qq @ K.t()) * scale
                big = ((qq.abs() @ K.abs().t()) * scale).masked_fill(~see, 0).amax(1, keepdim=True)
                s = s.masked_fill(~see, -math.inf)
                m = s.amax(1, keepdim=True)
                some = see.any(1, keepdim=True)
                p = torch.where(see, torch.exp(s - torch.where(some, m, 0.0)), 0.0)
                l = p.sum(1, keepdim=True)
                y = torch.where(some, (p @ V) / l, 0.0)
                A = torch.where(some, (p @ V.abs()) / l, 0.0)
                peak = torch.where(see, s.abs(), 0.0).amax(1, keepdim=True) * 1.4427
                err = 2 * (D * 2.0 ** -24 * big + 2.0 ** -23 * (peak + 1) + len(keys) * 2.0 ** -24)
                o[cu[b]:cu[b + 1], x] = y
                tol[cu[b]:cu[b + 1], x] = (u * y.abs() + A * (u + err)) * (1 + 2.0 ** -7) + 2.0 ** -25
    return o, tol


def run(pkg, c, layer=1, **kw):
    one = all(n == 1 for n in c["new"])
    kw.setdefault("cu_q", None if one else c["cu"])
    return pkg.attention.prefix_attention(c["q"], c["pool"], c["table"], c["lens"], c["prefix"], layer=layer, **kw)


def check(got, ref, rows=None):
    o, tol = ref
    rows = o.shape[0] if rows is None else rows
    off = (got.double() - o).abs()[:rows]
    # finite just where the definition is
    assert torch.equal(torch.isfinite(got[:rows]), torch.isfinite(o[:rows])), "not finite"
    bad = off > tol[:rows]
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} values off, worst "
                           f"{float((off / tol[:rows]).max()):.3g} of the tolerance; first at {bad.nonzero()[0].tolist()}")


@pytest.mark.parametrize("D", [64, 80, 96, 128, 256, 8, 40, 200])
@pytest.mark.parametrize("dtype,pool", [(BF, BF), (HF, HF), (BF, F8), (HF, F8)])
@pytest.mark.parametrize("prefix", [0, 70])
def test_decode(pkg, gpu, D, dtype, pool, prefix):
    """One token a request: lengths of one, of whole pages, idle rows."""
    if pool == F8 and D % 16:
        D = 16 if D < 16 else D // 16 * 16
    lens = [prefix + n for n in (1, 16, 33, 200, 15, 64, 129)] + [0, 0]
    c = make(gpu, D, lens, [1] * 9, 8, 2, D, dtype, pool, 16, prefix)
    kw = dict(ks=0.03, vs=0.02) if pool == F8 else {}
    sc = {"k_scale": torch.tensor([0.03], device=gpu), "v_scale": torch.tensor([0.02], device=gpu)} if pool == F8 else {}
    check(run(pkg, c, **sc), reference(c, **kw))


@pytest.mark.parametrize("Hq,Hk", [(1, 1), (4, 4), (14, 2), (32, 4), (17, 1), (71, 1), (128, 1), (130, 1)])
@pytest.mark.parametrize("prefix,B", [(0, 3), (160, 3), (600, 40)])
def test_head_groups(pkg, gpu, Hq, Hk, prefix, B):
    """Query heads to a K/V head from one to more than a tile's rows."""
    rng = np.random.default_rng(Hq)
    lens = [prefix + int(n) for n in rng.integers(1, 90, B)]
    c = make(gpu, Hq, lens, [1] * B, Hq, Hk, 64, BF, BF, 16, prefix)
    check(run(pkg, c), reference(c))


@pytest.mark.parametrize("P", [1, 2, 8, 64, 256])
def test_page_sizes(pkg, gpu, P):
    for prefix in (0, 77, 256):
        lens = [prefix + n for n in (3, 40, 150, 1, 300)]
        c = make(gpu, P + prefix, lens, [1, 1, 2, 1, 5], 8, 4, 64, HF, HF, P, prefix)
        check(run(pkg, c, max_q=5), reference(c))


@pytest.mark.parametrize("dtype,pool,D", [(BF, BF, 128), (HF, HF, 80), (BF, F8, 64), (HF, F8, 256), (BF, BF, 96)])
@pytest.mark.parametrize("new,prefix", [
    ([3, 1, 0, 5, 2], 0), ([3, 1, 0, 5, 2], 100), ([1, 130, 64, 0, 17], 0), ([1, 130, 64, 0, 17], 333),
    ([200, 65, 1, 128, 129], 64), ([33], 500), ([1], 2999), ([40, 40, 40], 5),
])
def test_extend(pkg, gpu, dtype, pool, D, new, prefix):
    """Several new tokens a request, none at all, more than a tile's rows."""
    rng = np.random.default_rng(len(new) + prefix)
    lens = [prefix + n + int(rng.integers(0, 150)) if n else prefix + 9 for n in new]
    c = make(gpu, prefix + D, lens, new, 8, 2, D, dtype, pool, 16, prefix)
    kw = dict(ks=0.03, vs=0.02) if pool == F8 else {}
    sc = {"k_scale": torch.tensor([0.03], device=gpu), "v_scale": torch.tensor([0.02], device=gpu)} if pool == F8 else {}
    check(run(pkg, c, cu_q=c["cu"], max_q=max(new), **sc), reference(c, **kw))


@pytest.mark.parametrize("prefix,own", [(0, 90), (40, 300), (500, 30), (500, 0)])
@pytest.mark.parametrize("n", [4, 8, 12, 16, 24, 32, 33, 64])
def test_rows_of_a_request(pkg, gpu, n, prefix, own):
    """A request's rows from one stream block's to two tiles', with much or little
    of its keys in the prefix: either kind of block, chosen by max_len too."""
    new = [n, 1, n - 3]
    lens = [prefix + own + m for m in new]
    c = make(gpu, n + prefix, lens, new, 8, 2, 64, BF, BF, 16, prefix)
    ref = reference(c)
    for max_len in (None, max(lens), prefix + 1):
        check(run(pkg, c, max_q=n, max_len=max_len), ref)
    check(run(pkg, c, max_q=(1 << 31) - 1), ref)


def test_queries_inside_the_prefix(pkg, gpu):
    """A request may end inside the prefix, and have more tokens than keys: its
    queries see what lies before them, the first ones nothing."""
    for new in ([5, 9, 30, 2], [150, 9, 300, 2]):
        lens = [40, 5, 130, 201]
        c = make(gpu, sum(new), lens, new, 8, 2, 64, BF, BF, 16, 0)
        c["prefix"] = 200
        c["table"][:3] = c["table"][3]                     # all on the longest one's pages
        check(run(pkg, c, cu_q=c["cu"], max_q=max(new)), reference(c))


def test_prefix_pages(pkg, gpu):
    """The prefix from a list of its own; the rows' first entries are not read."""
    lens = [90 + n for n in (4, 30, 1, 60)]
    for new in ([1] * 4, [4, 20, 1, 50], [4, 30, 1, 60]):
        c = make(gpu, 3, lens, new, 16, 2, 64, BF, BF, 16, 90)
        front = c["table"][0, :6].clone()
        c["table"][:, :5] = -1
        for kw in ({}, {"max_q": 60}):
            got = run(pkg, c, cu_q=c["cu"], prefix_pages=front, **kw)
            check(got, reference(c, prefix_pages=front))


def test_pages_outside_the_pool(pkg, gpu):
    """Keys on pages that are not there are left out, whoever sees them."""
    for new, prefix in (([1] * 5, 0), ([1] * 5, 64), ([40] * 5, 64), ([3] * 5, 64)):
        lens = [prefix + n for n in (300, 41, 90, 47, 64)]
        c = make(gpu, 17, lens, new, 8, 2, 64, BF, BF, 16, prefix)
        shared = prefix // 16
        c["table"][0, shared + 2] = -1
        c["table"][0, shared + 7] = c["pool_pages"]
        c["table"][1, shared:] = 2**31 - 1
        if prefix:
            c["table"][0, 1] = -7                          # of the prefix: for all
        check(run(pkg, c, cu_q=c["cu"], max_q=max(new)), reference(c))


def test_longer_than_the_row(pkg, gpu):
    """Lengths past what a table row can hold: the keys that it holds."""
    c = make(gpu, 5, [100, 64], [1, 1], 8, 2, 64, BF, BF, 16, 0)
    c["lens"] = torch.tensor([2**31 - 1, 5000], dtype=torch.int32, device=gpu)
    check(run(pkg, c), reference(c))                       # the first one's last page holds NaN behind its tokens
    c = make(gpu, 5, [112, 64], [1, 1], 8, 2, 64, BF, BF, 16, 0)
    c["lens"] = torch.tensor([2**31 - 1, 5000], dtype=torch.int32, device=gpu)
    check(run(pkg, c), reference(c))
    c["lens"] = torch.tensor([-5, 64], dtype=torch.int32, device=gpu)
    check(run(pkg, c), reference(c))


@pytest.mark.parametrize("kind", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("new,prefix,pool", [([6, 3], 0, BF), ([6, 3], 40, HF), ([150, 70], 0, BF), ([150, 70], 40, F8),
                                             ([5, 2], 0, F8)])
def test_not_finite_behind_a_query(pkg, gpu, kind, new, prefix, pool):
    """A value that is not finite reaches the queries that see it, and no other."""
    dtype = HF if pool == HF else BF
    if pool == F8 and math.isinf(kind):
        pytest.skip("e4m3 has no infinity")
    lens = [prefix + n + 20 for n in new]
    c = make(gpu, 8, lens, new, 8, 2, 64, dtype, pool, 16, prefix)
    clean = reference(c)
    P, b, back = 16, 0, 3                                   # three keys before the end of request 0
    pos = lens[b] - back
    page, place = int(c["table"][b, pos // P]), pos % P
    c["pool"].view(torch.uint8 if pool == F8 else torch.int16)[1, page, place, 1, 1, 5] = \
        torch.tensor([kind], dtype=torch.float32).to(pool).view(torch.uint8 if pool == F8 else torch.int16)[0].to(gpu)
    got = run(pkg, c, cu_q=c["cu"], max_q=max(new))
    hit = torch.zeros(got.shape, dtype=torch.bool, device=gpu)
    hit[new[0] - back:new[0], 4:8, 5] = True                # the last three queries, the second K/V head's group
    assert not torch.isfinite(got[hit]).any()
    off = (got.double() - clean[0]).abs()[~hit]
    assert torch.isfinite(got[~hit]).all() and (off <= clean[1][~hit]).all()


def test_not_finite_keys_and_queries(pkg, gpu):
    """A key that is not finite behind some queries, and a query that is not:
    the others keep their results."""
    for new in ([6, 3], [150, 70]):
        lens = [n + 20 for n in new]
        c = make(gpu, 9, lens, new, 8, 2, 64, BF, BF, 16, 0)
        clean = reference(c)
        pos = lens[0] - 2
        c["pool"][1, int(c["table"][0, pos // 16]), pos % 16, 0, 0, 3] = float("nan")
        c["q"][new[0] + 1, 5, 0] = float("inf")
        got = run(pkg, c, cu_q=c["cu"], max_q=max(new))
        hit = torch.zeros(got.shape[:2], dtype=torch.bool, device=gpu)
        hit[new[0] - 2:new[0], :4] = True
        hit[new[0] + 1, 5] = True
        assert torch.isnan(got[hit]).all()
        off = (got.double() - clean[0]).abs()[~hit]
        assert torch.isfinite(got[~hit]).all() and (off <= clean[1][~hit]).all()


def test_padded_rows_stay(pkg, gpu):
    for new in ([2, 1, 3], [100, 30, 3]):
        lens = [n + 50 for n in new]
        c = make(gpu, 4, lens, new + [], 8, 2, 64, BF, BF, 16, 32)
        n = sum(new)
        q = torch.full((n + 70, 8, 64), float("nan"), dtype=BF, device=gpu)
        q[:n] = c["q"]
        out = torch.full_like(q, 3.0)
        ref = reference(c)
        got = pkg.attention.prefix_attention(q, c["pool"], c["table"], c["lens"], 32, layer=1, cu_q=c["cu"], out=out,
                                             max_q=max(new))
        assert got is out
        check(got[:n], ref)
        assert (got[n:] == 3.0).all()


@pytest.mark.parametrize("prefix", [0, 32, 600])
@pytest.mark.parametrize("new", [[2, 1, 3], [100, 30, 3]])
def test_rows_before_the_first_request_stay(pkg, gpu, new, prefix):
    """Whether results are joined from parts or written at once."""
    c = make(gpu, 7, [n + prefix + 400 for n in new], new, 8, 2, 64, BF, BF, 16, prefix)
    ref, n, gap = reference(c), sum(new), 5
    q = torch.full((n + 2 * gap, 8, 64), float("nan"), dtype=BF, device=gpu)
    q[gap:gap + n] = c["q"]
    out = torch.full_like(q, 3.0)
    pkg.attention.prefix_attention(q, c["pool"], c["table"], c["lens"], prefix, layer=1, cu_q=c["cu"] + gap, out=out,
                                   max_q=max(new))
    check(out[gap:gap + n], ref)
    assert (out[:gap] == 3.0).all() and (out[gap + n:] == 3.0).all()


@pytest.mark.parametrize("prefix", [0, 2100])
def test_long_and_split(pkg, gpu, prefix):
    """Keys enough that blocks share them out; wrong hints change no result."""
    lens = [prefix + n for n in (5000, 1, 800, 2600)]
    c = make(gpu, 6, lens, [1] * 4, 8, 2, 128, BF, BF, 16, prefix, qscale=3.0)
    ref = reference(c)
    for kw in ({}, {"max_len": max(lens)}, {"max_len": 10}, {"max_q": 7, "cu_q": c["cu"]},
               {"max_q": 300, "cu_q": c["cu"]}):
        check(run(pkg, c, **kw), ref)


def test_scales(pkg, gpu):
    c = make(gpu, 2, [40, 300], [1, 1], 8, 2, 64, HF, HF, 16, 0, qscale=4.0)
    for scale in (1.0, 0.0, 0.01, 2.5):
        check(run(pkg, c, scale=scale), reference(c, scale=scale))


def test_negative_scale_of_keys(pkg, gpu):
    c = make(gpu, 2, [40, 300, 90], [1, 1, 1], 8, 2, 64, BF, F8, 16, 0)
    for ks, vs in ((-0.03, 0.02), (0.03, -0.5), (0.0, 1.0)):
        got = run(pkg, c, k_scale=torch.tensor([ks], device=gpu), v_scale=torch.tensor([vs], device=gpu))
        check(got, reference(c, ks=ks, vs=vs))


def test_peaked_scores(pkg, gpu):
    """Maxima that keep rising along the keys, and large scores."""
    c = make(gpu, 12, [700, 650], [4, 150], 8, 2, 64, BF, BF, 16, 0, qscale=8.0)
    ramp = torch.linspace(0.01, 4, c["pool"].shape[1], device=gpu)
    c["pool"][:, c["table"][0, :43].long()] *= ramp[: 43][None, :, None, None, None, None].to(BF)
    check(run(pkg, c, cu_q=c["cu"], max_q=150), reference(c))


def test_packed_and_unaligned_queries(pkg, gpu):
    lens, new = [90, 30, 200], [3, 1, 40]
    c = make(gpu, 13, lens, new, 8, 2, 64, BF, BF, 16, 16, packed=True)
    want = reference(c)
    check(run(pkg, c, cu_q=c["cu"]), want)
    flat = torch.zeros(c["q"].numel() + 3, dtype=BF, device=gpu)
    odd = flat[3:].view(c["q"].shape)
    odd.copy_(c["q"])
    c["q"] = odd
    check(run(pkg, c, cu_q=c["cu"]), want)
    out = torch.empty(c["q"].numel() + 1, dtype=BF, device=gpu)[1:].view(c["q"].shape)
    check(run(pkg, c, cu_q=c["cu"], out=out), want)


def test_same_bits_again(pkg, gpu):
    rng = np.random.default_rng(0)
    lens = [1000 + int(n) for n in rng.integers(1, 900, 20)]
    c = make(gpu, 14, lens, [1] * 20, 32, 8, 128, BF, BF, 16, 1000)
    first = run(pkg, c)
    for _ in range(5):
        assert torch.equal(run(pkg, c), first)


def test_shared_is_what_each_would_get(pkg, gpu):
    """The prefix computed once for all, against each request on its own."""
    lens = [520 + n for n in (1, 30, 200, 77)]
    c = make(gpu, 15, lens, [1] * 4, 32, 8, 128, BF, BF, 16, 520)
    ref = reference(c)
    check(run(pkg, c), ref)
    c["prefix"] = 0
    check(run(pkg, c), ref)


def test_captured(pkg, gpu):
    """Replays on other queries and lengths, with eager calls between them."""
    B, prefix = 12, 300
    c = make(gpu, 16, [prefix + 400] * B, [1] * B, 16, 4, 128, BF, BF, 16, prefix, junk=False)
    run(pkg, c)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(pkg, c)
    rng = np.random.default_rng(1)
    for i in range(4):
        c["q"].copy_(torch.randn(c["q"].shape, device=gpu))
        c["lens"].copy_(torch.tensor([prefix + int(n) for n in rng.integers(1, 400, B)], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        check(got, reference(c))
        assert torch.equal(run(pkg, c), got)


def test_two_streams_at_once(pkg, gpu):
    """Each call has a workspace of its own."""
    cs = [make(gpu, 20 + i, [400 + 100 * i + n for n in (5, 900, 77)], [1] * 3, 16, 4, 128, BF, BF, 16, 400) for i in range(2)]
    refs = [reference(c) for c in cs]
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in cs]
    outs = [None, None]
    for _ in range(4):
        for i, c in enumerate(cs):
            with torch.cuda.stream(side[i]):
                outs[i] = run(pkg, c)
    torch.cuda.synchronize()
    for o, r in zip(outs, refs):
        check(o, r)


def test_offsets_past_32_bits(pkg, gpu):
    """A layer of more than 4 GiB, the second of two: pages at its far end."""
    Hk, D, P = 8, 128, 16
    pages = (4608 << 20) // (P * 2 * Hk * D * 2)
    pool = torch.zeros(2, pages, P, 2, Hk, D, dtype=BF, device=gpu)
    ids = torch.tensor([pages - 1, 0, pages // 2, pages - 7, 3], dtype=torch.int32, device=gpu)
    pool[1, ids.long()] = torch.randn(5, P, 2, Hk, D, device=gpu).to(BF)
    for n, new in ((75, 1), (75, 40)):
        c = dict(pool=pool, table=ids[None].contiguous(), lens=torch.tensor([n], dtype=torch.int32, device=gpu), P=P,
                 cu=torch.tensor([0, new], dtype=torch.int32, device=gpu), prefix=0, new=[new], pool_pages=pages,
                 q=torch.randn(new, 32, D, device=gpu).to(BF))
        check(run(pkg, c, cu_q=c["cu"]), reference(c))
        c["prefix"] = 50
        check(run(pkg, c, cu_q=c["cu"]), reference(c))


def test_no_tokens(pkg, gpu):
    c = make(gpu, 1, [20, 30], [0, 0], 8, 2, 64, BF, BF, 16, 0)
    assert run(pkg, c, cu_q=c["cu"]).shape == (0, 8, 64)
