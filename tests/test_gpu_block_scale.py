"""A cache with block scales: written and read back, bit for bit.

Values are quantised by definition: V as given, K from the formulas in 64 bits rounded
to 32.  The kernel's K differs from these by some 2^-50 of the largest of the pair, so
its 32 bits, and its code, could only differ where the formula lies that near to the
middle of two 32-bit numbers and these to the middle of two codes; no code may differ
here.  Queries are as in norm + rotation: half a step and 2^-18 of the row's largest.
"""
import pytest
import torch

import blockref as ref
from test_gpu_norm_rotate import near, rotate64

pytestmark = pytest.mark.gpu

BF, HF, FF = torch.bfloat16, torch.float16, torch.float32


def case(seed, N, Hq, Hk, D, rot, dtype, bits, axes=1, interleaved=False, norm=True, weights=True, P=16, skew=0, spread=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(N, (Hq + 2 * Hk) * D + skew, generator=g)
    if spread:                                          # heads of very different size
        x = x * torch.exp2(torch.randint(-spread, spread + 1, (N, 1), generator=g).float())
    pages = -(-N // P) + 3
    data = torch.randint(0, 256, (2, pages, P, 2, ref.half_bytes(Hk, D, bits)), generator=g, dtype=torch.uint8)
    slots = torch.randperm(pages * P, generator=g)[:N].to(torch.int32)
    if N > 2:
        slots[N // 2] = -1
        slots[N - 1] = pages * P                        # past the pool
    pos = torch.randint(-3, 1 << 20, (axes, N) if axes > 1 else (N,), generator=g, dtype=torch.int32)
    half = rot // 2
    freqs = 10000.0 ** (-torch.arange(half, dtype=torch.float64) / max(half, 1))
    axis_of = torch.randint(0, axes, (half,), generator=g).to(torch.uint8) if axes > 1 else None
    w = lambda: (1 + 0.2 * torch.randn(D, generator=g)).to(dtype) if weights and norm else None  # noqa: E731
    return dict(x=x.to(dtype), data=data, slots=slots, pos=pos, freqs=freqs, axis_of=axis_of, wq=w(), wk=w(), N=N, Hq=Hq,
                Hk=Hk, D=D, interleaved=interleaved, norm=norm, skew=skew, dtype=dtype, bits=bits)


def split(c, x):
    N, Hq, Hk, D = c["N"], c["Hq"], c["Hk"], c["D"]
    x = x[:, c["skew"]:]
    return (x[:, :Hq * D].unflatten(1, (Hq, D)), x[:, Hq * D:(Hq + Hk) * D].unflatten(1, (Hk, D)),
            x[:, (Hq + Hk) * D:].unflatten(1, (Hk, D)))


def go(pkg, gpu, c, layer=1, factor=1.0, tokens=None, in_place=False):
    up = lambda t: None if t is None else t.to(gpu)  # noqa: E731
    x, data = up(c["x"]), up(c["data"])
    q, k, v = split(c, x)
    pool = pkg.blockscale.BlockPool(data, c["Hk"], c["D"], c["bits"])
    got = pkg.attention.norm_rotate_write(
        q, k, v, up(c["pos"]), up(c["freqs"]) if c["freqs"].numel() else None, pool, up(c["slots"]), layer=layer,
        norm=c["norm"], q_weight=up(c["wq"]), k_weight=up(c["wk"]), axis_of=up(c["axis_of"]),
        interleaved=c["interleaved"], factor=factor,
        tokens=None if tokens is None else torch.tensor([tokens], dtype=torch.int32, device=gpu),
        out=q if in_place else None)
    return got.cpu(), data.cpu()


def check(c, got, data, layer=1, factor=1.0, tokens=None):
    N = c["N"] if tokens is None else min(max(tokens, 0), c["N"])
    q, k, v = split(c, c["x"])
    rot = lambda t, w: rotate64(t, c["pos"], c["freqs"], c["axis_of"], c["interleaved"], factor, w, 1e-6, c["norm"])  # noqa: E731
    if N:
        want, scale = rot(q, c["wq"])
        near(got[:N], want[:N], scale[:N], c["dtype"], "q")
    heads, D, bits = c["Hk"], c["D"], c["bits"]
    keys = rot(k, c["wk"])[0].float()
    flat, was = data.view(2, -1, 2, data.shape[-1]), c["data"].view(2, -1, 2, data.shape[-1])
    code = heads * D * bits // 8
    end = code + heads * D // 32
    want = was.clone()
    for t in range(N):
        s = int(c["slots"][t])
        if not 0 <= s < flat.shape[1]:
            continue
        for i, y in enumerate((keys[t], v[t].float())):
            cd, sc = ref.quantise(y.reshape(-1), bits, c["dtype"])
            dead = (sc == 255).repeat_interleave(32)
            here = ref.unpack(flat[layer, s, i], heads, D, bits)[0].reshape(-1)
            cd = torch.where(dead, here, cd)              # the codes of a block of NaN are no matter
            want[layer, s, i, :code] = ref.pack(cd, bits)
            want[layer, s, i, code:end] = sc
    bad = (flat != want).nonzero()
    assert not len(bad), f"{len(bad)} bytes differ, the first at {bad[0].tolist()}: " \
                         f"{int(flat[tuple(bad[0])])} for {int(want[tuple(bad[0])])}; codes end at {code}"


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [BF, HF, FF], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("Hq,Hk,D,rot,inter", [(8, 2, 128, 128, False), (7, 1, 64, 32, True), (4, 4, 96, 96, False),
                                               (3, 3, 256, 128, False), (2, 1, 32, 32, True), (10, 5, 192, 0, False),
                                               (6, 2, 160, 48, False)])
def test_write(pkg, gpu, bits, dtype, Hq, Hk, D, rot, inter):
    c = case(Hq * D + bits, 37, Hq, Hk, D, rot, dtype, bits, interleaved=inter)
    check(c, *go(pkg, gpu, c))


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [BF, HF, FF], ids=["bf16", "fp16", "fp32"])
def test_write_one_value_a_lane(pkg, gpu, bits, dtype):
    """Rows that start off 16 bytes, and pairs that lie in no whole chunks."""
    for D, rot, skew, inter in ((128, 128, 3, False), (256, 256, 1, True), (96, 20, 0, False), (32, 6, 5, True), (224, 224, 1, False)):
        c = case(D + skew, 9, 3, 2, D, rot, dtype, bits, skew=skew, interleaved=inter)
        check(c, *go(pkg, gpu, c))


@pytest.mark.parametrize("bits", [8, 4])
def test_write_many_tokens(pkg, gpu, bits):
    """Waves of four query rows a group."""
    for dtype, Hq, Hk, D in ((BF, 8, 2, 128), (HF, 5, 1, 64), (FF, 12, 4, 96)):
        c = case(bits, 40, Hq, Hk, D, D, dtype, bits)
        # the checked tokens among many that have no slot and are compared as queries only
        n = 24 * 4096
        g = torch.Generator().manual_seed(5)
        x = torch.randn(n, c["x"].shape[1], generator=g).to(dtype)
        at = torch.randperm(n, generator=g)[:40].sort().values
        x[at] = c["x"]
        slots = torch.full((n,), -1, dtype=torch.int32)
        slots[at] = c["slots"]
        pos = torch.zeros(n, dtype=torch.int32)
        pos[at] = c["pos"]
        big = dict(c, x=x, slots=slots, pos=pos, N=n)
        got, data = go(pkg, gpu, big)
        check(c, got[at], data)
        others = torch.ones(n, dtype=torch.bool)
        others[at] = False
        q = split(big, x)[0][others][:2000]
        want, scale = rotate64(q, torch.zeros(2000), c["freqs"], None, False, 1.0, c["wq"], 1e-6, True)
        near(got[others][:2000], want, scale, dtype, "q")


@pytest.mark.parametrize("bits", [8, 4])
def test_write_forms(pkg, gpu, bits):
    for kw in (dict(axes=3), dict(norm=False), dict(weights=False), dict(norm=False, rot=0), dict(spread=12)):
        kw = {"rot": 64, **kw}
        c = case(11, 21, 4, 2, 128, dtype=BF, bits=bits, **kw)
        check(c, *go(pkg, gpu, c, layer=0, factor=1.25), layer=0, factor=1.25)
    c = case(12, 21, 4, 2, 128, 128, HF, bits)
    for n in (0, 1, 13, 21, 99, -4):
        check(c, *go(pkg, gpu, c, tokens=n), tokens=n)
    got, data = go(pkg, gpu, c, in_place=True)
    check(c, got, data)
    for N in (1, 2):
        c = case(13, N, 32, 8, 128, 128, BF, bits)
        check(c, *go(pkg, gpu, c))


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [BF, HF, FF], ids=["bf16", "fp16", "fp32"])
def test_write_edge_values(pkg, gpu, bits, dtype):
    """Blocks of zeros, of both zeros, at the type's ends, on midpoints and on the largest
    code, with infinities and NaN."""
    Hk, D, N = 2, 128, 16
    c = case(3, N, 1, Hk, D, 0, dtype, bits, norm=False)
    c["slots"] = torch.arange(N, dtype=torch.int32)
    fi = torch.finfo(dtype)
    g = torch.Generator().manual_seed(1)
    k, v = split(c, c["x"])[1:]
    for x in (k, v):
        x[0] = 0
        x[1] = torch.where(torch.rand(Hk, D, generator=g) < 0.5, -0.0, 0.0)
        x[2] = fi.max
        x[3] = -fi.max * torch.rand(Hk, D, generator=g)
        x[4] = fi.tiny * torch.rand(Hk, D, generator=g)                    # subnormal
        x[5] = fi.smallest_normal
        x[6, :, ::5] = 1e-7
        table = ref.E4M3[:127] if bits == 8 else ref.E2M1
        mid = torch.cat([table, (table[1:] + table[:-1]) / 2])
        n = mid.numel()
        for row, f in ((7, 1.0), (8, 2.0 ** -9), (9, -4.0)):
            pick = mid[torch.randint(0, n, (Hk * D,), generator=g)]
            pick[::32] = table[-1]                                         # each block's largest: the largest code
            x[row] = (pick * f).view(Hk, D).to(dtype)
        x[10] = (mid[torch.arange(Hk * D) % n] * 1.0).view(Hk, D).to(dtype)
        x[11, 0, 40] = float("inf")
        x[11, 1, 7] = -float("inf")
        x[12, 0, 100] = float("nan")
        x[13, 0, :32] = float("inf")
        x[14, :, 1] = fi.max
        x[15, :, 64] = table[-1] * 1.0000001 if dtype == FF else table[-1] * (1 + fi.eps)
    got, data = go(pkg, gpu, c)
    check(c, got, data)


@pytest.mark.parametrize("bits", [8, 4])
def test_same_bytes_in_any_launch(pkg, gpu, bits):
    """A token's bytes do not depend on what is written beside it, nor on how its row lies."""
    c = case(21, 64, 8, 4, 128, 128, BF, bits)
    c["slots"] = torch.arange(64, dtype=torch.int32)
    whole = go(pkg, gpu, c)[1].view(2, -1, 2, c["data"].shape[-1])[1, :64]
    for t in (0, 5, 63):
        one = dict(c, x=c["x"][t:t + 1], slots=c["slots"][:1], pos=c["pos"][t:t + 1], N=1)
        assert torch.equal(go(pkg, gpu, one)[1].view(2, -1, 2, c["data"].shape[-1])[1, 0], whole[t])
        skew = torch.nn.functional.pad(one["x"], (1, 0))
        assert torch.equal(go(pkg, gpu, dict(one, x=skew, skew=1))[1].view(2, -1, 2, c["data"].shape[-1])[1, 0], whole[t])


# ------------------------------------------------------------------ reading back
def expect(half, heads, D, bits, dtype):
    return ref.values(half, heads, D, bits).to(dtype)


def same(got, want, dtype):
    """Equal; numbers under the smallest normal one of 32 bits may be 0."""
    g, w = got.double(), want.double()
    ok = (g == w) | (torch.isnan(g) & torch.isnan(w))
    if dtype != HF:
        ok |= (g == 0) & (w.abs() < 2.0 ** -126)
    assert ok.all(), f"{int((~ok).sum())} values differ: {g[~ok][:4].tolist()} for {w[~ok][:4].tolist()}"


@pytest.mark.parametrize("dtype", [BF, HF, FF], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("bits", [8, 4])
def test_read_every_code_and_scale(pkg, gpu, bits, dtype):
    heads, D = 1, 32
    half = ref.half_bytes(heads, D, bits)
    codes = torch.arange(256).to(torch.uint8).view(-1, 32 * bits // 8)      # bytes: pairs of e2m1
    n = codes.shape[0]
    data = torch.zeros(1, 256 * n, 1, 2, half, dtype=torch.uint8)
    data[0, :, 0, :, :codes.shape[1]] = codes.repeat(256, 1)[:, None]
    data[0, :, 0, :, codes.shape[1]] = torch.arange(256).repeat_interleave(n).to(torch.uint8)[:, None]
    pool = pkg.blockscale.BlockPool(data.to(gpu), heads, D, bits)
    slots = torch.arange(256 * n, dtype=torch.int32)
    k, v = pkg.blockscale.read(pool, slots.to(gpu), dtype)
    want = expect(data[0, :, 0, 0], heads, D, bits, dtype)
    same(k.cpu(), want, dtype)
    assert torch.equal(k.nan_to_num(7.0), v.nan_to_num(7.0))


@pytest.mark.parametrize("dtype", [BF, HF, FF], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("bits,heads,D,P,N", [(8, 8, 128, 16, 300), (4, 8, 128, 16, 1), (4, 3, 96, 8, 77), (8, 1, 32, 1, 5),
                                              (8, 5, 64, 4, 1023), (4, 2, 256, 64, 130), (4, 1, 32, 2, 3), (8, 7, 160, 16, 33)])
def test_read(pkg, gpu, bits, heads, D, P, N, dtype):
    g = torch.Generator().manual_seed(N)
    pages = -(-N // P) + 2
    data = torch.randint(0, 256, (3, pages, P, 2, ref.half_bytes(heads, D, bits)), generator=g, dtype=torch.uint8)
    c = heads * D * bits // 8
    data[..., c:c + heads * D // 32] = torch.randint(110, 140, data[..., c:c + heads * D // 32].shape, generator=g).to(torch.uint8)
    slots = torch.randint(-2, pages * P + 2, (N,), generator=g).to(torch.int32)    # some twice, some out of the pool
    slots[:1] = pages * P - 1
    pool = pkg.blockscale.BlockPool(data.to(gpu), heads, D, bits)
    for layer in (0, 2):
        out = tuple(torch.full((N, heads, D), 5.0, dtype=dtype, device=gpu) for _ in range(2))
        got = pkg.blockscale.read(pool, slots.to(gpu), dtype, layer=layer)
        assert pkg.blockscale.read(pool, slots.to(gpu), dtype, layer=layer, out=out)[0] is out[0]
        has = (slots >= 0) & (slots < pages * P)
        half = data[layer].view(pages * P, 2, -1)[slots.long().clamp(0, pages * P - 1)]
        want = torch.where(has[:, None, None, None], ref.values(half, heads, D, bits), 0.0).to(dtype)
        for i in range(2):
            same(got[i].cpu(), want[:, i], dtype)
            same(out[i].cpu(), want[:, i], dtype)


def test_read_nothing(pkg, gpu):
    pool = pkg.blockscale.BlockPool.zeros(1, 2, 4, 2, 64, 8, device=gpu)
    k, v = pkg.blockscale.read(pool, torch.empty(0, dtype=torch.int32, device=gpu))
    assert k.shape == v.shape == (0, 2, 64)
    k, v = pkg.blockscale.read(pool, torch.zeros(3, dtype=torch.int32, device=gpu))
    assert not k.any() and not v.any()


def test_write_and_read_in_a_graph_on_another_stream(pkg, gpu):
    c = case(31, 33, 8, 2, 128, 128, BF, 4)
    up = lambda t: None if t is None else t.to(gpu)  # noqa: E731
    x, data, slots = up(c["x"]), up(c["data"]), up(c["slots"])
    pos, freqs, wq, wk = up(c["pos"]), up(c["freqs"]), up(c["wq"]), up(c["wk"])
    pool = pkg.blockscale.BlockPool(data, 2, 128, 4)

    def step():
        q, k, v = split(c, x)
        q = pkg.attention.norm_rotate_write(q, k, v, pos, freqs, pool, slots, layer=1, q_weight=wq, k_weight=wk)
        return (q, *pkg.blockscale.read(pool, slots, BF, layer=1))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = step()
    torch.cuda.current_stream().wait_stream(stream)
    for seed in range(3):
        new = case(40 + seed, 33, 8, 2, 128, 128, BF, 4)
        x.copy_(new["x"])
        data.copy_(c["data"])
        graph.replay()
        got = [t.clone() for t in out]
        after = data.clone()
        data.copy_(c["data"])
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(after, data)
        check(dict(c, x=new["x"]), got[0].cpu(), after.cpu())
