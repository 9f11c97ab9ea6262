"""Norm + rotation + cache write against the formulas in 64 bits.

Tolerance of a value: half a step of its type (eps/2 relative) for the one
rounding at the end, and 2^-18 of the row's largest value before it for the
32-bit arithmetic: the sum of squares of at most 512 values, at most 16 of them
in one lane and six additions across lanes, is off by at most 23 roundings of
2^-24 relative, its root by half of that; root, quotient and two products add
4, cos and sin at most 4 and their angle (rounded to 2^-26 turns) 2, the two
products and their sum 2 more: 24 * 2^-24 < 2^-19 of |a| + |b| <= 2 * largest.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, HF, FF, F8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn
ARITH = 2.0 ** -18
# spacing of the smallest values: half of it is the error of a value near zero
TINY = {BF: 2.0 ** -134, HF: 2.0 ** -25, FF: 2.0 ** -150, F8: 2.0 ** -10}


def rotate64(x, pos, freqs, axis_of, interleaved, factor, weight, eps, norm):
    x = x.double()
    if norm:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
        if weight is not None:
            x = x * weight.double()
    scale = x.abs().amax(-1, keepdim=True) * max(1.0, abs(factor))
    half = freqs.numel()
    if half:
        p = pos.double().reshape(-1, x.shape[0])
        ax = torch.zeros(half, dtype=torch.long) if axis_of is None else axis_of.long()
        ang = p[ax].t() * freqs.double()                      # [tokens, half]
        c, s = (torch.cos(ang) * factor)[:, None], (torch.sin(ang) * factor)[:, None]
        y = x.clone()
        i = torch.arange(half)
        ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        a, b = x[..., ia], x[..., ib]
        y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
        x = y
    return x, scale


def near(got, want, scale, dtype, what):
    got = got.double()
    tol = want.abs() * (torch.finfo(dtype).eps / 2) * (1 + 2.0 ** -10) + scale * ARITH + TINY[dtype]
    bad = (got - want).abs() > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} values off, worst {float(((got - want).abs() / tol).max()):.3g}"


def case(seed, N, Hq, Hk, D, rot, dtype, pool_dtype, axes=1, interleaved=False, norm=True, weights=True, packed=True,
         pages=None, P=16, skew=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(N, (Hq + 2 * Hk) * D + skew, generator=g).to(dtype)
    n_pages = pages or (-(-N // P) + 3)
    pool = (torch.randn(2, n_pages, P, 2, Hk, D, generator=g)).to(pool_dtype)
    slots = torch.randperm(n_pages * P, generator=g)[:N].to(torch.int32)
    if N > 2:
        slots[N // 2] = -1
        slots[N - 1] = n_pages * P                             # past the pool
    pos = torch.randint(-3, 1 << 20, (axes, N) if axes > 1 else (N,), generator=g, dtype=torch.int32)
    half = rot // 2
    freqs = 10000.0 ** (-torch.arange(half, dtype=torch.float64) / max(half, 1))
    axis_of = torch.randint(0, axes, (half,), generator=g).to(torch.uint8) if axes > 1 else None
    wq = (1 + 0.2 * torch.randn(D, generator=g)).to(dtype) if weights and norm else None
    wk = (1 + 0.2 * torch.randn(D, generator=g)).to(dtype) if weights and norm else None
    return dict(x=x, pool=pool, slots=slots, pos=pos, freqs=freqs, axis_of=axis_of, wq=wq, wk=wk, N=N, Hq=Hq, Hk=Hk,
                D=D, interleaved=interleaved, norm=norm, skew=skew, dtype=dtype)


def split(c, x):
    N, Hq, Hk, D = c["N"], c["Hq"], c["Hk"], c["D"]
    x = x[:, c["skew"]:]
    return (x[:, :Hq * D].unflatten(1, (Hq, D)), x[:, Hq * D:(Hq + Hk) * D].unflatten(1, (Hk, D)),
            x[:, (Hq + Hk) * D:].unflatten(1, (Hk, D)))


def go(pkg, gpu, c, layer=1, factor=1.0, eps=1e-6, scales=None, tokens=None, in_place=False, out=None):
    up = lambda t: None if t is None else t.to(gpu)  # noqa: E731
    x, pool = up(c["x"]), up(c["pool"])
    q, k, v = split(c, x)
    sc = (None, None) if scales is None else tuple(torch.tensor([s], device=gpu) for s in scales)
    got = pkg.attention.norm_rotate_write(
        q, k, v, up(c["pos"]), up(c["freqs"]) if c["freqs"].numel() else None, pool, up(c["slots"]), layer=layer,
        norm=c["norm"], q_weight=up(c["wq"]), k_weight=up(c["wk"]), eps=eps, axis_of=up(c["axis_of"]),
        interleaved=c["interleaved"], factor=factor, k_scale=sc[0], v_scale=sc[1],
        tokens=None if tokens is None else torch.tensor([tokens], dtype=torch.int32, device=gpu),
        out=q if in_place else up(out))
    return got.cpu(), pool.cpu(), x.cpu()


def check(c, got, pool, layer=1, factor=1.0, eps=1e-6, scales=None, tokens=None):
    N = c["N"] if tokens is None else min(max(tokens, 0), c["N"])
    q, k, v = split(c, c["x"])
    rot = lambda t, w: rotate64(t, c["pos"], c["freqs"], c["axis_of"], c["interleaved"], factor, w, eps, c["norm"])  # noqa: E731
    wq, sq = rot(q, c["wq"])
    near(got[:N], wq[:N], sq[:N], c["dtype"], "q")
    wk, sk = rot(k, c["wk"])
    ks, vs = scales or (1.0, 1.0)
    pt = c["pool"].dtype
    L, pages, P, _, Hk, D = pool.shape
    flat, was = pool.view(L, -1, 2, Hk, D), c["pool"].view(L, -1, 2, Hk, D)
    touched = torch.zeros(flat.shape[1], dtype=torch.bool)
    for t in range(N):
        s = int(c["slots"][t])
        if not 0 <= s < flat.shape[1]:
            continue
        touched[s] = True
        for i, (w, scale, f) in enumerate(((wk[t], sk[t], ks), (v[t].double(), v[t].double().abs().amax(-1, keepdim=True), vs))):
            want = w / f
            if pt == F8:
                want = want.clamp(-448.0, 448.0)
            near(flat[layer, s, i], want, scale / f, pt, f"pool slot {s} {'KV'[i]}")
    raw = lambda t: t.view(torch.uint8)  # noqa: E731
    assert torch.equal(raw(flat[1 - layer]), raw(was[1 - layer])), "the other layer was written"
    assert torch.equal(raw(flat[layer])[~touched], raw(was[layer])[~touched]), "a slot of no token was written"


@pytest.mark.parametrize("N", [1, 2, 17, 300])
@pytest.mark.parametrize("Hq,Hk,D,rot", [(32, 8, 128, 128), (8, 8, 64, 64), (7, 1, 80, 80), (4, 2, 96, 48),
                                         (3, 3, 256, 256), (5, 1, 512, 128)])
@pytest.mark.parametrize("dtype,pool", [(BF, BF), (HF, F8), (FF, FF)])
def test_shapes(pkg, gpu, N, Hq, Hk, D, rot, dtype, pool):
    c = case(N * 7 + D, N, Hq, Hk, D, rot, dtype, pool)
    scales = (0.02, 0.011) if pool == F8 else None
    got, after, _ = go(pkg, gpu, c, scales=scales)
    check(c, got, after, scales=scales)


@pytest.mark.parametrize("D,rot,interleaved,axes", [
    (128, 128, True, 1), (128, 64, True, 3), (128, 128, False, 3), (64, 0, False, 1), (80, 48, True, 2),
    (24, 20, False, 1), (24, 20, True, 3), (40, 40, False, 1), (16, 16, False, 1), (18, 6, False, 2), (510, 510, True, 1),
    (104, 64, False, 1)])
@pytest.mark.parametrize("dtype,pool", [(BF, BF), (HF, HF), (BF, F8), (FF, F8)])
def test_rotations(pkg, gpu, D, rot, interleaved, axes, dtype, pool):
    """Pairs of halves and of neighbours, part of a head, several axes, sizes
    that are no whole 16-byte chunks."""
    c = case(D + rot, 33, 6, 2, D, rot, dtype, pool, axes=axes, interleaved=interleaved)
    got, after, _ = go(pkg, gpu, c, layer=0, factor=1.25)
    check(c, got, after, layer=0, factor=1.25)


@pytest.mark.parametrize("norm,weights", [(False, False), (True, False)])
def test_no_norm_no_weight(pkg, gpu, norm, weights):
    c = case(4, 50, 8, 2, 128, 128, BF, BF, norm=norm, weights=weights)
    got, after, _ = go(pkg, gpu, c, eps=1e-2)
    check(c, got, after, eps=1e-2)


@pytest.mark.parametrize("skew", [1, 8])
def test_offsets(pkg, gpu, skew):
    """Rows that start on no 16-byte address, and rows that do again."""
    c = case(5, 40, 8, 2, 128, 128, BF, BF, skew=skew)
    got, after, _ = go(pkg, gpu, c)
    check(c, got, after)


def test_in_place(pkg, gpu):
    c = case(6, 64, 8, 2, 128, 128, BF, BF)
    got, after, x = go(pkg, gpu, c, in_place=True)
    check(c, got, after)
    q, k, v = split(c, x)
    assert torch.equal(q, got)
    assert torch.equal(k, split(c, c["x"])[1]) and torch.equal(v, split(c, c["x"])[2])


@pytest.mark.parametrize("tokens", [0, 1, 20, 64, 1000, -4])
def test_padded_step(pkg, gpu, tokens):
    """Tokens behind the step's last one are left as they were."""
    c = case(8, 64, 8, 2, 128, 128, BF, BF)
    mark = torch.full((64, 8, 128), 7.0, dtype=BF)
    got, after, _ = go(pkg, gpu, c, tokens=tokens, out=mark)
    check(c, got, after, tokens=tokens)
    assert (got[min(max(tokens, 0), 64):] == 7.0).all()


def test_no_tokens(pkg, gpu):
    c = case(9, 0, 8, 2, 128, 128, BF, BF)
    got, after, _ = go(pkg, gpu, c)
    assert got.shape == (0, 8, 128) and torch.equal(after.view(torch.uint8), c["pool"].view(torch.uint8))


def test_extremes(pkg, gpu):
    """Rows of zeros, of the largest values, infinities and NaN: each row keeps
    its own, and an fp8 pool stops at its largest value."""
    c = case(10, 12, 4, 1, 64, 64, FF, F8)
    x = c["x"].view(12, 6, 64)
    x[1] = 0.0
    x[2, :4] = 1e18
    x[3, 5] = 1e30
    x[4, 5, 3] = float("inf")
    x[4, 5, 4] = -float("inf")
    x[5, 5, 7] = float("nan")
    x[6, 0, 0] = float("nan")
    x[7, 1, 0] = float("inf")
    scales = (0.001, 0.5)
    got, pool, _ = go(pkg, gpu, c, scales=scales)
    fine = torch.ones(12, 4, dtype=torch.bool)
    fine[6, 0] = fine[7, 1] = False
    assert torch.isfinite(got).all(-1).eq(fine).all()
    flat = pool.view(2, -1, 2, 1, 64)[1]
    s = c["slots"].tolist()
    assert (flat[s[3], 1].float() == 448.0).all()
    assert flat[s[4], 1, 0, 3].float() == 448.0 and flat[s[4], 1, 0, 4].float() == -448.0
    assert torch.isnan(flat[s[5], 1, 0].float()).sum() == 1
    assert (got[1] == 0).all()
    # keys of an fp8 pool at a scale too small for them stop at the largest value
    assert float(flat[s[0], 0].float().abs().max()) == 448.0


def test_far_positions(pkg, gpu):
    """Angles keep their 64 bits out to the last position of 31 bits."""
    c = case(12, 64, 4, 1, 128, 128, FF, FF)
    c["pos"] = torch.randint(2**31 - 10**6, 2**31 - 1, (64,), generator=torch.Generator().manual_seed(1)).to(torch.int32)
    got, after, _ = go(pkg, gpu, c)
    check(c, got, after)


def test_one_position_row_for_all_axes(pkg, gpu):
    """Positions of text tokens, expanded over the axes without a copy."""
    c = case(13, 30, 4, 2, 64, 64, BF, BF, axes=3)
    one = c["pos"][0].clone()
    c["pos"] = one[None].expand(3, 30).contiguous()
    want = go(pkg, gpu, c)
    x, pool = c["x"].to(gpu), c["pool"].to(gpu)
    q, k, v = split(c, x)
    got = pkg.attention.norm_rotate_write(q, k, v, one.to(gpu)[None].expand(3, 30), c["freqs"].to(gpu), pool,
                                          c["slots"].to(gpu), layer=1, q_weight=c["wq"].to(gpu),
                                          k_weight=c["wk"].to(gpu), axis_of=c["axis_of"].to(gpu))
    assert torch.equal(got.cpu(), want[0]) and torch.equal(pool.cpu(), want[1])


@pytest.mark.parametrize("N,Hq,Hk,D,dtype,pool", [(50000, 9, 3, 128, BF, BF), (17000, 32, 8, 128, HF, HF),
                                                  (33001, 26, 4, 64, BF, BF), (99000, 4, 2, 64, torch.float32, torch.float32)])
def test_large_step_takes_the_deep_kernel(pkg, gpu, N, Hq, Hk, D, dtype, pool):
    """Enough rows that a wave takes three of each group (98304 waves of one
    each): the same bytes as in small calls."""
    waves = N * -(-(Hq + 2 * Hk) // (64 // (D // 16)))
    assert waves >= 12 * 256 * 32
    c = case(14, N, Hq, Hk, D, D, dtype, pool)
    whole = go(pkg, gpu, c)
    x, pool = c["x"].to(gpu), c["pool"].to(gpu)
    q, k, v = split(c, x)
    parts = []
    for a in range(0, N, 5000):
        b = min(a + 5000, N)
        parts.append(pkg.attention.norm_rotate_write(
            q[a:b], k[a:b], v[a:b], c["pos"][a:b].to(gpu), c["freqs"].to(gpu), pool, c["slots"][a:b].to(gpu), layer=1,
            q_weight=c["wq"].to(gpu), k_weight=c["wk"].to(gpu)))
    assert torch.equal(torch.cat(parts).cpu(), whole[0]) and torch.equal(pool.cpu(), whole[1])


def test_captured(pkg, gpu):
    c = case(15, 70, 8, 2, 128, 128, BF, BF)
    x, pool, pos, slots = c["x"].to(gpu), c["pool"].to(gpu), c["pos"].to(gpu), c["slots"].to(gpu)
    freqs, wq, wk = c["freqs"].to(gpu), c["wq"].to(gpu), c["wk"].to(gpu)

    def call():
        q, k, v = split(c, x)
        return pkg.attention.norm_rotate_write(q, k, v, pos, freqs, pool, slots, layer=1, q_weight=wq, k_weight=wk)

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for seed in (21, 22, 23):
        c2 = case(seed, 70, 8, 2, 128, 128, BF, BF)
        c2.update(wq=c["wq"], wk=c["wk"])
        x.copy_(c2["x"]), pool.copy_(c2["pool"]), pos.copy_(c2["pos"]), slots.copy_(c2["slots"])
        graph.replay()
        torch.cuda.synchronize()
        check(c2, got.cpu(), pool.cpu())


def test_offsets_past_32_bits(pkg, gpu):
    """A pool layer of more than 4 GiB: slots at both ends."""
    Hk, D, P = 8, 128, 16
    pages = (5 << 30) // (P * 2 * Hk * D * 2)
    pool = torch.zeros(1, pages, P, 2, Hk, D, dtype=BF, device=gpu)
    n = pages * P
    slots = torch.tensor([0, n - 1, n // 2, 1 << 20], dtype=torch.int32, device=gpu)
    kv = torch.randn(2, 4, Hk, D, device=gpu).to(BF)
    q = torch.randn(4, Hk, D, device=gpu).to(BF)
    pkg.attention.norm_rotate_write(q, kv[0], kv[1], None, None, pool, slots, norm=False)
    flat = pool.view(n, 2, Hk, D)
    assert torch.equal(flat[slots.long()].transpose(0, 1), kv)
    assert int(torch.count_nonzero(flat[1:1000])) == 0
