"""Large steps, in which a wave takes three rows of each group, in every form that
takes that kernel: fp8 pools, pairs of neighbours, part of a head, several axes,
heads whose rows take no power of two of lanes.  Tokens at the ends, at the borders of
a block's work and some between, against the formulas in 64 bits."""
import pytest
import torch

from test_gpu_norm_rotate import BF, F8, FF, HF, case, near, rotate64, split

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N,Hq,Hk,D,rot,dtype,pool,axes,interleaved", [
    (17001, 32, 8, 128, 128, HF, F8, 1, False), (17001, 32, 8, 128, 64, BF, F8, 1, True),
    (25003, 28, 4, 128, 128, BF, BF, 3, False), (25003, 28, 4, 128, 96, FF, F8, 3, True),
    (20011, 32, 4, 80, 80, BF, BF, 1, True), (20011, 31, 5, 96, 64, HF, F8, 2, False),
    (33333, 13, 3, 80, 48, HF, HF, 1, False), (16400, 13, 5, 256, 256, BF, F8, 1, False),
    (20011, 5, 5, 512, 128, BF, BF, 1, False), (50021, 30, 1, 64, 0, BF, BF, 1, False),
])
def test_forms(pkg, gpu, N, Hq, Hk, D, rot, dtype, pool, axes, interleaved):
    units = rot // 16 + -(-(D - rot) // 16)
    groups = 64 >> (units - 1).bit_length()
    assert N * -(-(Hq + 2 * Hk) // groups) >= 12 * 256 * 32          # else one row of a group a wave
    c = case(N + D, N, Hq, Hk, D, rot, dtype, pool, axes=axes, interleaved=interleaved)
    if pool == F8:                                                   # (the last row of a token has no slot by default)
        c["slots"][N - 1] = (set(range(c["pool"].shape[1] * 16)) - set(c["slots"].tolist())).pop()
    scales = (0.02, 0.011) if pool == F8 else None
    x, held = c["x"].to(gpu), c["pool"].to(gpu)
    q, k, v = split(c, x)
    sc = [None, None] if scales is None else [torch.tensor([s], device=gpu) for s in scales]
    up = lambda t: None if t is None else t.to(gpu)  # noqa: E731
    got = pkg.attention.norm_rotate_write(
        q, k, v, up(c["pos"]), up(c["freqs"]) if rot else None, held, up(c["slots"]), layer=1, q_weight=up(c["wq"]),
        k_weight=up(c["wk"]), axis_of=up(c["axis_of"]), interleaved=interleaved, factor=0.75, k_scale=sc[0],
        v_scale=sc[1]).cpu()
    held = held.cpu()
    g = torch.Generator().manual_seed(1)
    some = torch.unique(torch.cat([torch.arange(70), torch.arange(N - 70, N), torch.tensor([N // 2]),
                                   torch.randint(0, N, (400,), generator=g)]))
    pos = c["pos"][..., some]
    q, k, v = (t[some] for t in split(c, c["x"]))
    rot64 = lambda t, w: rotate64(t, pos, c["freqs"], c["axis_of"], interleaved, 0.75, w, 1e-6, True)  # noqa: E731
    wq, sq = rot64(q, c["wq"])
    near(got[some], wq, sq, dtype, "q")
    wk, sk = rot64(k, c["wk"])
    slots = c["slots"][some].long()
    flat, was = held.view(2, -1, 2, Hk, D), c["pool"].view(2, -1, 2, Hk, D)
    kept = (slots >= 0) & (slots < flat.shape[1])
    assert kept.sum() > 400
    for i, (want, size, f) in enumerate(((wk, sk, 0.02), (v.double(), v.double().abs().amax(-1, keepdim=True), 0.011))):
        if pool != F8:
            f = 1.0
        want = want / f
        if pool == F8:
            want = want.clamp(-448.0, 448.0)
        near(flat[1, slots[kept], i], want[kept], size[kept] / f, pool, "KV"[i])
    raw = lambda t: t.contiguous().view(torch.uint8)  # noqa: E731
    assert torch.equal(raw(flat[0]), raw(was[0]))
    free = torch.ones(flat.shape[1], dtype=torch.bool)
    every = c["slots"].long()
    free[every[(every >= 0) & (every < flat.shape[1])]] = False
    assert torch.equal(raw(flat[1][free]), raw(was[1][free]))
