"""Scores far past what a 32-bit number resolves to a power of two: finite inputs
whose best keys stand out give those keys' values, whatever the scores' size."""
import pytest
import torch

from test_gpu_prefix_attention import BF, F8, HF, make, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,sizes", [(BF, (2.0 ** 9, 2.0 ** 15, 2.0 ** 22, 2.0 ** 31, 3.0 * 2.0 ** 45, 2.0 ** 100)),
                                         (HF, (2.0 ** 9, 2.0 ** 15, 2.0 ** 22, 3.0 * 2.0 ** 25, 2.0 ** 29))])
@pytest.mark.parametrize("new,prefix", [([1, 1, 1], 0), ([1] * 20, 200), ([1, 1], 200), ([40, 9], 0), ([40, 90], 200)])
@pytest.mark.parametrize("sign", [1, -1])
def test_the_best_keys(pkg, gpu, dtype, sizes, new, prefix, sign):
    """Scores are exact products of few bits: sign * size * (1, 15/16, ..., 9/16), so
    the best are at least 2^5 apart from the rest and get all the weight (2^-46 for
    the next), equal ones an equal share: the plain mean of their values, which
    differs by the rounding of the result (half a step), of 32-bit sums, and of the
    weights, which are equal, not at all."""
    lens = [prefix + n + 260 for n in new]
    c = make(gpu, 81, lens, new, 8, 2, 64, dtype, dtype, 16, prefix)
    g = torch.Generator().manual_seed(82)
    L, pages, P, _, Hk, D = c["pool"].shape
    level = torch.randint(0, 8, (pages, P), generator=g).to(gpu)
    c["pool"][1, :, :, 0] = 0
    big = 2.0 ** 60 if dtype == BF else 2.0 ** 15
    u = torch.finfo(dtype).eps / 2
    flat = c["pool"][1].view(-1, 2, Hk, D)
    for size in sizes:
        a = min(size / 2, big)                                # the query's value, the key's makes up the rest
        c["pool"][1, :, :, 0, :, 3] = (size / a * (16 - level).double() / 16)[..., None].to(dtype)
        c["q"].zero_()
        c["q"][..., 3] = sign * a
        got = run(pkg, c, cu_q=c["cu"], max_q=max(new), scale=1.0).double()
        tab, cu = c["table"].tolist(), c["cu"].tolist()
        for b, n in enumerate(lens):
            at = torch.tensor([(tab[0] if j < prefix else tab[b])[j // P] * P + j % P for j in range(n)], device=gpu)
            lev, V = level.view(-1)[at], flat[at, 1].double()
            for i in range(cu[b], cu[b + 1]):
                see = n - (cu[b + 1] - cu[b]) + i - cu[b] + 1
                best = lev[:see] == (lev[:see].min() if sign > 0 else lev[:see].max())
                want = V[:see][best].mean(0).repeat_interleave(4, 0)
                size_v = V[:see][best].abs().mean(0).repeat_interleave(4, 0)
                tol = u * want.abs() * (1 + 2.0 ** -7) + size_v * 2.0 ** -14 + 2.0 ** -25
                assert ((got[i] - want).abs() <= tol).all(), (size, b, i, got[i, 0, :3].tolist(), want[0, :3].tolist())


@pytest.mark.parametrize("new,prefix", [([1, 1, 1], 0), ([1] * 20, 300), ([60, 9], 0), ([60, 90], 300)])
def test_large_queries(pkg, gpu, new, prefix):
    """Random queries of up to 2^40: finite, and V of the best key where 32-bit sums
    leave no doubt which that is."""
    lens = [prefix + n + 300 for n in new]
    for dtype, up in ((BF, 20), (BF, 40), (HF, 14)):
        c = make(gpu, 83, lens, new, 8, 2, 64, dtype, dtype, 16, prefix)
        c["q"] = (c["q"].double().clamp(-1.9, 1.9) * 2.0 ** up).to(dtype)
        got = run(pkg, c, cu_q=c["cu"], max_q=max(new)).double()
        assert torch.isfinite(got).all()
        flat, tab, cu = c["pool"][1].view(-1, 2, 2, 64).double(), c["table"].tolist(), c["cu"].tolist()
        sure = 0
        for b, n in enumerate(lens):
            at = torch.tensor([(tab[0] if j < prefix else tab[b])[j // 16] * 16 + j % 16 for j in range(n)], device=gpu)
            for i in range(cu[b], cu[b + 1]):
                see = n - (cu[b + 1] - cu[b]) + i - cu[b] + 1
                K, V = flat[at[:see], 0].repeat_interleave(4, 1), flat[at[:see], 1].repeat_interleave(4, 1)
                q = c["q"][i].double()
                s, size = torch.einsum("hd,khd->hk", q, K) / 8, torch.einsum("hd,khd->hk", q.abs(), K.abs()) / 8
                two = s.topk(2, 1)
                clear = two.values[:, 0] - two.values[:, 1] > 2 * 64 * 2.0 ** -24 * size.amax(1) + 60
                sure += int(clear.sum())
                want = V[two.indices[:, 0], torch.arange(8, device=gpu)]
                assert torch.equal(got[i][clear], want[clear]), (dtype, up, b, i)
        assert sure > 4 * sum(new)
