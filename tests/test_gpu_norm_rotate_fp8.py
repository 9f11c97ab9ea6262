"""An fp8 pool's values, value / scale rounded to 8 bits, bit for bit, in every
kernel of the cache write."""
import pytest
import torch

from test_gpu_norm_rotate import BF, F8, FF, HF

pytestmark = pytest.mark.gpu


def e4m3(x):
    """Quotients in 32 bits to e4m3, to nearest even, the largest past +-448."""
    return x.clamp(-448.0, 448.0).to(F8)


def ties(g, shape, scale, dtype):
    """Values next to `scale` times the midpoints of e4m3's steps."""
    exp, man = torch.randint(-6, 8, shape, generator=g), torch.randint(8, 16, shape, generator=g)
    sign = torch.randint(0, 2, shape, generator=g) * 2 - 1
    mid = sign * (man + 0.5) / 8 * 2.0 ** exp
    near = (mid.double() * float(torch.tensor(scale, dtype=torch.float32))).to(torch.float32)
    return near.to(dtype)


@pytest.mark.parametrize("dtype", [FF, BF, HF])
@pytest.mark.parametrize("N,Hq,Hk,D,half", [
    (60, 4, 2, 128, 64), (33, 3, 3, 80, 20), (41, 2, 1, 20, 10),           # eight values a lane; one
    (20000, 40, 8, 64, 32)])                                              # three rows of a group a wave
def test_values_at_the_midpoints(pkg, gpu, dtype, N, Hq, Hk, D, half):
    g = torch.Generator().manual_seed(N + D)
    P, pages = 16, -(-N // 16)
    slots = torch.randperm(pages * P, generator=g)[:N].to(torch.int32)
    q = torch.randn(N, Hq, D, generator=g).to(dtype)
    pos = torch.zeros(N, dtype=torch.int32)
    freqs = torch.ones(half, dtype=torch.float64)
    for scale in (0.02, 0.7, 1 / 3, 3.3e-4, 1.0):
        kv = ties(g, (2, N, Hk, D), scale, dtype)
        pool = torch.zeros(1, pages, P, 2, Hk, D, device=gpu).to(F8)
        s = torch.tensor([scale], device=gpu)
        # not turned (position 0) and not normed: K is value / scale as well
        pkg.attention.norm_rotate_write(q.to(gpu), kv[0].to(gpu), kv[1].to(gpu), pos.to(gpu), freqs.to(gpu), pool,
                                        slots.to(gpu), norm=False, k_scale=s, v_scale=s)
        want = e4m3(kv.float() / torch.tensor(scale)).view(torch.uint8)
        flat = pool.view(torch.uint8).view(-1, 2, Hk, D)[slots.to(gpu).long()].cpu().transpose(0, 1)
        both_zero = ((flat & 0x7F) == 0) & ((want & 0x7F) == 0)
        bad = (flat != want) & ~both_zero
        assert not bad.any(), f"scale {scale}: {int(bad.sum())} of {bad.numel()} bytes"


@pytest.mark.parametrize("D", [64, 20])
def test_scales_whose_reciprocal_overflows(pkg, gpu, D):
    """0 / scale is 0, whatever the scale; anything else stops at the largest value."""
    kv = torch.zeros(2, 4, 1, D)
    kv[:, 1] = 1.0
    kv[:, 2] = -1e-30
    kv[:, 3, 0, 3] = float("nan")
    for scale in (1e-39, 2e-45):
        s = torch.tensor([scale], device=gpu)
        pool = torch.ones(1, 1, 4, 2, 1, D, device=gpu).to(F8)
        slots = torch.arange(4, dtype=torch.int32, device=gpu)
        pkg.attention.norm_rotate_write(kv[0].to(gpu), kv[0].to(gpu), kv[1].to(gpu), None, None, pool, slots, norm=False,
                                        k_scale=s, v_scale=s)
        got = pool.float().cpu()[0, 0]
        assert (got[0] == 0).all() and (got[1] == 448).all() and (got[2] == -448).all()
        assert torch.isnan(got[3, :, 0, 3]).all() and int(torch.isnan(got).sum()) == 2
