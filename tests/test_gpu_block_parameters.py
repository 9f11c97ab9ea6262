"""eps and factor of a write into a cache with block scales: 32-bit numbers of the call, from which
keys are computed in 64 bits.  The bytes are those of the formulas with both rounded to 32 bits."""
import numpy as np
import pytest
import torch

import test_gpu_block_scale as scale
from test_gpu_norm_rotate import rotate64

pytestmark = pytest.mark.gpu

EPS = float(np.float32(1e-6))


@pytest.fixture(autouse=True)
def eps_as_given(monkeypatch):
    """The reference's eps (1e-6 in 64 bits) as the 32-bit number that the call takes."""
    def rotate(x, pos, freqs, axis_of, interleaved, factor, weight, eps, norm):
        assert eps == 1e-6
        return rotate64(x, pos, freqs, axis_of, interleaved, factor, weight, EPS, norm)
    monkeypatch.setattr(scale, "rotate64", rotate)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("factor", [1.1386, 0.1, 1 / 3, -0.7071067811865476])
def test_factors_that_32_bits_do_not_hold(pkg, gpu, bits, factor):
    for D, rot, inter, skew in ((128, 128, False, 0), (64, 32, True, 0), (96, 20, False, 1)):
        c = scale.case(D + bits, 300, 2, 4, D, rot, torch.float32, bits, interleaved=inter, skew=skew)
        got, data = scale.go(pkg, gpu, c, factor=factor)
        scale.check(c, got, data, factor=float(np.float32(factor)))


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "fp16", "fp32"])
def test_rows_under_eps(pkg, gpu, bits, dtype):
    """Heads whose mean square is far under eps, about it, and 0."""
    c = scale.case(bits, 300, 2, 4, 128, 128, dtype, bits)
    g = torch.Generator().manual_seed(3)
    c["x"] *= torch.exp2(-torch.randint(8, 15, (300, 1), generator=g).float()).to(dtype)
    c["x"][::50] = 0
    scale.check(c, *scale.go(pkg, gpu, c))
