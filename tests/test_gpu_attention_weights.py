"""The softmax's weights where 16 bits are short for them."""
import math

import pytest
import torch

from test_gpu_prefix_attention import BF, HF

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [HF, BF])
@pytest.mark.parametrize("drop,n", [(16, 32768), (22, 1 << 18), (25.5, 1 << 18)])
@pytest.mark.parametrize("new,prefix,max_len", [(1, 0, 10), (40, 0, 10), (40, 0, 0), (1, 1, 0), (24, 1, 10)])
def test_a_long_tail_under_a_peak(pkg, gpu, dtype, drop, n, new, prefix, max_len):
    """The first key weighs 1 with V = 0, each other one t = 2^-drop with V = 1: with
    n' of those the output is n' t / (1 + n' t).  Tolerance, with the names of the
    general one: half a step of the result, u; of each weight's rounding, u and a
    2^-22 of its power, relative, and half a step of the smallest fp16 numbers, whose
    unit the largest weight exceeds 2^7 times at least: n' 2^-32; sums of n' terms,
    n' 2^-24 relative.  Both sums are off so."""
    t, D = 2.0 ** -drop, 64
    B = 3 if prefix else 1                                    # enough rows for tile blocks of the shared part
    if prefix:
        prefix = n - 64
    P = 64
    width = -(-(n + new) // P)
    pool = torch.zeros(1, width, P, 2, 1, D, dtype=dtype, device=gpu)
    flat = pool.view(-1, 2, 1, D)
    flat[:, 1] = 1.0
    flat[0, 1] = 0.0
    flat[0, 0, 0, 0] = drop
    q = torch.zeros(B * new, 16, D, dtype=dtype, device=gpu)
    q[..., 0] = 1.0
    table = torch.arange(width, dtype=torch.int32, device=gpu)[None].expand(B, -1).contiguous()
    lens = torch.full((B,), n + new, dtype=torch.int32, device=gpu)
    cu = torch.arange(B + 1, dtype=torch.int32, device=gpu) * new
    got = pkg.attention.prefix_attention(q, pool, table, lens, prefix, cu_q=cu, max_q=new, max_len=max_len or None,
                                         scale=math.log(2.0))
    tail = (n + torch.arange(new, dtype=torch.float64, device=gpu)).repeat(B) * t
    want = (tail / (1 + tail))[:, None, None]
    u = torch.finfo(dtype).eps / 2
    one = tail * (u + 2.0 ** -22 + (n + new) * 2.0 ** -24)
    if dtype == HF:
        one = one + (n + new) * 2.0 ** -32
    tol = u * want + (2 * one / (1 + tail))[:, None, None] * 1.01
    off = (got.double() - want).abs()
    assert (off <= tol).all(), f"{float((off / tol).max()):.3g} of the tolerance, {got[0, 0, 0]} for {float(want[0, 0, 0])}"


@pytest.mark.parametrize("dtype,up", [(BF, 128.445), (HF, 128.0624)])
@pytest.mark.parametrize("new,prefix", [(1, 0), (3, 0), (40, 0), (1, 192), (3, 192)])
def test_the_average_of_equal_values(pkg, gpu, dtype, up, new, prefix):
    """V is one value, so the result is that value, whatever the weights are rounded
    to: it differs by 32-bit sums only.  Here one key outweighs the first by `up`,
    which is nearly half a step off what 16 bits hold and too little to move the
    running maximum; the others weigh nothing."""
    D, P, n = 64, 16, 200
    value = 2.0 - torch.finfo(dtype).eps
    width = -(-(n + new) // P)
    pool = torch.zeros(1, width, P, 2, 1, D, dtype=dtype, device=gpu)
    flat = pool.view(-1, 2, 1, D)
    flat[:, 1] = value
    flat[1:, 0, 0, 0] = -60.0
    flat[130, 0, 0, 0] = 7.0
    flat[130, 0, 0, 1] = math.log2(up) - 7.0
    B = 3 if prefix else 1
    q = torch.zeros(B * new, 16, D, dtype=dtype, device=gpu)
    q[..., :2] = 1.0
    table = torch.arange(width, dtype=torch.int32, device=gpu)[None].expand(B, -1).contiguous()
    lens = torch.full((B,), n + new, dtype=torch.int32, device=gpu)
    cu = torch.arange(B + 1, dtype=torch.int32, device=gpu) * new
    got = pkg.attention.prefix_attention(q, pool, table, lens, prefix, cu_q=cu, max_q=new, max_len=10, scale=math.log(2.0))
    assert (got == value).all(), f"{float(got[0, 0, 0])} for {value}"
