"""The largest values of each type in a cache with block scales: what the documents say becomes of them."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, HF, FF = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("dtype", [BF, HF, FF], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("bits", [8, 4])
def test_largest_values(pkg, gpu, bits, dtype):
    """Past the last that does not round past its type's largest: that one, whatever they are read back as;
    those up to it as any other."""
    top = 2.0 ** (15 if dtype == HF else 127)
    last = top * (1.875 if bits == 8 else 1.5)
    most = torch.finfo(dtype).max
    v = torch.zeros(4, 1, 32)
    v[0, 0, :3] = torch.tensor([most, -most, last])
    v[1, 0, :2] = torch.tensor([last, -last])
    v[2, 0, :2] = torch.tensor([top, top * 1.25])            # (codes of 8 bits hold both, of 4 bits the first)
    v[3, 0, 0] = (last + most) / 2 if dtype != FF else last / 2 + most / 2
    v = v.to(dtype).to(gpu)
    pool = pkg.blockscale.BlockPool.zeros(1, 1, 4, 1, 32, bits, device=gpu)
    slots = torch.arange(4, dtype=torch.int32, device=gpu)
    pkg.attention.norm_rotate_write(v, v, v, None, None, pool, slots, norm=False)
    for as_ in (FF, dtype):
        k, got = pkg.blockscale.read(pool, slots, as_)
        assert torch.equal(k, got) and torch.isfinite(got).all()
        got = got[:, 0].double().cpu()
        assert got[0, :3].tolist() == [last, -last, last] and got[1, :2].tolist() == [last, -last]
        assert got[2, 0] == top and (bits == 4 or got[2, 1] == 1.25 * top) and got[3, 0] == last
