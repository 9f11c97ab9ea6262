"""The prefix's pages come from `prefix_pages` alone, in every kind of block and at
every unit of keys: the rows' own entries for those positions name pages of NaN, or no
pages at all."""
import pytest
import torch

from test_gpu_prefix_attention import BF, F8, HF, check, make, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,pool,D", [(BF, BF, 64), (HF, HF, 64), (BF, F8, 64), (BF, BF, 96), (HF, F8, 96), (BF, BF, 128),
                                          (HF, HF, 128), (HF, F8, 128), (BF, BF, 256), (BF, F8, 256)])
@pytest.mark.parametrize("prefix", [40, 300, 1245, 1280])
@pytest.mark.parametrize("new", [[1, 1, 1], [1] * 30, [60, 1, 90], [150, 40]])
def test_not_from_the_rows(pkg, gpu, dtype, pool, D, prefix, new):
    lens = [prefix + n + 150 for n in new]
    c = make(gpu, 71, lens, new, 4, 2, D, dtype, pool, 16, prefix)
    front = c["table"][0, :-(-prefix // 16)].clone()
    kw = dict(ks=0.03, vs=0.02) if pool == F8 else {}
    sc = {"k_scale": torch.tensor([0.03], device=gpu), "v_scale": torch.tensor([0.02], device=gpu)} if pool == F8 else {}
    ref = reference(c, prefix_pages=front, **kw)
    empty = sorted(set(range(c["pool_pages"])) - set(c["table"].flatten().tolist()))[0]      # NaN throughout
    for entry in (empty, -1):
        c["table"][:, :prefix // 16] = entry
        for max_len in (max(lens), prefix + 400, None):
            got = pkg.attention.prefix_attention(c["q"], c["pool"], c["table"], c["lens"], prefix, layer=1, cu_q=c["cu"],
                                                 max_q=max(new), max_len=max_len, prefix_pages=front, **sc)
            check(got, ref)


@pytest.mark.parametrize("dtype,pool,D", [(BF, BF, 64), (HF, F8, 96), (BF, BF, 128), (BF, BF, 256)])
@pytest.mark.parametrize("prefix", [300, 1245, 1280])
@pytest.mark.parametrize("new", [[1] * 30, [60, 1, 90]])
def test_prefix_pages_that_are_not_there(pkg, gpu, dtype, pool, D, prefix, new):
    """Prefix pages outside the pool are left out for all, whatever the rows say."""
    lens = [prefix + n + 150 for n in new]
    c = make(gpu, 72, lens, new, 4, 2, D, dtype, pool, 16, prefix)
    front = c["table"][0, :-(-prefix // 16)].clone()
    front[: prefix // 16] = -1
    front[1] = c["table"][0, 1]
    kw = dict(ks=0.03, vs=0.02) if pool == F8 else {}
    sc = {"k_scale": torch.tensor([0.03], device=gpu), "v_scale": torch.tensor([0.02], device=gpu)} if pool == F8 else {}
    ref = reference(c, prefix_pages=front, **kw)
    for max_len in (max(lens), prefix + 400, None):
        got = pkg.attention.prefix_attention(c["q"], c["pool"], c["table"], c["lens"], prefix, layer=1, cu_q=c["cu"],
                                             max_q=max(new), max_len=max_len, prefix_pages=front, **sc)
        check(got, ref)
