"""Arguments of a step's calls at and past their limits: a ValueError that says so,
or the nearest thing that they can mean."""
import pytest
import torch

from test_gpu_prefix_attention import BF, check, make, reference, run

pytestmark = pytest.mark.gpu

FAR = 1 << 80


def test_hints_past_every_size(pkg, gpu):
    """max_q and max_len only bound and split the work: more than there can be is all."""
    c = make(gpu, 61, [90, 30, 200], [3, 1, 40], 8, 2, 64, BF, BF, 16, 16)
    ref = reference(c)
    for kw in ({"max_q": FAR}, {"max_q": 1 << 31}, {"max_len": FAR, "max_q": 40}, {"max_len": 1 << 63}):
        check(run(pkg, c, **kw), ref)


def test_attention_ranges(pkg, gpu):
    c = make(gpu, 62, [90, 30], [1, 1], 8, 2, 64, BF, BF, 16, 0)
    f = lambda **kw: run(pkg, c, **kw)  # noqa: E731
    for kw in ({"max_q": -1, "cu_q": c["cu"]}, {"max_q": -FAR, "cu_q": c["cu"]}, {"max_len": -1}, {"scale": 1e39},
               {"scale": -1e39}, {"layer": 2}, {"layer": -1}, {"layer": FAR}):
        with pytest.raises(ValueError):
            f(**kw)
    c["prefix"] = FAR
    with pytest.raises(ValueError):
        f()
    c["prefix"] = -FAR
    with pytest.raises(ValueError):
        f()


def test_tables_ranges(pkg, gpu):
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device=gpu)  # noqa: E731
    good = dict(page_table=i(2, 4), cached=i(2), new=i(2), free_pages=i(3), pool_pages=8, page_tokens=16, max_tokens=4)
    pkg.paged.step_tables(**good)
    for bad in ({"pool_pages": FAR}, {"page_tokens": 1 << 31}, {"page_tokens": -FAR}, {"max_tokens": FAR},
                {"max_tokens": 1 << 31}, {"pool_pages": -FAR}):
        with pytest.raises(ValueError):
            pkg.paged.step_tables(**{**good, **bad})


def test_write_ranges(pkg, gpu):
    x = torch.zeros(4, 2, 64, dtype=BF, device=gpu)
    pool = torch.zeros(1, 2, 4, 2, 2, 64, dtype=BF, device=gpu)
    slots = torch.arange(4, dtype=torch.int32, device=gpu)
    for kw in ({"eps": 1e39}, {"factor": -1e39}, {"layer": 1}, {"layer": FAR}):
        with pytest.raises(ValueError):
            pkg.attention.norm_rotate_write(x, x, x, None, None, pool, slots, **kw)
