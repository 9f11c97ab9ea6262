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


def test_a_step_without_tokens(pkg, gpu):
    """All requests idle in a padded step: nothing is written, every row is zeros; the
    attention alone leaves its rows."""
    pool = torch.full((1, 8, 16, 2, 2, 64), 5.0, dtype=BF, device=gpu)
    table = torch.tensor([[1, 2, -1], [3, -1, -1]], dtype=torch.int32, device=gpu)
    be = pkg.serving.PagedBackend(pool, table, freqs=pkg.attention.rotary_frequencies(64, device=gpu))
    i = lambda *x: torch.tensor(x, dtype=torch.int32, device=gpu)  # noqa: E731
    free = torch.arange(4, 8, dtype=torch.int32, device=gpu)
    for tokens in (0, 6):
        batch = be.begin(i(20, 9), i(0, 0), free, tokens, 0)
        q, k, v = (torch.ones(tokens, h, 64, dtype=BF, device=gpu) for h in (4, 2, 2))
        out = be.forward_extend(batch, q, k, v)
        assert out.shape == (tokens, 4, 64) and (out == 0).all()
        assert int(batch.taken) == 0 and batch.seq_lens.tolist() == [20, 9] and (batch.slot_mapping == -1).all()
    assert (pool == 5.0).all() and table.tolist() == [[1, 2, -1], [3, -1, -1]]
    out = torch.full((6, 4, 64), 3.0, dtype=BF, device=gpu)
    got = pkg.attention.prefix_attention(q, pool, table, i(20, 9), cu_q=i(0, 0, 0), max_q=0, out=out)
    assert got is out and (out == 3.0).all()
    # without cu_q there is one token a request, whatever max_q says
    c = make(gpu, 63, [90, 30], [1, 1], 8, 2, 64, BF, BF, 16, 0)
    check(run(pkg, c, max_q=0), reference(c))
