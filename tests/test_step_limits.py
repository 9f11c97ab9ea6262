"""Sizes that no launch can have, and arguments that no call can, are refused on
the host with a code or a ValueError (CPU only: the addresses are made up)."""
import ctypes as C

import pytest
import torch

from test_step_refusals import at, no_gpu, nr  # noqa: F401


@pytest.mark.parametrize("kw", [
    # one block of 256 threads for each of 2^24 rows joins the parts
    dict(tokens=1 << 21, batch=1 << 21, cu_q=1 << 56, max_q=1, prefix=100),
    dict(tokens=1 << 20, batch=1 << 20, heads=16, prefix=100),
    # 2^24 stream blocks: a request's rows by max_q, 16 a block
    dict(tokens=1 << 20, batch=1 << 15, cu_q=1 << 56, max_q=1 << 20, prefix=128, max_len=128),
    dict(tokens=1 << 14, batch=1 << 19, cu_q=1 << 56, max_q=1 << 14, heads=64, kv_heads=64, prefix=0, max_len=1),
])
def test_attention_grids(pkg, kw):
    L = pkg._lib.lib()
    f = dict(q=1 << 50, out=1 << 51, pool=1 << 52, page_table=1 << 53, seq_lens=1 << 54, prefix_pages=1 << 55)
    f.update(kw)
    heads = f.get("heads", 8)
    f.update(q_stride=heads * 64, o_stride=heads * 64)
    call = at(pkg, **f)
    assert L.kvec_prefix_attention_workspace(C.byref(call)) == -1
    assert b"launch" in L.kvec_last_error()
    assert L.kvec_prefix_attention(C.byref(call), 1 << 57, 1 << 60, None) == -2
    assert b"launch" in L.kvec_last_error()


def test_norm_rotate_grid(pkg):
    L = pkg._lib.lib()
    far = dict(q=1 << 50, k=1 << 51, v=1 << 52, q_out=1 << 53, positions=1 << 54, pool=1 << 55, slots=1 << 56,
               axis_stride=1 << 26)
    call = nr(pkg, tokens=1 << 26, heads=1, kv_heads=1, dim=64, q_stride=64, o_stride=64, k_stride=64, v_stride=64, **far)
    assert L.kvec_norm_rotate_write(C.byref(call), None) == -2
    assert b"launch" in L.kvec_last_error()


def test_gradients_are_refused(pkg):
    """There is no backward pass: a result that silently lost its history would train
    nothing.  Without gradients in play the call goes on (to its other checks)."""
    A = pkg.attention
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    q, kv = torch.zeros(4, 2, 64), torch.zeros(4, 2, 64)
    pool, w = torch.zeros(1, 2, 4, 2, 2, 64), torch.zeros(64)

    def write(**g):
        t = {n: x.clone().requires_grad_(n in g) for n, x in (("q", q), ("k", kv), ("v", kv), ("w", w), ("pool", pool))}
        A.norm_rotate_write(t["q"], t["k"], t["v"], None, None, t["pool"], i(4), q_weight=t["w"], k_weight=w)

    for n in ("q", "k", "v", "w", "pool"):
        with pytest.raises(ValueError, match="no backward"):
            write(**{n: True})
        with torch.no_grad(), pytest.raises(ValueError, match="GPU"):
            write(**{n: True})
    with pytest.raises(ValueError, match="GPU"):
        write()
    with torch.no_grad(), pytest.raises(ValueError, match="GPU"):
        A.norm_rotate_write(q, kv, kv, None, None, pool, i(4), q_weight=torch.nn.Parameter(w))
    for n in ("q", "pool"):
        t = {"q": q.half(), "pool": pool.half()}
        t[n].requires_grad_()
        with pytest.raises(ValueError, match="no backward"):
            A.prefix_attention(t["q"], t["pool"], i(4, 3), i(4))
        with torch.inference_mode(), pytest.raises(ValueError, match="GPU"):
            A.prefix_attention(t["q"], t["pool"], i(4, 3), i(4))


def rows_meet(n, s, h, t, length):
    at = sorted(i * s + j * t for i in range(n) for j in range(h))
    return any(b - a < length for a, b in zip(at, at[1:]))


@pytest.mark.parametrize("n,h", [(1, 1), (1, 5), (5, 1), (2, 2), (4, 8), (7, 3)])
def test_rows_of_the_result_that_overlap(pkg, n, h):
    """Every pair of strides: refused just where two rows share a value (a call that is
    taken goes on to the next refusal)."""
    L = pkg._lib.lib()
    seen = set()
    for s in (0, 4, 8, 12, 16, 20, 24, 40, 64, 100, 1 << 40):
        for t in (0, 4, 8, 12, 16, 20, 24, 32, 56, 57, 1 << 40):
            meet = rows_meet(n, s, h, t, 8)
            seen.add(meet)
            call = nr(pkg, tokens=n, heads=h, kv_heads=1, dim=8, rot=0, o_stride=s, o_head_stride=t, q_stride=8 * h,
                      q_head_stride=8, q_out=1 << 27, pool=1 << 27)
            assert L.kvec_norm_rotate_write(C.byref(call), None) == -1
            assert (b"rows of q_out overlap" in L.kvec_last_error()) == meet, (s, t)
            call = at(pkg, tokens=n, batch=n, heads=h, kv_heads=1, dim=8, o_stride=s, o_head_stride=t, q_stride=8 * h,
                      q_head_stride=8, prefix=0)
            call.out = call.pool
            assert L.kvec_prefix_attention(C.byref(call), 1 << 50, 1 << 40, None) == -1
            assert (b"rows of out overlap" in L.kvec_last_error()) == meet, (s, t)
    assert seen == ({False} if n * h == 1 else {False, True})


def test_scales_that_overflow(pkg):
    """A scale whose product with log2(e) is no 32-bit number would make NaN of every row."""
    L = pkg._lib.lib()
    for scale, code in ((2.5e38, -1), (3.4e38, -1), (2.2e38, 0)):
        call = at(pkg, scale=scale)
        need = L.kvec_prefix_attention_workspace(C.byref(call))
        assert (need < 0) == (code < 0)
        if code:
            assert b"scale" in L.kvec_last_error()
