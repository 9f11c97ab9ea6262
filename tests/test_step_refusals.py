"""The serving-step entry points refuse bad arguments on the host, before any
launch (CPU only: the addresses are made up)."""
import ctypes as C

import pytest
import torch


@pytest.fixture(autouse=True)
def no_gpu():
    if torch.cuda.is_available():
        pytest.skip("made-up device addresses: CPU-only test")


def step(pkg, **kw):
    f = dict(page_table=1 << 20, batch=4, pages_per_seq=8, page_tokens=16, pool_pages=100, cached=1 << 21,
             new_tokens=(1 << 21) + 64, free_pages=1 << 22, n_free=10, slots=1 << 23, positions=1 << 24,
             max_tokens=64, cu_new=1 << 25, seq_lens=1 << 26, taken=1 << 27)
    f.update(kw)
    return pkg._lib.Step(**f)


@pytest.mark.parametrize("bad,code,word", [
    ({"batch": -1}, -1, b"sizes"),
    ({"pages_per_seq": 0}, -1, b"sizes"),
    ({"max_tokens": -1}, -1, b"sizes"),
    ({"page_tokens": 12}, -1, b"power of two"),
    ({"page_tokens": 0}, -1, b"power of two"),
    ({"pool_pages": (1 << 27) + 1}, -2, b"2^31"),
    ({"batch": 1 << 20, "pages_per_seq": 1 << 11}, -2, b"2^31"),
    ({"page_table": None}, -1, b"null"),
    ({"slots": None}, -1, b"null"),
    ({"free_pages": None}, -1, b"null"),
    ({"taken": None}, -1, b"null"),
    ({"slots": (1 << 24) + 4}, -1, b"overlaps"),
    ({"free_pages": 1 << 20}, -1, b"overlaps"),
])
def test_step_tables_refuses(pkg, bad, code, word):
    L = pkg._lib.lib()
    assert L.kvec_step_tables(C.byref(step(pkg, **bad)), None) == code
    assert word in L.kvec_last_error()


def test_step_tables_null(pkg):
    assert pkg._lib.lib().kvec_step_tables(None, None) == -1


def nr(pkg, **kw):
    f = dict(tokens=4, heads=8, kv_heads=2, dim=64, dtype=1, q=1 << 20, k=1 << 21, v=1 << 22, q_stride=512,
             q_head_stride=64, k_stride=128, k_head_stride=64, v_stride=128, v_head_stride=64, q_out=1 << 23,
             o_stride=512, o_head_stride=64, norm=1, eps=1e-6, rot=64, interleaved=0, axes=1, positions=1 << 24,
             axis_stride=4, freqs=1 << 25, factor=1.0, pool=1 << 26, pool_dtype=1, n_slots=64, slots=1 << 27)
    f.update(kw)
    return pkg._lib.NormRotate(**f)


@pytest.mark.parametrize("bad,code,word", [
    ({"tokens": -1}, -1, b"sizes"),
    ({"kv_heads": 0}, -1, b"sizes"),
    ({"dim": 1024}, -2, b"dim"),
    ({"rot": 63}, -1, b"rot"),
    ({"rot": 66}, -1, b"rot"),
    ({"dtype": 3}, -1, b"dtype"),
    ({"pool_dtype": 2}, -1, b"pool_dtype"),
    ({"k_scale": 1 << 28}, -1, b"scales"),
    ({"axes": 9}, -1, b"axes"),
    ({"axes": 0}, -1, b"axes"),
    ({"axis_stride": -4}, -1, b"axis_stride"),
    ({"eps": -1.0}, -1, b"eps"),
    ({"eps": float("nan")}, -1, b"eps"),
    ({"q": None}, -1, b"null"),
    ({"slots": None}, -1, b"null"),
    ({"freqs": None}, -1, b"null"),
    ({"pool": None}, -1, b"null"),
    ({"k_stride": -128}, -1, b"stride"),
    ({"o_head_stride": 32}, -1, b"overlap"),
    ({"q_out": (1 << 20) + 64}, -1, b"overlaps"),      # part of q, not q itself
    ({"pool": 1 << 22}, -1, b"overlaps"),              # v
    ({"q_out": 1 << 26}, -1, b"overlaps"),             # the pool
])
def test_norm_rotate_refuses(pkg, bad, code, word):
    L = pkg._lib.lib()
    assert L.kvec_norm_rotate_write(C.byref(nr(pkg, **bad)), None) == code
    assert word in L.kvec_last_error()


def test_no_tokens_is_no_launch(pkg):
    L = pkg._lib.lib()
    assert L.kvec_norm_rotate_write(C.byref(nr(pkg, tokens=0, q=None, k=None, v=None)), None) == 0


def test_python_refusals(pkg):
    """The wrappers name what is wrong with host tensors, types and shapes."""
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(ValueError, match="GPU"):
        pkg.paged.step_tables(i(2, 4), i(2), i(2), i(3), 8, 16, 4)
    with pytest.raises(ValueError, match="int32"):
        pkg.paged.step_tables(i(2, 4).long(), i(2), i(2), i(3), 8, 16, 4)
    with pytest.raises(ValueError, match="one entry"):
        pkg.paged.step_tables(i(2, 4), i(3), i(2), i(3), 8, 16, 4)
    x = torch.zeros(4, 2, 64)
    pool = torch.zeros(1, 2, 4, 2, 2, 64)
    with pytest.raises(ValueError, match="GPU"):
        pkg.attention.norm_rotate_write(x, x, x, None, None, pool, i(4))
    with pytest.raises(ValueError, match="one type"):
        pkg.attention.norm_rotate_write(x, x.half(), x, None, None, pool, i(4))
    with pytest.raises(ValueError, match="kv_heads"):
        pkg.attention.norm_rotate_write(x, x[:3], x, None, None, pool, i(4))


def test_rotary_helpers(pkg):
    f = pkg.attention.rotary_frequencies(64, 10000.0, device="cpu")
    assert f.dtype == torch.float64 and f.shape == (32,) and float(f[0]) == 1.0
    assert abs(float(f[16]) - 0.01) < 1e-15
    a = pkg.attention.rotary_axes([2, 0, 3], device="cpu")
    assert a.tolist() == [0, 0, 2, 2, 2] and a.dtype == torch.uint8
    for bad in (0, 3):
        with pytest.raises(ValueError):
            pkg.attention.rotary_frequencies(bad, device="cpu")
    with pytest.raises(ValueError):
        pkg.attention.rotary_axes([1, -1], device="cpu")


def at(pkg, **kw):
    f = dict(tokens=4, batch=4, heads=8, kv_heads=2, dim=64, dtype=1, q=1 << 20, q_stride=512, q_head_stride=64,
             out=1 << 21, o_stride=512, o_head_stride=64, pool=1 << 22, pool_dtype=1, pool_pages=50, page_tokens=16,
             page_table=1 << 23, pages_per_seq=8, seq_lens=1 << 24, max_q=1, prefix=20, prefix_pages=1 << 25,
             scale=0.125)
    f.update(kw)
    return pkg._lib.Attention(**f)


@pytest.mark.parametrize("bad,code,word", [
    ({"tokens": -1}, -1, b"sizes"),
    ({"heads": 7}, -1, b"sizes"),
    ({"prefix": -1}, -1, b"sizes"),
    ({"dtype": 0}, -1, b"dtype"),
    ({"pool_dtype": 2}, -1, b"pool_dtype"),
    ({"v_scale": 1 << 28}, -1, b"scales"),
    ({"dim": 264}, -2, b"dim"),
    ({"dim": 60}, -2, b"dim"),
    ({"dim": 72, "pool_dtype": 3}, -2, b"dim"),
    ({"page_tokens": 24}, -1, b"power of two"),
    ({"pool_pages": 1 << 28}, -2, b"2^31"),
    ({"pages_per_seq": 1 << 27}, -2, b"2^31"),
    ({"prefix": 129}, -1, b"prefix"),
    ({"tokens": 5}, -1, b"max_q"),
    ({"cu_q": 1 << 26, "max_q": 0}, -1, b"max_q"),
    ({"scale": -0.5}, -1, b"scale"),
    ({"scale": float("nan")}, -1, b"scale"),
    ({"scale": float("inf")}, -1, b"scale"),
    ({"tokens": 1 << 23, "batch": 1 << 23}, -2, b"rows"),
])
def test_attention_refuses(pkg, bad, code, word):
    L = pkg._lib.lib()
    assert L.kvec_prefix_attention(C.byref(at(pkg, **bad)), 1 << 30, 1 << 30, None) == code
    assert word in L.kvec_last_error()
    assert L.kvec_prefix_attention_workspace(C.byref(at(pkg, **bad))) == -1


@pytest.mark.parametrize("bad,word", [
    ({"q": None}, b"null"),
    ({"prefix_pages": None}, b"null"),
    ({"seq_lens": None}, b"null"),
    ({"pool": (1 << 22) + 8}, b"aligned"),
    ({"q_stride": -1}, b"stride"),
    ({"o_head_stride": 32}, b"overlap"),
    ({"out": 1 << 20}, b"overlaps"),
    ({"out": 1 << 22}, b"overlaps"),
])
def test_attention_refuses_arrays(pkg, bad, word):
    L = pkg._lib.lib()
    assert L.kvec_prefix_attention(C.byref(at(pkg, **bad)), 1 << 30, 1 << 30, None) == -1
    assert word in L.kvec_last_error()


def test_attention_workspace(pkg):
    L = pkg._lib.lib()
    call = at(pkg)
    need = L.kvec_prefix_attention_workspace(C.byref(call))
    assert need >= 2 * 32 * (64 * 4 + 8)               # two parts of 32 rows at least
    for ws, n in ((None, need), (1 << 30, need - 1), ((1 << 30) + 8, need)):
        assert L.kvec_prefix_attention(C.byref(call), ws, n, None) == -1
        assert b"workspace" in L.kvec_last_error()
    assert L.kvec_prefix_attention_workspace(C.byref(at(pkg, tokens=0, batch=0))) == 0
    assert L.kvec_prefix_attention(C.byref(at(pkg, tokens=0, batch=0, q=None)), None, 0, None) == 0


@pytest.mark.parametrize("kw", [{}, {"prefix": 0}, {"heads": 64}, {"tokens": 300}, {"tokens": 300, "prefix": 0}])
def test_attention_longest_request(pkg, kw):
    """No request has more tokens than there are: a larger max_q splits the same."""
    L = pkg._lib.lib()
    call = at(pkg, cu_q=1 << 26, **kw)
    need = []
    for m in (call.tokens, call.tokens + 1, 1 << 24, (1 << 31) - 1):
        call.max_q = m
        need.append(L.kvec_prefix_attention_workspace(C.byref(call)))
    assert need[0] >= 0 and need == [need[0]] * 4


def test_attention_python_refusals(pkg):
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    q, pool = torch.zeros(4, 8, 64, dtype=torch.half), torch.zeros(1, 8, 16, 2, 2, 64, dtype=torch.half)
    with pytest.raises(ValueError, match="GPU"):
        pkg.attention.prefix_attention(q, pool, i(4, 3), i(4))
    with pytest.raises(ValueError, match="bfloat16 or float16"):
        pkg.attention.prefix_attention(q.float(), pool, i(4, 3), i(4))
    with pytest.raises(ValueError, match="seq_lens"):
        pkg.attention.prefix_attention(q, pool, i(4, 3), i(3))
    with pytest.raises(ValueError, match="one query token"):
        pkg.attention.prefix_attention(q[:3], pool, i(4, 3), i(4))
    with pytest.raises(ValueError, match="int32"):
        pkg.attention.prefix_attention(q, pool, i(4, 3).long(), i(4))


def test_packed_structs_are_the_structs(pkg):
    """struct.pack's bytes are the C layouts': every field at its place."""
    L = pkg._lib
    for fmt, cls in ((L.STEP_FORMAT, L.Step), (L.NORM_ROTATE_FORMAT, L.NormRotate), (L.ATTENTION_FORMAT, L.Attention)):
        vals = [float(i) + 0.5 if t is C.c_float else i + 1 for i, (_, t) in enumerate(cls._fields_)]
        raw = fmt.pack(*vals)
        got = cls.from_buffer_copy(raw.ljust(C.sizeof(cls), b"\0"))
        assert [getattr(got, n) for n, _ in cls._fields_] == vals
        assert len(raw) <= C.sizeof(cls) < len(raw) + 8


def test_paged_backend_shape_checks(pkg):
    serving = pkg.serving
    pool = torch.zeros(2, 6, 4, 2, 1, 8)
    be = serving.PagedBackend(pool, torch.zeros(1, 3, dtype=torch.int32), layer=1)
    assert be.kv_buffer.shape == (24, 2, 1, 8)
    assert be.kv_buffer.data_ptr() == pool[1].data_ptr()
    with pytest.raises(ValueError, match="layer"):
        serving.PagedBackend(pool, torch.zeros(1, 3, dtype=torch.int32), layer=2)
    with pytest.raises(ValueError, match="pool"):
        serving.PagedBackend(pool[0], torch.zeros(1, 3, dtype=torch.int32))
