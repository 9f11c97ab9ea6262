"""How stream blocks over a cache with block scales share out keys: by the lengths that the requests
have, whatever max_len says.  A part of the workspace that holds keys has a maximum."""
import ctypes as C

import pytest
import torch

from test_gpu_block_attention import BF, case, check, run
from test_gpu_prefix_attention import reference

pytestmark = pytest.mark.gpu


def parts_with_keys(pkg, c, width, max_len):
    """(parts of each request's rows that hold keys, the call's output); the workspace: [parts][rows][dim]
    outputs, then [parts][rows] maxima and sums."""
    q, pool = c["q"], c["records"]
    N, Hq, D = q.shape
    table = torch.full((len(c["new"]), width), -1, dtype=torch.int32, device=q.device)
    table[:, :c["table"].shape[1]] = c["table"]
    out = torch.empty_like(q)
    base, _ = pool.layer(1)
    s = pkg._lib.Attention(
        tokens=N, batch=len(c["new"]), heads=Hq, kv_heads=pool.kv_heads, dim=D, dtype=1, q=q.data_ptr(), q_stride=Hq * D,
        q_head_stride=D, out=out.data_ptr(), o_stride=Hq * D, o_head_stride=D, pool=base, pool_dtype=pool.code,
        pool_pages=pool.shape[1], page_tokens=pool.shape[2], page_table=table.data_ptr(), pages_per_seq=width,
        seq_lens=c["lens"].data_ptr(), cu_q=None, max_q=1, max_len=max_len, prefix=0, prefix_pages=None, scale=D ** -0.5)
    lib = pkg._lib.lib()
    need = lib.kvec_prefix_attention_workspace(C.byref(s))
    rows = N * Hq
    parts = (need - 16) // (rows * (D * 4 + 8))
    ws = torch.empty(need, dtype=torch.uint8, device=q.device)
    pkg._lib.call("kvec_prefix_attention", C.byref(s), ws.data_ptr(), need, pkg._lib.stream_handle(q.device))
    tops = ws[parts * rows * D * 4:][:parts * rows * 8].view(torch.float32).view(parts, N, Hq, 2)[..., 0]
    return (tops != -float("inf")).sum(0).amin(-1).tolist(), out


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("lens,keys", [([4096], 262144), ([4096, 4000, 4090, 4096], 131072), ([4096, 1, 300, 64, 2000], 65536)])
@pytest.mark.parametrize("hint", [0, 1 << 16])
def test_short_requests_in_a_long_table(pkg, gpu, bits, lens, keys, hint):
    """A table, or a hint, of 16 to 64 times the longest request: the keys still go to many blocks."""
    B = len(lens)
    c = case(pkg, gpu, B, lens, [1] * B, 32, 8, 64, BF, bits, 16)
    parts, out = parts_with_keys(pkg, c, keys // 16, hint)
    check(out, reference(c))
    # 64 keys a run at least, and no more than twice that where parts are enough
    for n, p in zip(lens, parts):
        assert -(-n // 128) <= p <= -(-n // 64), (n, p)


@pytest.mark.parametrize("bits", [8, 4])
def test_many_requests_in_a_long_table(pkg, gpu, bits):
    """More requests than a wave's lanes: the longest one is found wherever it is; all keys are covered."""
    B = 300
    for at in (0, 63, 64, 255, 256, 299):
        lens = [40] * B
        lens[at] = 1500
        c = case(pkg, gpu, at, lens, [1] * B, 2, 1, 64, BF, bits, 16)
        want = reference(c)
        for max_len in (None, 1500, 65536):
            check(run(pkg, c, max_len=max_len), want)
        parts, out = parts_with_keys(pkg, c, 4096, 0)
        check(out, want)
        assert parts[at] >= 16 and max(parts[:at] + parts[at + 1:]) <= 4


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("prefix", [0, 45, 500])
def test_behind_a_prefix_in_a_long_table(pkg, gpu, bits, prefix):
    """Own keys behind a prefix, some requests with none, one idle; drafts and single tokens."""
    for new in ([1] * 6, [2, 1, 2, 0, 1, 2]):
        own = [900, 0, 2500, 0, 31, 32]
        lens = [prefix + o + n if n else 0 for o, n in zip(own, new)]
        c = case(pkg, gpu, prefix + sum(new), lens, new, 8, 4, 64, BF, bits, 16, prefix, width=8192)
        want = reference(c)
        for max_len in (None, max(lens), 1, 1 << 30):
            check(run(pkg, c, max_q=max(new), max_len=max_len), want)


@pytest.mark.parametrize("bits", [8, 4])
def test_a_graph_of_a_long_table(pkg, gpu, bits):
    """Captured once for the table's width, replayed on lengths from one key to thousands."""
    top = [6000, 300, 2000]
    c = case(pkg, gpu, bits, top, [1] * 3, 8, 2, 64, BF, bits, 16, width=16384)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run(pkg, c)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = run(pkg, c)
    torch.cuda.current_stream().wait_stream(s)
    for lens in ([1, 1, 1], [6000, 1, 0], [100, 300, 2000], top, [64, 65, 63]):
        c["lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        got = out.clone()
        assert torch.equal(got, run(pkg, c))
        check(got, reference(c))
