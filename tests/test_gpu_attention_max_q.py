"""A request with more tokens than max_q: its tokens from max_q on are left as they
were, and everything else is as it would be."""
import pytest
import torch

from test_gpu_prefix_attention import BF, check, make, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("prefix", [0, 48, 600])
@pytest.mark.parametrize("new,max_q", [
    ([5, 2, 1, 9], 2), ([1, 7, 0, 1], 1), ([3, 3, 3, 3], 1),               # stream blocks
    ([100, 64, 300, 7], 64), ([300, 10, 64, 200], 64), ([40, 3, 129, 1], 33),  # tile blocks
    ([5, 9, 2, 1], 4), ([70] * 80, 3),
])
@pytest.mark.parametrize("cached", [30, 2500])
def test_more_than_max_q(pkg, gpu, new, max_q, prefix, cached):
    if len(new) > 10 and cached > 30:
        cached = 300
    lens = [prefix + cached + n for n in new]
    c = make(gpu, 41, lens, new, 8, 2, 64, BF, BF, 16, prefix)
    o, tol = reference(c)
    out = torch.full_like(c["q"], 3.0)
    pkg.attention.prefix_attention(c["q"], c["pool"], c["table"], c["lens"], prefix, layer=1, cu_q=c["cu"], out=out,
                                   max_q=max_q)
    at = torch.cat([torch.arange(n) for n in new]).to(gpu)
    check(out[at < max_q], (o[at < max_q], tol[at < max_q]))
    assert (out[at >= max_q] == 3.0).all()


@pytest.mark.parametrize("cached", [30, 2500])
def test_lengths_grow_under_a_graph(pkg, gpu, cached):
    """A captured call whose requests come to differ from what it was captured for."""
    new = [20, 20, 20, 20]
    c = make(gpu, 42, [cached + 80] * 4, new, 8, 2, 64, BF, BF, 16, 0)
    out = torch.empty_like(c["q"])

    def call():
        pkg.attention.prefix_attention(c["q"], c["pool"], c["table"], c["lens"], 0, layer=1, cu_q=c["cu"], out=out,
                                       max_q=20)

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for now in ([20, 20, 20, 20], [50, 10, 20, 0], [0, 80, 0, 0], [10, 20, 30, 20]):
        ends = torch.tensor([0] + now).cumsum(0).to(torch.int32)
        c["cu"].copy_(ends)
        o, tol = reference(c)
        for eager in (False, True):
            out.fill_(3.0)
            call() if eager else graph.replay()
            torch.cuda.synchronize()
            at = torch.cat([torch.arange(n) for n in now]).to(gpu)
            check(out[at < 20], (o[at < 20], tol[at < 20]))
            assert (out[at >= 20] == 3.0).all()


@pytest.mark.parametrize("B", [64, 65, 130, 5000])
def test_many_requests(pkg, gpu, B):
    """Requests enough that a row's is looked for in one, two and three steps, idle
    ones among them, joined from parts."""
    new = [(1, 0, 2, 1, 3)[i * 7 % 5] for i in range(B)]
    c = make(gpu, 43, [64 + 1 + n for n in new], new, 2, 1, 64, BF, BF, 16, 64)
    o, tol = reference(c)
    out = torch.full_like(c["q"], 3.0)
    pkg.attention.prefix_attention(c["q"], c["pool"], c["table"], c["lens"], 64, layer=1, cu_q=c["cu"], out=out, max_q=2)
    at = torch.cat([torch.arange(n) for n in new]).to(gpu)
    check(out[at < 2], (o[at < 2], tol[at < 2]))
    assert (out[at >= 2] == 3.0).all()
