"""A serving step's operators together, as a program runs them: tables, cache
write and attention behind the hooked forward_extend, against one plain
64-bit model of the whole cache; the hook's parity of what they wrote; and
pages lost and rebuilt under them.

Tolerance: the reference attends over the pool's own (rounded) K and V with
queries rounded to the type, as the kernels do, so a result differs by what
attention alone may (u = eps/2: u |o| + A (u + 2^-13), A <= the largest |v|: sums
of up to 2^10 keys) and by queries that round to the other side (a step of
their type in a few values of 64: scores off by 2 u max|q k| scale at most, taken
as 4 u of A)."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


class Runner:
    def __init__(self, be):
        self.attn_backend = be


class Model:
    """The requests' whole histories, plainly kept: rotated keys, values."""

    def __init__(self, B, Hk, D, freqs, wq, wk):
        self.k = [torch.zeros(0, Hk, D, dtype=torch.float64) for _ in range(B)]
        self.v = [torch.zeros(0, Hk, D, dtype=torch.float64) for _ in range(B)]
        self.freqs, self.wq, self.wk = freqs, wq, wk

    def turn(self, x, pos, w):
        x = x.double()
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.double()
        a = pos.double()[:, None] * self.freqs[None]
        c, s = a.cos()[:, None], a.sin()[:, None]
        h = self.freqs.numel()
        y = torch.cat([x[..., :h] * c - x[..., h:] * s, x[..., :h] * s + x[..., h:] * c], -1)
        return y.to(BF).double()

    def extend(self, b, q, k, v):
        n0, n = self.k[b].shape[0], q.shape[0]
        pos = torch.arange(n0, n0 + n)
        q = self.turn(q, pos, self.wq)
        self.k[b] = torch.cat([self.k[b], self.turn(k, pos, self.wk)])
        self.v[b] = torch.cat([self.v[b], v.double()])
        G = q.shape[1] // k.shape[1]
        s = torch.einsum("qhd,khd->hqk", q, self.k[b].repeat_interleave(G, 1)) * q.shape[2] ** -0.5
        s = s.masked_fill(torch.arange(n0 + n)[None, None] > pos[None, :, None], -float("inf"))
        return torch.einsum("hqk,khd->qhd", s.softmax(-1), self.v[b].repeat_interleave(G, 1))


def setup(pkg, gpu, seed=0, B=5, Hq=8, Hk=2, D=64, P=16, prefix=32, pages=200, width=24):
    g = torch.Generator().manual_seed(seed)
    freqs = pkg.attention.rotary_frequencies(D, device="cpu")
    wq, wk = ((1 + 0.1 * torch.randn(D, generator=g)).to(BF) for _ in range(2))
    pool = torch.full((2, pages, P, 2, Hk, D), float("nan"), dtype=BF, device=gpu)
    table = torch.full((B, width), -1, dtype=torch.int32, device=gpu)
    be = pkg.serving.PagedBackend(pool, table, layer=1, prefix=prefix, freqs=freqs.to(gpu), q_weight=wq.to(gpu),
                                  k_weight=wk.to(gpu))
    model = Model(B, Hk, D, freqs, wq, wk)
    free = torch.randperm(pages, generator=g).to(torch.int32)
    return g, be, model, free, (B, Hq, Hk, D, P)


def tokens(g, n, Hq, Hk, D):
    return (torch.randn(n, h, D, generator=g).to(BF) for h in (Hq, Hk, Hk))


def near(got, want, what):
    u = 2.0 ** -8
    tol = u * want.abs() + (5 * u + 2.0 ** -13) * 4.5             # |v| of N(0, 1) in bf16 stays under 4.5
    off = (got.double() - want).abs()
    assert (off <= tol).all(), f"{what}: {float((off / tol).max())}"


def start_prefix(be, model, g, free, dims, prefix, gpu):
    """Request 0 prefills the shared prompt; the others' rows get its pages."""
    B, Hq, Hk, D, P = dims
    n = torch.zeros(B, dtype=torch.int32, device=gpu)
    new = n.clone()
    new[0] = prefix
    batch = be.begin(n, new, free.to(gpu), prefix, prefix)
    q, k, v = tokens(g, prefix, Hq, Hk, D)
    out = be.forward_extend(batch, q.to(gpu), k.to(gpu), v.to(gpu))
    near(out.cpu(), model.extend(0, q, k, v), "prefix")
    for b in range(1, B):
        model.k[b], model.v[b] = model.k[0].clone(), model.v[0].clone()
    be.page_table[1:, :prefix // P] = be.page_table[0, :prefix // P]
    return int(batch.taken)


@pytest.mark.parametrize("prefix", [32, 96])
def test_steps_with_parity(pkg, ora, gpu, tmp_path, prefix):
    g, be, model, free, dims = setup(pkg, gpu, seed=prefix, prefix=prefix)
    B, Hq, Hk, D, P = dims
    hook = pkg.serving.install(Runner(be), pkg.serving.KVParityHook(star_base=3, metrics_file=None, prog_start_mono=0.0),
                               on_error=lambda e: (_ for _ in ()).throw(e))
    at = start_prefix(be, model, g, free, dims, prefix, gpu)
    rng = np.random.default_rng(prefix)
    for step in range(7):
        new = rng.integers(0, 30, B) if step < 3 else np.ones(B, np.int64)
        if step == 5:
            new[2] = 0                                             # an idle row
        cached = [m.shape[0] for m in model.k]
        n, pad = int(new.sum()), 5
        d = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32, device=gpu)  # noqa: E731
        batch = be.begin(d(cached), d(new), free[at:].to(gpu), n + pad, max(1, int(new.max())))
        q, k, v = tokens(g, n + pad, Hq, Hk, D)
        out = be.forward_extend(batch, q.to(gpu), k.to(gpu), v.to(gpu)).cpu()
        hook.flush()
        at += int(batch.taken)
        t = 0
        for b in range(B):
            m = int(new[b])
            if m:
                near(out[t:t + m], model.extend(b, q[t:t + m], k[t:t + m], v[t:t + m]), f"step {step} request {b}")
            t += m
        assert (out[n:] == 0).all()
        # the parity of the step's slots, read back from the pool
        slots = batch.slot_mapping[batch.slot_mapping != -1].cpu().long()
        assert slots.numel() == n
        host = be.kv_buffer.cpu().view(torch.int16).numpy().view(np.uint16)
        row = np.concatenate([host[slots, 0].reshape(-1), host[slots, 1].reshape(-1)])
        rows = np.zeros((3, row.size), np.uint16)
        rows[0] = row
        ora.gs_parity(rows, 1, row.size, 3)
        got = [p.numpy().view(np.uint16) for p in hook.last_parity]
        assert np.array_equal(got[0], rows[1]) and np.array_equal(got[1], rows[2])
    assert not torch.isnan(be.kv_buffer[batch.slot_mapping[:n].long()].float()).any()
    assert torch.isnan(be.pool[0].float()).all(), "the other layer was written"


def test_lost_pages_come_back_the_same(pkg, gpu):
    """Pages coded, wiped and rebuilt: the next step's attention has the same bits."""
    prefix = 64
    g, be, model, free, dims = setup(pkg, gpu, seed=1, prefix=prefix)
    B, Hq, Hk, D, P = dims
    at = start_prefix(be, model, g, free, dims, prefix, gpu)
    d = lambda a: torch.tensor(a, dtype=torch.int32, device=gpu)  # noqa: E731
    n = 64
    batch = be.begin(d([prefix] * B), d([n] * B), free[at:].to(gpu), n * B, n)
    q, k, v = tokens(g, n * B, Hq, Hk, D)
    be.forward_extend(batch, q.to(gpu), k.to(gpu), v.to(gpu))
    at += int(batch.taken)
    step = be.begin(d([prefix + n] * B), d([1] * B), free[at:].to(gpu), B, 1)
    q, k, v = (x.to(gpu) for x in tokens(g, B, Hq, Hk, D))
    want = be.forward_extend(step, q, k, v)
    # the layer's own-token pages of all requests as one chunk (whole pages), RDP over p = 7
    layer = be.pool[1:2]
    kv = pkg.paged.PagedKV(layer, be.page_table, prefix, n)
    R = pkg.paged.rdp_row_bytes_for(kv, 6, 7)
    mk = lambda: torch.empty(6 * R, dtype=torch.uint8, device=gpu)  # noqa: E731
    data, P_, Q_ = [mk() for _ in range(6)], mk(), mk()
    pkg.paged.rdp_encode_paged(kv, data, P_, Q_, p=7, row_bytes=R)
    before = layer.clone()
    stream = kv.gather()
    for e in (1, 4):
        stream[e * 6 * R:(e + 1) * 6 * R].fill_(0xFF)
        data[e].fill_(0xFF)
    kv.scatter(stream)
    assert not torch.equal(layer.view(torch.int16), before.view(torch.int16))
    pkg.paged.rdp_decode_paged(kv, P_, Q_, erased=[1, 4], k=6, p=7, row_bytes=R)
    assert torch.equal(layer.view(torch.int16), before.view(torch.int16))
    again = pkg.attention.prefix_attention(
        pkg.attention.norm_rotate_write(q, k, v, step.positions, be.freqs, be.pool, step.slot_mapping, layer=1, **be.norm),
        be.pool, be.page_table, step.seq_lens, prefix, layer=1, cu_q=step.cu_new, max_q=1, max_len=step.max_len)
    assert torch.equal(again, want)


def test_whole_step_captured(pkg, gpu):
    """Tables, write and attention in one graph, replayed as requests grow, with
    eager steps of other requests between the replays."""
    prefix = 32
    g, be, model, free, dims = setup(pkg, gpu, seed=2, prefix=prefix)
    B, Hq, Hk, D, P = dims
    at = start_prefix(be, model, g, free, dims, prefix, gpu)
    cached = torch.full((B,), prefix, dtype=torch.int32, device=gpu)
    new = torch.ones(B, dtype=torch.int32, device=gpu)
    pages = free.to(gpu).clone()
    bufs = [x.to(gpu) for x in tokens(g, B, Hq, Hk, D)]
    pages[:free.numel() - at] = free[at:].to(gpu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    table0 = be.page_table.clone()
    with torch.cuda.stream(side):
        be.forward_extend(be.begin(cached, new, pages, B, 1), *bufs)
    torch.cuda.current_stream().wait_stream(side)
    be.page_table.copy_(table0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        batch = be.begin(cached, new, pages, B, 1)
        out = be.forward_extend(batch, *bufs)
    for i in range(20):
        q, k, v = tokens(g, B, Hq, Hk, D)
        for dst, src in zip(bufs, (q, k, v)):
            dst.copy_(src)
        pages[:free.numel() - at] = free[at:].to(gpu)
        cached.fill_(prefix + i)
        graph.replay()
        torch.cuda.synchronize()
        for b in range(B):
            near(out[b:b + 1].cpu(), model.extend(b, q[b:b + 1], k[b:b + 1], v[b:b + 1]), f"replay {i} request {b}")
        at += int(batch.taken)


def test_fp8_pool(pkg, gpu):
    """K and V held in 8 bits with scales: written and read by the same ones."""
    g = torch.Generator().manual_seed(4)
    B, Hq, Hk, D, P, n = 3, 8, 2, 64, 16, 40
    ks, vs = (torch.tensor([x], device=gpu) for x in (0.02, 0.015))
    pool = torch.zeros(1, 40, P, 2, Hk, D, device=gpu).to(torch.float8_e4m3fn)
    table = torch.full((B, 6), -1, dtype=torch.int32, device=gpu)
    be = pkg.serving.PagedBackend(pool, table, freqs=pkg.attention.rotary_frequencies(D, device=gpu), k_scale=ks, v_scale=vs)
    d = lambda a: torch.tensor(a, dtype=torch.int32, device=gpu)  # noqa: E731
    batch = be.begin(d([0] * B), d([n] * B), torch.randperm(40, generator=g).to(torch.int32).to(gpu), n * B, n)
    q, k, v = (x.to(gpu) for x in tokens(g, n * B, Hq, Hk, D))
    out = be.forward_extend(batch, q, k, v)
    turned = pkg.attention.norm_rotate_write(q, k, v, batch.positions, be.freqs, pool, batch.slot_mapping, k_scale=ks,
                                             v_scale=vs).double().cpu()
    kv = be.kv_buffer[batch.slot_mapping.long()].double().cpu()
    for b in range(B):
        r = slice(b * n, (b + 1) * n)
        K, V = kv[r, 0] * float(ks), kv[r, 1] * float(vs)
        s = torch.einsum("qhd,khd->hqk", turned[r], K.repeat_interleave(4, 1)) * D ** -0.5
        s = s.masked_fill(torch.arange(n)[None, None] > torch.arange(n)[None, :, None], -float("inf"))
        near(out[r].cpu(), torch.einsum("hqk,khd->qhd", s.softmax(-1), V.repeat_interleave(4, 1)), f"request {b}")
    # the values are within half a step of the 8-bit type of what was written
    err = (kv[:, 1] * float(vs) - v.double().cpu()).abs()
    assert (err <= v.double().cpu().abs() * 2.0 ** -4 * 1.01 + float(vs) * 2.0 ** -10).all()


def test_first_request_leaves(pkg, gpu):
    """The request whose row the prefix came from ends, and its row is emptied: with
    the prefix's pages given on their own the others still see them."""
    prefix = 48
    g, be, model, free, dims = setup(pkg, gpu, seed=6, prefix=prefix)
    B, Hq, Hk, D, P = dims
    at = start_prefix(be, model, g, free, dims, prefix, gpu)
    be.prefix_pages = be.page_table[0, :prefix // P].clone()
    d = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32, device=gpu)  # noqa: E731
    for new in ([0, 1, 1, 1, 1], [0, 20, 0, 3, 7]):
        cached = [0] + [m.shape[0] for m in model.k[1:]]
        n = sum(new)
        batch = be.begin(d(cached), d(new), free[at:].to(gpu), n, max(new))
        q, k, v = tokens(g, n, Hq, Hk, D)
        out = be.forward_extend(batch, q.to(gpu), k.to(gpu), v.to(gpu)).cpu()
        at += int(batch.taken)
        assert (be.page_table[0] == -1).all()
        t = 0
        for b in range(B):
            if new[b]:
                r = slice(t, t + new[b])
                near(out[r], model.extend(b, q[r], k[r], v[r]), f"request {b}")
            t += new[b]
