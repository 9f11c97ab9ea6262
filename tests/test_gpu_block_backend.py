"""Steps of a serving program on a cache with block scales: tables, write, attention, the
hook's parity over the records, pages lost and rebuilt, tokens read back."""
import numpy as np
import pytest
import torch

import blockref as ref
from test_gpu_norm_rotate import rotate64

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


class Server:
    """Requests that grow, beside what their tokens' K and V are by definition."""

    def __init__(self, pkg, gpu, bits, dtype, Hq=8, Hk=2, D=64, B=4, P=8, pages=96, prefix=0):
        self.pkg, self.gpu, self.bits, self.dtype, self.P, self.Hq, self.Hk, self.D = pkg, gpu, bits, dtype, P, Hq, Hk, D
        self.g = torch.Generator().manual_seed(bits + prefix)
        self.pool = pkg.blockscale.BlockPool.zeros(2, pages, P, Hk, D, bits, device=gpu)
        self.table = torch.full((B, pages // 2), -1, dtype=torch.int32, device=gpu)
        self.freqs = pkg.attention.rotary_frequencies(D, device=gpu)
        self.wq, self.wk = ((1 + 0.1 * torch.randn(D, generator=self.g)).to(dtype).to(gpu) for _ in range(2))
        self.free = (torch.randperm(pages - 1, generator=self.g) + 1).to(torch.int32).to(gpu)
        self.cached = np.zeros(B, dtype=np.int64)
        self.kv = [[] for _ in range(B)]                     # per request: K and V as written, in 64 bits
        self.backend = pkg.serving.PagedBackend(self.pool, self.table, layer=1, prefix=prefix, freqs=self.freqs,
                                                q_weight=self.wq, k_weight=self.wk)

    def step(self, new, pad=3):
        N = int(sum(new)) + pad
        shape = (N, self.Hq + 2 * self.Hk, self.D)
        x = torch.randn(shape, generator=self.g).to(self.dtype).to(self.gpu)
        q, k, v = x[:, :self.Hq], x[:, self.Hq:self.Hq + self.Hk], x[:, self.Hq + self.Hk:]
        dev = lambda a: torch.tensor(list(a), dtype=torch.int32, device=self.gpu)  # noqa: E731
        batch = self.backend.begin(dev(self.cached), dev(new), self.free, N, max(new))
        out = self.backend.forward_extend(batch=batch, q=q, k=k, v=v)
        self.free = self.free[int(batch.taken):]
        # by definition
        pos = batch.positions.cpu()
        rot = lambda t, w: rotate64(t.cpu(), pos, self.freqs.cpu(), None, False, 1.0, w.cpu(), 1e-6, True)  # noqa: E731
        qr = rot(q, self.wq)[0]
        kr = rot(k, self.wk)[0].float()
        at = 0
        for b, n in enumerate(new):
            for i in range(n):
                halves = []
                for y in (kr[at + i], v[at + i].float().cpu()):
                    c, s = ref.quantise(y.reshape(-1), self.bits, self.dtype)
                    halves.append(torch.cat([ref.pack(c, self.bits), s]))
                self.kv[b].append(ref.values(torch.stack(halves), self.Hk, self.D, self.bits))
            at += n
        self.cached += np.array(new)
        return batch, qr[: sum(new)], out

    def check(self, batch, qr, out, new):
        """The step's output by the formulas over what the requests hold."""
        rounded = qr.to(self.dtype)                          # as the write leaves the queries: within a step of each
        G, n0 = self.Hq // self.Hk, 0
        u = torch.finfo(self.dtype).eps / 2
        for b, n in enumerate(new):
            if not n:
                continue
            kv = torch.stack(self.kv[b])                     # [keys, 2, Hk, D]
            total = kv.shape[0]
            see = torch.arange(total)[None] <= total - n + torch.arange(n)[:, None]
            for h in range(self.Hq):
                K, V = kv[:, 0, h // G], kv[:, 1, h // G]
                qq = rounded[n0:n0 + n, h].double()
                s = (qq @ K.t()) * self.D ** -0.5
                s = s.masked_fill(~see, -np.inf)
                p = torch.exp(s - s.amax(1, keepdim=True))
                p = p / p.sum(1, keepdim=True)
                want = p @ V
                got = out[n0:n0 + n, h].double().cpu()
                # a query value may be a step beside (2 u of it): the scores move by up to 2 u sum
                # |q||k| / sqrt(D) either way, every weight by that relative to itself; the weights'
                # and the output's own roundings add 2 u
                move = 2 * u * ((qq.abs() @ K.abs().t()) * self.D ** -0.5).masked_fill(~see, 0).amax(1, keepdim=True)
                A = p @ V.abs()
                tol = A * (2 * torch.expm1(2 * move) + 2.5 * u) + u * want.abs() + 1e-6
                assert ((got - want).abs() <= tol).all(), float(((got - want).abs() / tol).max())
            n0 += n
        assert not out[n0:].any()


@pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "fp16"])
@pytest.mark.parametrize("bits", [8, 4])
def test_steps_with_parity(pkg, gpu, bits, dtype, tmp_path):
    """Prefill, decode, drafts; the hook codes each step's records; a lost slot is found in the parity."""
    s = Server(pkg, gpu, bits, dtype)
    hook = pkg.serving.install(type("R", (), {"attn_backend": s.backend})(), pkg.serving.KVParityHook(metrics_file=str(tmp_path / "m.jsonl")))
    for i, new in enumerate(([40, 7, 0, 1], [1, 1, 33, 1], [1, 1, 1, 1], [5, 2, 1, 3], [1, 0, 1, 1], [90, 1, 1, 12])):
        batch, qr, out = s.step(new)
        s.check(batch, qr, out, new)
        hook.flush()
        assert hook.counter.count == i + 1
        # one rank: P is the step's records themselves, K then V, as 2-byte words
        slots = batch.slot_mapping[batch.slot_mapping >= 0].long()
        words = s.backend.kv_buffer[slots]                   # [n, 2, 1, words]
        row = torch.cat([words[:, 0].reshape(-1), words[:, 1].reshape(-1)]).cpu()
        assert torch.equal(hook.last_parity[0].view(torch.int16)[: row.numel()], row)
    # and what the records hold is what was written, read back by slot
    for b in range(4):
        n = int(s.cached[b])
        pos = torch.arange(n, device=gpu)
        slots = (s.table[b, pos // s.P] * s.P + pos % s.P).to(torch.int32)
        k, v = pkg.blockscale.read(s.pool, slots, dtype, layer=1)
        want = torch.stack(s.kv[b]).to(dtype)
        assert torch.equal(k.cpu(), want[:, 0]) and torch.equal(v.cpu(), want[:, 1])


@pytest.mark.parametrize("bits", [8, 4])
def test_records_lost_and_rebuilt(pkg, gpu, bits):
    """Two shards of the records' stream erased, rebuilt into the pool, byte for byte; attention as before."""
    s = Server(pkg, gpu, bits, BF, Hq=8, Hk=4, D=128, P=16, pages=64)
    new = [64, 64, 64, 64]
    batch, qr, out = s.step(new, pad=0)
    s.check(batch, qr, out, new)
    kv = pkg.paged.PagedKV(s.pool, s.table[:, :4].contiguous(), 0, 64)
    assert kv.token_bytes == ref.half_bytes(4, 128, bits)
    k, p = 6, 7
    R = pkg.paged.rdp_row_bytes_for(kv, k, p)
    data = [torch.zeros((p - 1) * R, dtype=torch.uint8, device=gpu) for _ in range(k)]
    P, Q = torch.zeros_like(data[0]), torch.zeros_like(data[0])
    pkg.paged.rdp_encode_paged(kv, data, P, Q, p, R)
    was = s.pool.data.clone()
    stream = kv.gather()
    size = (p - 1) * R
    whole = torch.cat(data)
    for e in (1, 4):
        data[e].fill_(0xA5)
    broken = stream.clone()
    for e in (1, 4):
        broken[e * size:(e + 1) * size] = 0xFF
    kv.scatter(broken)
    assert not torch.equal(s.pool.data, was)
    pkg.paged.rdp_decode_paged(kv, P, Q, [1, 4], k, p, R, data=data)
    assert torch.equal(s.pool.data, was) and torch.equal(torch.cat(data), whole)


def test_a_step_in_a_graph(pkg, gpu):
    """A decode step over a pool of 4 bits, captured; replayed it does as eager calls do."""
    s = Server(pkg, gpu, 4, BF, Hq=16, Hk=4, D=128, P=16, pages=128)
    s.step([100, 3, 47, 16], pad=0)
    B = 4
    cached = torch.tensor(s.cached, dtype=torch.int32, device=gpu)
    new = torch.ones(B, dtype=torch.int32, device=gpu)
    x = torch.randn(B, 24, 128, generator=s.g).to(BF).to(gpu)

    def step():
        batch = s.backend.begin(cached, new, s.free, B, 1)
        return s.backend.forward_extend(batch, x[:, :16], x[:, 16:20], x[:, 20:])

    table, data = s.table.clone(), s.pool.data.clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = step()
    torch.cuda.current_stream().wait_stream(stream)
    for seed in range(3):
        x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(seed)))
        s.table.copy_(table), s.pool.data.copy_(data)
        graph.replay()
        got, bytes_ = out.clone(), s.pool.data.clone()
        s.table.copy_(table), s.pool.data.copy_(data)
        assert torch.equal(step(), got) and torch.equal(s.pool.data, bytes_)


def test_shared_prefix(pkg, gpu):
    """Requests behind a prefix on pages of its own, in one call with it and without."""
    s = Server(pkg, gpu, 8, BF, B=3, P=8)
    s.step([40, 0, 0], pad=0)                                # the prefix: 40 tokens of request 0
    front = s.table[0, :5].clone()
    s.table[1, :5], s.table[2, :5] = front, front
    s.kv[1], s.kv[2] = list(s.kv[0]), list(s.kv[0])
    s.cached[:] = 40
    s.backend = pkg.serving.PagedBackend(s.pool, s.table, layer=1, prefix=40, prefix_pages=front, freqs=s.freqs,
                                         q_weight=s.wq, k_weight=s.wk)
    for new in ([1, 1, 1], [3, 1, 20], [1, 1, 1]):
        batch, qr, out = s.step(new)
        s.check(batch, qr, out, new)


def test_two_streams_at_once(pkg, gpu):
    """Two calls on two streams, each with its own workspace, on one pool."""
    s = Server(pkg, gpu, 4, BF, Hq=8, Hk=2, D=128, P=16, pages=256)
    s.step([1000, 700, 3, 500], pad=0)
    lens = torch.tensor(s.cached, dtype=torch.int32, device=gpu)
    qs = [torch.randn(4, 8, 128, generator=s.g).to(BF).to(gpu) for _ in range(2)]
    alone = [pkg.attention.prefix_attention(q, s.pool, s.table, lens, layer=1) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [None, None]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                outs[i] = pkg.attention.prefix_attention(qs[i], s.pool, s.table, lens, layer=1)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(alone, outs))
