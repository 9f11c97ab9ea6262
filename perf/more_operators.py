"""A paged K/V cache in 8 or 4 bits with block scales: written, read back and attended over, for timing.

A serving program that keeps its cache quantised runs these on a pool whose
token records are bytes, [layers, pages, page_tokens, 2 (K, V), half]: the half
holds kv_heads * head_dim codes (e4m3, or e2m1 two to a byte, the first in the
low half), then a byte for each block of 32 neighbouring values (the power of
two by which their codes are multiplied, plus 127), then zeros to 16 bytes.  The
scale of a block is the smallest power of two with which no value of it passes
the largest code.

  write    queries and keys normed by head and turned to their positions, K and
           V quantised into their slots, and the step's tokens read back
  read     tokens of the cache read back by slot, as when a request leaves
  attend   attention over the cache: new tokens, drafts, chunks of prompts, with
           and without a prefix that the requests share

Sizes are those of this package's tests and benchmark (32 query and 8 K/V heads
of 128, pages of 16 tokens, 16 requests of 2048 tokens, one of 32768) or
generic.  Page 0 is the pool's dummy page: no request holds it.

listed()         the named cases
draw(rng)        one more case of the same ranges
prepare(c, s)    what the program holds before the call, made from the seed
run(state)       one pass: plain torch operations, or (own) the package's calls
work(c)          bytes and operations that one pass cannot do without
exact(c, s)      the outputs in 64 bits
"""
import functools
import importlib
import math
import zlib

import numpy as np
import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
BLOCK = 32
EPS = 1e-6
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # The tokens of a decode step of sixteen requests.  Latency.
        {"name": "write_decode", "kind": "write", "tokens": 16, "heads": 32, "kv_heads": 8, "dim": 128,
         "rot": 128, "interleaved": False, "dtype": "bf16", "bits": 4, "page": 16},
        # A whole prefill step of 16 requests of 2048 tokens.
        {"name": "write_prefill", "kind": "write", "tokens": 32768, "heads": 32, "kv_heads": 8, "dim": 128,
         "rot": 128, "interleaved": False, "dtype": "bf16", "bits": 8, "page": 16},
        # Two ragged prompts, half of each head turned, in pairs of neighbours.
        {"name": "write_ragged", "kind": "write", "tokens": 3998, "heads": 32, "kv_heads": 4, "dim": 128,
         "rot": 64, "interleaved": True, "dtype": "fp16", "bits": 4, "page": 16},
        # A short request leaves for another engine.  Latency.
        {"name": "read_short", "kind": "read", "tokens": 500, "kv_heads": 8, "dim": 128, "dtype": "bf16",
         "bits": 4, "page": 16},
        # A long request, or a step's sixteen, read back whole.
        {"name": "read_long", "kind": "read", "tokens": 32768, "kv_heads": 8, "dim": 128, "dtype": "bf16",
         "bits": 8, "page": 16},
        # Smaller heads, an odd number of tokens, long pages.
        {"name": "read_ragged", "kind": "read", "tokens": 5001, "kv_heads": 4, "dim": 96, "dtype": "fp16",
         "bits": 4, "page": 32},
        # A few short requests decoding.  Latency.
        {"name": "attend_small", "kind": "attend", "batch": 4, "empty": 0, "heads": 32, "kv_heads": 8, "dim": 128,
         "prefix": 0, "cached": 576, "new": 1, "dtype": "bf16", "bits": 8, "page": 16},
        # Sixty-four ragged requests decoding, 8 bits.
        {"name": "attend_decode", "kind": "attend", "batch": 64, "empty": 0, "heads": 32, "kv_heads": 8,
         "dim": 128, "prefix": 0, "cached": 8192, "new": 1, "dtype": "bf16", "bits": 8, "page": 16},
        # Two hundred and fifty-six, 4 bits: what the smaller cache has room for.
        {"name": "attend_decode_4bit", "kind": "attend", "batch": 256, "empty": 0, "heads": 32, "kv_heads": 8,
         "dim": 128, "prefix": 0, "cached": 4096, "new": 1, "dtype": "bf16", "bits": 4, "page": 16},
        # One request with a very long history: the keys are all there is to share out.
        {"name": "attend_long", "kind": "attend", "batch": 1, "empty": 0, "heads": 32, "kv_heads": 8, "dim": 128,
         "prefix": 0, "cached": 262144, "new": 1, "dtype": "bf16", "bits": 4, "page": 16},
        # A padded batch that checks drafts of up to five tokens, behind a common prompt
        # that ends inside a page; smaller heads, some rows without a request.
        {"name": "attend_drafts", "kind": "attend", "batch": 24, "empty": 5, "heads": 8, "kv_heads": 8, "dim": 64,
         "prefix": 1003, "cached": 300, "new": 5, "dtype": "fp16", "bits": 4, "page": 16},
        # A prefill step of short questions behind a long common prompt.
        {"name": "attend_extend", "kind": "attend", "batch": 16, "empty": 0, "heads": 32, "kv_heads": 8,
         "dim": 128, "prefix": 4096, "cached": 0, "new": 128, "dtype": "bf16", "bits": 8, "page": 16},
    ]


# ------------------------------------------------------------------- drawing
def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(["write", "read", "attend", "attend"])
    c = {"kind": kind, "page": rng.choice([1, 8, 16, 16, 32, 64]), "bits": rng.choice([8, 4]),
         "dtype": rng.choice(["bf16", "bf16", "fp16"]), "kv_heads": rng.choice([1, 2, 4, 8]),
         "dim": rng.choice([64, 96, 128, 128, 128, 192, 256])}
    if kind == "read":
        c["tokens"] = _log(rng, 1, 32768 * 8 * 128 // (c["kv_heads"] * c["dim"]))
        return c
    c["heads"] = c["kv_heads"] * rng.choice([1, 2, 4, 4, 7, 8])
    if kind == "write":
        c["rot"] = rng.choice([c["dim"], c["dim"], c["dim"] // 2])
        c["interleaved"] = rng.random() < 0.3
        c["tokens"] = _log(rng, 1, 32768 * 48 * 128 // ((c["heads"] + 2 * c["kv_heads"]) * c["dim"]))
        return c
    c["new"] = rng.choice([1, 1, 1, rng.randint(2, 8), _log(rng, 8, 512)])
    c["batch"] = _log(rng, 1, 256 if c["new"] == 1 else max(1, min(64, 2048 // c["new"])))
    c["prefix"] = rng.choice([0, 0, _log(rng, 16, 8192)])
    # the keys and the products of the largest listed cases at most
    rows = c["batch"] * c["new"] * c["heads"] * c["dim"]
    c["prefix"] = min(c["prefix"], (2048 * 32 * 128 * 4096) // rows)
    held = min(256 * 4096 * 8 * 128 // (c["batch"] * c["kv_heads"] * c["dim"]), 2048 * 32 * 128 * 4096 // rows)
    c["cached"] = _log(rng, 1, max(1, min(32768, held)))
    if c["prefix"] and rng.random() < 0.3:
        c["cached"] = 0
    c["empty"] = rng.choice([0, 0, c["batch"] // 5])
    return c


# ------------------------------------------------------------------- lengths
def _lengths(c):
    """What the case's requests hold and their new tokens, as (cached, new): drawn from
    the case itself, so that the work is the case's; the seed only orders them."""
    r = np.random.RandomState(zlib.crc32(repr(sorted((k, v) for k, v in c.items() if k != "name")).encode()))
    B = c["batch"]
    cached = r.randint(0, c["cached"] + 1, B) if B > 1 else np.full(1, c["cached"])
    new = np.full(B, c["new"]) if c["cached"] == 0 or c["new"] == 1 else r.randint(1, c["new"] + 1, B)
    gone = np.arange(B) >= B - c["empty"]
    return np.where(gone, 0, cached), np.where(gone, 0 if c["new"] > 1 else 1, new)


def _ordered(c, seed):
    cached, new = _lengths(c)
    at = np.random.RandomState(int(seed) & 0x7FFFFFFF).permutation(len(new) - c["empty"])
    at = np.concatenate([at, np.arange(len(at), len(new))])     # rows without a request come last
    return cached[at], new[at]


def _half(c):
    """Bytes of a record's half: codes and scales of one token's K (or V)."""
    n = c["kv_heads"] * c["dim"]
    return (n * c["bits"] // 8 + n // BLOCK + 15) // 16 * 16


# ------------------------------------------------ codes and scales, in plain form
def _quantise(y, bits, dtype):
    """Records' halves [.., half] of values y [.., heads, dim] in 32 bits, which were computed from `dtype`."""
    lead = y.shape[:-2]
    blocks = y.reshape(*lead, -1, BLOCK)
    # a value that would round past the type's largest: as the last that does not
    most = {torch.float16: 2.0 ** 15, torch.bfloat16: 2.0 ** 127}[dtype] * (1.875 if bits == 8 else 1.5)
    raw = blocks.abs().amax(-1)
    blocks = blocks.clamp(-most, most)
    a = blocks.abs().amax(-1).view(torch.int32)
    top, part = (8, 0x600000) if bits == 8 else (2, 0x400000)      # 448 = 1.75 * 2^8, 6 = 1.5 * 2^2
    e = ((a >> 23) - 127 - top + ((a & 0x7FFFFF) > part)).clamp(min=-127)
    e = torch.where(a == 0, -127, e)
    x = blocks * ((127 - e) << 23).view(torch.float32)[..., None]       # 2^-e
    if bits == 8:
        code = x.to(torch.float8_e4m3fn).view(torch.uint8).flatten(-2)
    else:
        m = x.abs()
        n = (m > 0.25).to(torch.uint8)
        n = n + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5) + (m >= 3.5) + (m > 5.0)   # ties to even codes
        n = (n + 8 * torch.signbit(x)).flatten(-2).to(torch.uint8)
        code = n[..., 0::2] | (n[..., 1::2] << 4)
    scale = torch.where(torch.isfinite(raw), e + 127, 255).to(torch.uint8)
    out = torch.cat([code, scale], -1)
    return torch.nn.functional.pad(out, (0, -out.shape[-1] % 16))


def _values(half, c):
    """Values [.., kv_heads, dim] in 32 bits of records' halves [.., half]."""
    n = c["kv_heads"] * c["dim"]
    code, scale = half[..., : n * c["bits"] // 8], half[..., n * c["bits"] // 8:][..., : n // BLOCK].int()
    if c["bits"] == 8:
        v = code.contiguous().view(torch.float8_e4m3fn).float()
    else:
        e2m1 = torch.tensor(E2M1 + tuple(-x for x in E2M1), device=half.device)
        v = e2m1[torch.stack([code & 15, code >> 4], -1).flatten(-2).int()]
    power = torch.where(scale == 0, 0x400000, scale << 23).view(torch.float32)             # 2^(scale - 127)
    power = torch.where(scale == 255, math.nan, power)
    v = v.unflatten(-1, (-1, BLOCK)) * power[..., None]
    return v.reshape(*half.shape[:-1], c["kv_heads"], c["dim"])


# ----------------------------------------------------------------- preparing
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _dev(a, dtype=torch.int32):
    return torch.from_numpy(np.ascontiguousarray(a)).to("cuda", dtype)


def _randn(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda", dtype=DTYPES[dtype]) * scale).to(DTYPES[dtype])


def _pages(g, n):
    """Pages 1 .. n in no order (0 is the dummy)."""
    return (torch.randperm(n, generator=g, device="cuda") + 1).to(torch.int32)


def _pool(g, c, pages):
    """A pool of one layer that holds what a model's cache holds."""
    x = _randn(g, (1, pages, c["page"], 2, c["kv_heads"], c["dim"]), c["dtype"])
    return _quantise(x.float(), c["bits"], DTYPES[c["dtype"]])


def prepare(c, seed):
    g, kind = _gen(seed), c["kind"]
    st = {"case": c, "kind": kind}
    if kind != "attend":
        N, Hk, D, pt = c["tokens"], c["kv_heads"], c["dim"], c["page"]
        pages = -(-N // pt) + 4
        st["pool"] = _pool(g, c, pages + 1)
        ids = _pages(g, pages)[: -(-N // pt)].long()
        slots = (ids[:, None] * pt + torch.arange(pt, device="cuda")[None]).reshape(-1)[:N].to(torch.int32)
        # one token in a hundred has no slot (a request out of pages)
        st["slots"] = torch.where(torch.rand(N, generator=g, device="cuda") < 0.01, -1, slots).to(torch.int32)
        if kind == "read":
            return st
        st["qkv"] = _randn(g, (N, (c["heads"] + 2 * Hk) * D), c["dtype"])      # the projection's output
        st["positions"] = torch.randint(0, 131072, (N,), generator=g, device="cuda", dtype=torch.int32)
        half = c["rot"] // 2
        st["freqs"] = 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
        st["wq"] = (1 + 0.1 * torch.randn(D, generator=g, device="cuda")).to(DTYPES[c["dtype"]])
        st["wk"] = (1 + 0.1 * torch.randn(D, generator=g, device="cuda")).to(DTYPES[c["dtype"]])
        return st
    cached, new = _ordered(c, seed)
    B, Hq, D, pt, P = c["batch"], c["heads"], c["dim"], c["page"], c["prefix"]
    live = np.arange(B) < B - c["empty"]
    lens = np.where(live, P + cached + new, 0)
    width = max(1, int(-(-lens.max() // pt)))
    shared = P // pt                                       # whole pages of the prefix are the same for all
    need = np.maximum(0, -(-lens // pt) - shared)
    pages = shared + int(need.sum())
    ids = _pages(g, max(pages, 1))
    table = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    col = torch.arange(width, device="cuda")[None]
    dneed, dlive = _dev(need)[:, None], _dev(live, torch.bool)[:, None]
    table[(col >= shared) & (col < shared + dneed) & dlive] = ids[shared:pages]
    table = torch.where((col < shared) & dlive, torch.nn.functional.pad(ids[:shared], (0, width - shared))[None], table)
    pool = _pool(g, c, max(pages, 1) + 1)
    if P % pt:
        # the page in which the prefix ends is each request's own copy
        rows = table[: int(live.sum()), shared].long()
        pool[0, rows, : P % pt] = pool[0, rows[:1], : P % pt].clone()
    cu = np.concatenate([[0], np.cumsum(new)])
    st.update(pool=pool, table=table.contiguous(), lens=_dev(lens), cu=_dev(cu),
              q=_randn(g, (int(cu[-1]), Hq, D), c["dtype"], 1.5), max_q=int(new.max()),
              max_own=int(max(0, (lens - P).max())))
    return st


# ------------------------------------------------------------- plain operators
def _split(st):
    c = st["case"]
    N, Hq, Hk, D = c["tokens"], c["heads"], c["kv_heads"], c["dim"]
    x = st["qkv"].view(N, Hq + 2 * Hk, D)
    return x[:, :Hq], x[:, Hq:Hq + Hk], x[:, Hq + Hk:]


def _plain_read(st):
    c, slots = st["case"], st["slots"].long()
    half = st["pool"].view(-1, 2, st["pool"].shape[-1])[slots.clamp(min=0)]
    v = torch.where((slots >= 0)[:, None, None, None], _values(half, c), 0.0).to(DTYPES[c["dtype"]])
    return {"k": v[:, 0].contiguous(), "v": v[:, 1].contiguous()}


def _plain_write(st):
    c = st["case"]
    q, k, v = _split(st)
    half, rot = c["rot"] // 2, c["rot"]
    # far positions lose their angle in 32 bits
    angle = st["positions"].double()[:, None] * st["freqs"][None]
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]

    def turn(x, w, cos, sin):
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.to(x.dtype)
        if c["interleaved"]:
            a, b = x[..., 0:rot:2], x[..., 1:rot:2]
            y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
        else:
            a, b = x[..., :half], x[..., half:rot]
            y = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
        return torch.cat([y, x[..., rot:]], -1) if rot < c["dim"] else y

    q = turn(q.float(), st["wq"], cos.float(), sin.float()).to(q.dtype)
    # a code is a decision at a border: keys in 64 bits, rounded to 32 before it
    k = turn(k.double(), st["wk"], cos, sin).float()
    half = _quantise(torch.stack([k, v.float()], 1), c["bits"], v.dtype)
    flat, slots = st["pool"].view(-1, 2, half.shape[-1]), st["slots"].long()
    # tokens without a slot go to the dummy page's first slot as what it holds
    flat[slots.clamp(min=0)] = torch.where((slots >= 0)[:, None, None], half, flat[0])
    return {"q": q, **_plain_read(st)}


def _plain_attend(st):
    c = st["case"]
    B, Hq, Hk, D, pt, P = c["batch"], c["heads"], c["kv_heads"], c["dim"], c["page"], c["prefix"]
    G, M, S = Hq // Hk, st["max_q"], max(st["max_own"], 1)
    dev = st["q"].device
    table, lens, cu = st["table"].long(), st["lens"].long(), st["cu"].long()
    N = st["q"].shape[0]
    pool = st["pool"][0].view(-1, 2, st["pool"].shape[-1])
    q = st["q"].float().view(N, Hk, G, D) * (1 / math.sqrt(D))

    def keys(rows, pos, ok):
        """K and V [.., Hk, len, D] in 32 bits, zeros where there is no key."""
        page = rows.gather(1, (pos // pt).clamp(max=rows.shape[1] - 1).expand(rows.shape[0], -1))
        ok = ok & (page >= 0)
        kv = _values(pool[torch.where(ok, page * pt + pos % pt, 0)], c)
        kv = torch.where(ok[:, :, None, None, None], kv, 0.0)
        return kv[:, :, 0].transpose(1, 2).contiguous(), kv[:, :, 1].transpose(1, 2).contiguous(), ok

    n_new = cu[1:] - cu[:-1]
    t = torch.arange(N, device=dev)
    b = torch.searchsorted(cu[1:], t, right=True).clamp(max=B - 1)
    i = t - cu[b]
    limit = lens[b] - n_new[b] + i + 1                              # keys that a query sees

    def soften(s, ok, V):
        s = torch.where(ok, s, -math.inf)
        m = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
        return m, p.sum(-1, keepdim=True), p @ V

    # each request's own keys, for its queries padded to the most that one has
    at = torch.arange(M, device=dev)
    qi = (cu[:-1, None] + at).clamp(max=N - 1)
    qs = q[qi].permute(0, 2, 1, 3, 4).reshape(B, Hk, M * G, D)
    pos = P + torch.arange(S, device=dev)[None]
    K, V, ok = keys(table, pos, pos < lens[:, None])
    seen = ok[:, None, :] & (pos[:, None, :] < (lens - n_new)[:, None, None] + at[None, :, None] + 1)
    seen = seen[:, None, :, None, :].expand(B, 1, M, G, S).reshape(B, 1, M * G, S)
    m, l, o = soften(qs @ K.transpose(-1, -2).contiguous(), seen, V)
    m, l, o = (x.view(B, Hk, M, G, -1)[b, :, i] for x in (m, l, o))
    if P:
        # the prefix once for all queries
        pos = torch.arange(P, device=dev)[None]
        K, V, ok = keys(table[:1], pos, pos < P)
        qp = q.transpose(0, 1).reshape(Hk, N * G, D)
        seen = ok[0] & (pos[0] < limit[:, None])
        seen = seen[:, None].expand(N, G, P).reshape(1, N * G, P)
        m1, l1, o1 = soften(qp @ K[0].transpose(-1, -2).contiguous(), seen, V[0])
        m1, l1, o1 = (x.view(Hk, N, G, -1).transpose(0, 1) for x in (m1, l1, o1))
        top = torch.maximum(m, m1)
        top = torch.where(top == -math.inf, 0.0, top)
        f, f1 = torch.exp(m - top), torch.exp(m1 - top)
        l, o = l * f + l1 * f1, o * f + o1 * f1
    o = torch.where(l > 0, o / l, 0.0)
    return o.reshape(N, Hq, D).to(st["q"].dtype)


# ------------------------------------------------------------------- running
@functools.lru_cache(maxsize=1)
def _package():
    return importlib.import_module("26mlsys-ae-ghostserve_amd")


def run(st):
    c, kind = st["case"], st["kind"]
    if not own:
        return {"write": _plain_write, "read": _plain_read, "attend": _plain_attend}[kind](st)
    pkg = _package()
    pool = pkg.blockscale.BlockPool(st["pool"], c["kv_heads"], c["dim"], c["bits"])
    if kind == "attend":
        return pkg.attention.prefix_attention(
            st["q"], pool, st["table"], st["lens"], c["prefix"], cu_q=st["cu"] if c["new"] > 1 else None,
            max_q=st["max_q"], max_len=c["prefix"] + st["max_own"])
    out = {}
    if kind == "write":
        q, k, v = _split(st)
        out["q"] = pkg.attention.norm_rotate_write(
            q, k, v, st["positions"], st["freqs"], pool, st["slots"], q_weight=st["wq"], k_weight=st["wk"],
            eps=EPS, interleaved=c["interleaved"])
    out["k"], out["v"] = pkg.blockscale.read(pool, st["slots"], DTYPES[c["dtype"]])
    return out


# --------------------------------------------------------------- its own work
def work(c):
    Hk, D, es = c["kv_heads"], c["dim"], 2
    n = Hk * D
    token = 2 * (n * c["bits"] // 8 + n // BLOCK)            # codes and scales of a token
    if c["kind"] == "read":
        return {"bytes": c["tokens"] * (token + 2 * n * es + 4), "flops": 2 * n * c["tokens"]}
    if c["kind"] == "write":
        N, Hq = c["tokens"], c["heads"]
        # projections in, queries out, the records, and K and V as they read back
        b = N * ((2 * Hq + 4 * Hk) * D * es + token + 8) + 2 * D * es + 4 * c["rot"]
        return {"bytes": b, "flops": N * (8 * (Hq + Hk) * D + 4 * n)}
    cached, new = _lengths(c)
    Hq, P = c["heads"], c["prefix"]
    live = np.arange(c["batch"]) < c["batch"] - c["empty"]
    cached, new = cached[live].astype(np.int64), new[live].astype(np.int64)
    b = token * (P + int((cached + new).sum())) + 2 * es * Hq * D * int(new.sum())
    pairs = int((new * (P + cached) + new * (new + 1) // 2).sum())
    return {"bytes": b, "flops": 4 * Hq * D * pairs}


# ------------------------------------------------------------------ in 64 bits
def _power64(e):
    """2^e of whole numbers, exactly (torch's pow is off by a step for some)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _decode64(half, c):
    """Values [.., heads, dim] of records' halves by the formats' definitions."""
    n = c["kv_heads"] * c["dim"]
    if c["bits"] == 8:
        x = half[..., :n].long()
        e, m = (x >> 3) & 15, x & 7
        mag = torch.where(e == 0, m.double() / 512, (8 + m).double() * _power64(e - 10))
        v = torch.where(x >= 128, -mag, mag)
    else:
        x = half[..., : n // 2].long()
        x = torch.stack([x % 16, x // 16], -1).flatten(-2)
        e, m = (x >> 1) & 3, x & 1
        mag = torch.where(e == 0, m.double() / 2, (2 + m).double() * _power64(e - 2))
        v = torch.where(x >= 8, -mag, mag)
    power = _power64(half[..., n * c["bits"] // 8:][..., : n // BLOCK].long() - 127)
    return (v.unflatten(-1, (-1, BLOCK)) * power[..., None]).reshape(*half.shape[:-1], c["kv_heads"], c["dim"])


def _nearest64(y, bits):
    """Each value of y by the nearest one that its block's codes and scale stand for."""
    blocks = y.unflatten(-1, (-1, BLOCK))
    a = blocks.abs().amax(-1, keepdim=True)
    p, top, low = (3, 448.0, -6) if bits == 8 else (1, 6.0, 0)      # bits of a code's fraction; its exponents' least
    e = torch.ceil(torch.log2(a / top))
    e = torch.where(a > 0, e, 0.0)
    e = torch.where(a > top * _power64(e), e + 1, torch.where(a <= top * _power64(e - 1), e - 1, e)).clamp(min=-127)
    x = blocks / _power64(e)
    step = _power64(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** low))).clamp(min=low) - p)
    return ((x / step).round() * step * _power64(e)).flatten(-2)


def _exact_write(c, st):
    q, k, v = (x.double() for x in _split(st))
    half, rot = c["rot"] // 2, c["rot"]
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                       st["positions"].double()[:, None] * st["freqs"])
    order = np.arange(rot).reshape(half, 2) if c["interleaved"] else np.arange(rot).reshape(2, half).T
    order = torch.from_numpy(np.ascontiguousarray(order)).cuda()

    def apply(x, w):
        x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / c["dim"] + EPS) * w.double()
        z = torch.complex(x[..., order[:, 0]], x[..., order[:, 1]]) * turn[:, None]
        y = x.clone()
        y[..., order[:, 0]], y[..., order[:, 1]] = z.real, z.imag
        return y

    # the definition rounds a key to 32 bits before it is quantised
    k = _nearest64(apply(k, st["wk"]).float().double(), c["bits"])
    has = (st["slots"] >= 0)[:, None, None]
    return {"q": apply(q, st["wq"]), "k": torch.where(has, k, 0.0), "v": torch.where(has, _nearest64(v, c["bits"]), 0.0)}


def _exact_read(c, st):
    flat = st["pool"].view(-1, 2, st["pool"].shape[-1])
    v = torch.zeros((c["tokens"], 2, c["kv_heads"], c["dim"]), dtype=torch.float64, device="cuda")
    has = st["slots"] >= 0
    v[has] = _decode64(flat[st["slots"][has].long()], c)
    return {"k": v[:, 0], "v": v[:, 1]}


def _exact_attend(c, st):
    Hq, Hk, D, pt, P = c["heads"], c["kv_heads"], c["dim"], c["page"], c["prefix"]
    G = Hq // Hk
    table, lens, cu = st["table"].cpu().numpy(), st["lens"].tolist(), st["cu"].tolist()
    flat = st["pool"][0].view(-1, 2, st["pool"].shape[-1])

    def rows(b, lo, hi):
        """K and V [heads, keys, D] of positions lo .. hi - 1 of request b."""
        j = np.arange(lo, hi)
        kv = _decode64(flat[_dev(table[b][j // pt].astype(np.int64) * pt + j % pt, torch.long)], c)
        return kv[:, 0].transpose(0, 1), kv[:, 1].transpose(0, 1)

    out = torch.zeros((st["q"].shape[0], Hq, D), dtype=torch.float64, device="cuda")
    pre = rows(0, 0, P) if P else None
    for b, n in enumerate(lens):
        nq = cu[b + 1] - cu[b]
        if n == 0 or nq == 0:
            continue
        K, V = rows(b, P, n)
        if pre is not None:
            K, V = torch.cat([pre[0], K], 1), torch.cat([pre[1], V], 1)
        hidden = torch.arange(n, device="cuda")[None] > n - nq + torch.arange(nq, device="cuda")[:, None]
        for h in range(Hk):
            x = st["q"][cu[b]:cu[b + 1], h * G:(h + 1) * G].double().transpose(0, 1)
            s = (x @ K[h].t() / math.sqrt(D)).masked_fill(hidden, -math.inf)
            s = (s - s.amax(-1, keepdim=True)).exp()
            out[cu[b]:cu[b + 1], h * G:(h + 1) * G] = (s @ V[h] / s.sum(-1, keepdim=True)).transpose(0, 1)
    return out


def exact(c, seed):
    if c["kind"] == "attend" and work(c)["flops"] > 4e12:
        return None
    st = prepare(c, seed)
    return {"write": _exact_write, "read": _exact_read, "attend": _exact_attend}[c["kind"]](c, st)
