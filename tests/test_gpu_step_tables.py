"""Page tables and slots of a step against a plain loop over the requests."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

INT_MAX = 2**31 - 1


def reference(table, cached, new, free, pool_pages, P, T):
    """One request, one page and one token at a time."""
    table = table.copy()
    B, W = table.shape
    slots, pos = np.full(T, -1, np.int64), np.zeros(T, np.int64)
    cu, lens, at, t = [0], [], 0, 0
    for b in range(B):
        c, n = max(int(cached[b]), 0), max(int(new[b]), 0)
        held, end = min(-(-c // P), W), min(-(-min(c + n, INT_MAX) // P), W)
        for j in range(held, W):
            if j < end:
                table[b, j] = free[at] if at < len(free) else -1
                at += 1
            else:
                table[b, j] = -1
        for i in range(min(n, max(T - t, 0))):
            p = min(c + i, INT_MAX)                            # the positions are 32-bit
            pos[t + i] = p
            page = table[b, p // P] if p // P < W else -1
            if 0 <= page < pool_pages:
                slots[t + i] = page * P + p % P
        t += n
        cu.append(min(t, INT_MAX))
        lens.append(min(c + n, INT_MAX))
    return table, slots, pos, cu, lens, at


def run(pkg, gpu, table, cached, new, free, pool_pages, P, T, out=None):
    d = lambda a: torch.from_numpy(np.asarray(a, np.int32).copy()).to(gpu)  # noqa: E731
    tab = d(table)
    st = pkg.paged.step_tables(tab, d(cached), d(new), d(free), pool_pages, P, T, out=out)
    return tab, st


def check(got, want):
    tab, st = got
    names = ("table", "slots", "positions", "cu_new", "seq_lens", "taken")
    for name, g, w in zip(names, (tab,) + tuple(st), want):
        same = np.array_equal(g.cpu().numpy().reshape(-1), np.asarray(w, np.int64).reshape(-1))
        assert same, name


def make(rng, B, W, P, max_new, decode=0.5, idle=0.1, junk=True):
    room = W * P
    new = np.where(rng.random(B) < decode, 1, rng.integers(0, max_new + 1, B))
    cached = rng.integers(0, max(room - max_new, 0) + 1, B)
    quiet = rng.random(B) < idle
    cached, new = np.where(quiet, 0, cached), np.where(quiet, 0, new)
    held = -(-cached // P)
    pages = int((-(-(cached + new) // P)).sum()) + 5
    ids = rng.permutation(pages) + 1
    table = rng.integers(-5, pages + 9, (B, W)) if junk else np.full((B, W), -1)
    at = 0
    for b in range(B):
        table[b, :held[b]] = ids[at:at + held[b]]
        at += held[b]
    return table.astype(np.int32), cached, new, ids[at:], pages + 1


@pytest.mark.parametrize("B,W,P,max_new", [
    (1, 1, 1, 1), (1, 7, 16, 40), (3, 5, 4, 9), (16, 128, 16, 1), (17, 33, 8, 100), (255, 12, 16, 60),
    (256, 3, 1, 3), (257, 64, 32, 500), (1024, 40, 16, 64), (1025, 9, 2, 8), (2500, 31, 4, 20), (2, 9000, 1, 2000),
])
def test_tables_match(pkg, gpu, B, W, P, max_new):
    rng = np.random.default_rng(B * 1000 + W)
    table, cached, new, free, pool_pages = make(rng, B, W, P, max_new)
    T = int(new.sum()) + 37
    check(run(pkg, gpu, table, cached, new, free, pool_pages, P, T),
          reference(table, cached, new, free, pool_pages, P, T))


def test_tables_edges(pkg, gpu):
    """Lists that run out, requests past their row, too little room for the
    tokens, negative and huge lengths, entries outside the pool."""
    rng = np.random.default_rng(7)
    table, cached, new, free, pages = make(rng, 20, 8, 4, 12)
    T = int(new.sum())
    cases = [
        (table, cached, new, free[:3], pages, T),                # the list is too short
        (table, cached, new, free[:0], pages, T),                # and empty
        (table, cached, new + 40, free, pages, T + 900),         # past the row
        (table, cached + 100, new, free, pages, T),              # held past the row
        (table, cached, new, free, pages, T // 2),               # no room for all tokens
        (table, cached, new, free, pages, 0),                    # none at all
        (table, cached, new, free, 9, T),                        # pages outside the pool
        (table, cached, new, free, 0, T),
        (table, cached - 20, new - 5, free, pages, T),           # negative lengths
        (table, np.full(20, INT_MAX - 3), new + 9, free, pages, T + 180),
        (table, cached, np.full(20, INT_MAX), free, pages, 64),  # sums stay at 2^31 - 1
    ]
    for tab, c, n, f, pp, t in cases:
        if n[0] == INT_MAX:
            got = run(pkg, gpu, tab, c, n, f, pp, 4, t)[1]
            assert got.cu_new.tolist() == [0] + [INT_MAX] * 20
            assert got.seq_lens.tolist() == [INT_MAX] * 20
            continue
        check(run(pkg, gpu, tab, c, n, f, pp, 4, t), reference(tab, c, n, f, pp, 4, t))


def test_no_requests(pkg, gpu):
    tab, st = run(pkg, gpu, np.zeros((0, 4)), np.zeros(0), np.zeros(0), np.arange(3), 8, 16, 5)
    assert st.slots.tolist() == [-1] * 5 and st.positions.tolist() == [0] * 5
    assert st.cu_new.tolist() == [0] and st.taken.tolist() == [0]


def test_twice_is_once(pkg, gpu):
    """The same step again finds its own entries behind what the requests hold."""
    rng = np.random.default_rng(3)
    table, cached, new, free, pages = make(rng, 50, 16, 16, 90)
    d = lambda a: torch.from_numpy(np.asarray(a, np.int32)).to(gpu)  # noqa: E731
    tab, args = d(table), (d(cached), d(new), d(free), pages, 16, int(new.sum()) + 3)
    first = pkg.paged.step_tables(tab, *args)
    want = [x.clone() for x in (tab,) + tuple(first)]
    again = pkg.paged.step_tables(tab, *args, out=first)
    assert again is first
    assert all(torch.equal(a, b) for a, b in zip(want, (tab,) + tuple(again)))


def test_steps_follow(pkg, gpu):
    """Steps one after another: what a step takes, the next one holds."""
    rng = np.random.default_rng(11)
    B, W, P, pages = 9, 20, 8, 400
    free = rng.permutation(pages)
    table, cached, at = np.full((B, W), -1, np.int32), np.zeros(B, np.int64), 0
    seen = {}
    for step in range(12):
        new = rng.integers(0, 14, B)
        tab, st = run(pkg, gpu, table, cached, new, free[at:], pages, P, int(new.sum()))
        slots, pos = st.slots.tolist(), st.positions.tolist()
        t = 0
        for b in range(B):
            for i in range(int(new[b])):
                assert slots[t] >= 0 and pos[t] == cached[b] + i
                assert slots[t] not in seen
                seen[slots[t]] = (b, pos[t])
                t += 1
        at += int(st.taken)
        table, cached = tab.cpu().numpy(), cached + new
    # every slot that was given out is where the table says the token lies
    for s, (b, p) in seen.items():
        assert table[b, p // P] * P + p % P == s


def test_captured(pkg, gpu):
    """Replayed on new lengths, each replay gives the eager call's tables."""
    rng = np.random.default_rng(5)
    B, W, P, T = 40, 32, 16, 4096
    sets = [make(rng, B, W, P, 90, junk=False) for _ in range(4)]
    F, pages = max(len(s[3]) for s in sets), max(s[4] for s in sets)
    d = lambda a: torch.from_numpy(np.asarray(a, np.int32)).to(gpu)  # noqa: E731
    pad = lambda f: np.concatenate([f, np.full(F - len(f), -1)])  # noqa: E731
    tab, c, n, f = d(sets[0][0]), d(sets[0][1]), d(sets[0][2]), d(pad(sets[0][3]))
    pkg.paged.step_tables(tab, c, n, f, pages, P, T)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        st = pkg.paged.step_tables(tab, c, n, f, pages, P, T)
    for s in sets:
        for dst, src in zip((tab, c, n, f), (s[0], s[1], s[2], pad(s[3]))):
            dst.copy_(d(src))
        graph.replay()
        torch.cuda.synchronize()
        check((tab, st), reference(s[0], s[1], s[2], pad(s[3]), pages, P, T))


def test_other_stream(pkg, gpu):
    rng = np.random.default_rng(9)
    table, cached, new, free, pages = make(rng, 64, 16, 16, 50)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = run(pkg, gpu, table, cached, new, free, pages, 16, int(new.sum()))
    side.synchronize()
    check(got, reference(table, cached, new, free, pages, 16, int(new.sum())))
