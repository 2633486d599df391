"""kv_cache_copy and kv_cache_fork: whole pages, bit for bit, and the books of a host."""

import random

import pytest
import torch

from paged_ops_helpers import fork_books

pytestmark = pytest.mark.gpu

E4, E5, BF, FH = torch.float8_e4m3fn, torch.float8_e5m2, torch.bfloat16, torch.float16


def _ops():
    import primus_turbo.pytorch as turbo

    return turbo.ops


def _pools(L, P, H, page, D, dtype, ranges=False, seed=0):
    """Pools of random bits (L = 0: without a dimension of layers)."""
    g = torch.Generator("cuda").manual_seed(seed)
    lead = (L,) if L else ()

    def bits(*shape, to):
        n = torch.empty((), dtype=to).element_size()
        return torch.randint(0, 256, (*lead, *shape[:-1], shape[-1] * n), generator=g, dtype=torch.uint8, device="cuda").view(to)

    out = [bits(P, H, page, D, to=dtype) for _ in range(2)]
    out += [bits(P, H, page, to=torch.float32) for _ in range(2)] if dtype in (E4, E5) else [None, None]
    return out + [bits(P, H, 2, D, to=BF) if ranges else None]


def _bytes(t):
    return None if t is None else t.view(torch.uint8)


def _moved(pools, pairs, layers):
    """The pools with pages copied, in host memory."""
    out = []
    for t in pools:
        if t is None:
            out.append(None)
            continue
        x = _bytes(t).cpu()
        y = x.clone()
        for s, d in pairs:
            if layers:
                y[:, d] = x[:, s]
            else:
                y[d] = x[s]
        out.append(y)
    return out


def _same(pools, want):
    return all(a is None or torch.equal(_bytes(a).cpu(), b) for a, b in zip(pools, want))


@pytest.mark.parametrize("L,P,H,page,D,dtype,ranges", [
    (0, 9, 2, 16, 64, E4, False), (0, 40, 1, 7, 16, E5, True), (3, 21, 3, 5, 48, E4, True), (2, 12, 8, 64, 128, E4, False),
    (0, 30, 4, 1, 80, BF, False), (5, 8, 2, 33, 256, FH, True), (1, 700, 1, 1, 16, E4, True)])
@pytest.mark.parametrize("idx", [torch.int32, torch.int64])
def test_copy(L, P, H, page, D, dtype, ranges, idx):
    r = random.Random(P * page)
    order = r.sample(range(P), P)
    n = P // 2
    pairs = list(zip(order[:n], order[n:2 * n]))
    if n > 2:
        pairs[1] = (pairs[0][0], pairs[1][1])  # one source twice
        pairs[2] = (pairs[2][0], pairs[2][0])  # onto itself
    pools = _pools(L, P, H, page, D, dtype, ranges)
    want = _moved(pools, pairs, L)
    src, dst = ([p[i] for p in pairs] for i in (0, 1))
    # pages that the pool has not
    src += [-1, P, order[0], order[0]]
    dst += [order[-1], order[-1], P, -5]
    if idx == torch.int64:
        src, dst = src + [2 ** 40, order[0]], dst + [order[-1], -(2 ** 40)]
    src, dst = (torch.tensor(x, dtype=idx, device="cuda") for x in (src, dst))
    _ops().kv_cache_copy(pools[0], pools[1], src, dst, pools[2], pools[3], key_ranges=pools[4])
    assert _same(pools, want)


@pytest.mark.parametrize("L,P,H,page,D,n", [(2, 300, 8, 64, 128, 100), (3, 90, 5, 33, 80, 40), (2, 2600, 8, 64, 128, 1100)])
def test_copy_much(L, P, H, page, D, n):
    """More than one piece a thread; more than the last cache holds."""
    pools = _pools(L, P, H, page, D, E4, ranges=True)
    start = [t.clone() for t in pools]
    order = torch.randperm(P, generator=torch.Generator().manual_seed(P)).cuda()
    src, dst = order[:n].contiguous(), order[n:2 * n].contiguous()
    _ops().kv_cache_copy(pools[0], pools[1], src, dst, pools[2], pools[3], key_ranges=pools[4])
    for x, y in zip(pools, start):
        x, y = _bytes(x), _bytes(y)
        y[:, dst] = y[:, src]
        assert torch.equal(x, y)


def test_copy_nothing():
    ops = _ops()
    pools = _pools(0, 4, 2, 8, 32, E4)
    want = _moved(pools, [], 0)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    ops.kv_cache_copy(pools[0], pools[1], none, none, pools[2], pools[3])
    assert _same(pools, want)
    e = _pools(0, 0, 2, 8, 32, E4)
    one = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.kv_cache_copy(e[0], e[1], one, one, e[2], e[3])
    e = [t.new_zeros((0, 4, *t.shape[1:])) if t is not None else None for t in pools]
    ops.kv_cache_copy(e[0], e[1], one, one, e[2], e[3])


def test_copy_offsets_past_32_bits():
    P, H, page, D = 4200, 8, 512, 256  # 4.4e9 bytes a pool
    kc, vc = (torch.zeros((P, H, page, D), dtype=torch.uint8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros((P, H, page), device="cuda") for _ in range(2))
    for i, t in enumerate((kc, vc, ks, vs)):
        t[P - 1] = 17 + i
        t[3] = 40 + i
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    _ops().kv_cache_copy(kc.view(E4), vc.view(E4), i32(P - 1, 3), i32(1, P - 2), ks, vs)
    for i, t in enumerate((kc, vc, ks, vs)):
        assert bool((t[1] == 17 + i).all()) and bool((t[P - 2] == 40 + i).all())
        assert not bool(t[0].any()) and not bool(t[2].any()) and not bool(t[P - 3].any())


def _case(r, B, N, M, page, P, wild):
    """Tables of sequences that share pages as forks leave them; with `wild`, anything."""
    free = r.sample(range(P), P)
    table, lens = [], []
    for b in range(B):
        n = min(r.choice((0, 1, page, r.randint(0, M * page))), M * page)
        row = []
        if b and r.random() < 0.6:
            other = r.randrange(b)
            row = table[other][:min(lens[other], n) // page]
        need = -(-n // page) - len(row)
        if need > len(free):
            n, row, need = 0, [], 0
        row = row + [free.pop() for _ in range(need)]
        table.append(row + [-1] * (M - len(row)))
        lens.append(n)
    parents = [r.randrange(B) if B else 0 for _ in range(N)]
    if wild:
        for row in table:
            for j in range(M):
                if r.random() < 0.2:
                    row[j] = r.choice((-1, P, -7, 2 ** 31 - 1, r.randrange(P)))
        lens = [r.choice((n, n, -3, M * page + 5, 2 ** 31 - 1)) for n in lens]
        parents = [r.choice((p, p, p, -1, B, 2 ** 31 - 1)) for p in parents]
    return table, lens, parents


@pytest.mark.parametrize("compact", [False, True])
@pytest.mark.parametrize("wild", [False, True])
@pytest.mark.parametrize("B,N,M,page,P,reserve", [(1, 1, 1, 1, 1, 0), (1, 5, 3, 4, 20, 0), (4, 4, 6, 3, 40, 1), (6, 9, 5, 8, 70, 20),
                                                  (8, 40, 7, 2, 60, 3), (30, 11, 9, 5, 300, 0), (3, 0, 4, 4, 10, 2), (40, 40, 3, 16, 130, 33)])
def test_fork(B, N, M, page, P, reserve, wild, compact):
    ops = _ops()
    for seed in range(4):
        r = random.Random(1000 * seed + B + N + P)
        table, lens, parents = _case(r, B, N, M, page, P, wild)
        layers = seed % 3
        pools = _pools(layers, P, 2, page, 16, (E4, BF)[seed % 2], ranges=seed > 1, seed=seed)
        rows, new_lens, pairs = fork_books(table, lens, parents, page, P, reserve, compact)
        want = _moved(pools, pairs, layers)
        t = torch.tensor(table, dtype=torch.int32).view(B, M)
        if seed == 1:  # rows of a wider table
            t = torch.cat((t, torch.full((B, 3), 5, dtype=torch.int32)), dim=1)
        t = t.cuda()[:, :M]
        got = ops.kv_cache_fork(pools[0], pools[1], t, torch.tensor(lens, dtype=torch.int32).cuda(),
                                torch.tensor(parents, dtype=(torch.int32, torch.int64)[seed % 2]).cuda(), pools[2], pools[3],
                                key_ranges=pools[4], reserve=reserve, compact=compact)
        assert got[0].tolist() == rows and got[1].tolist() == new_lens, f"seed {seed}"
        assert torch.equal(t.cpu(), torch.tensor(table, dtype=torch.int32).view(B, M)), "the old table is left as it is"
        # what no sequence has may hold anything, and holds what it did
        assert _same(pools, want), f"seed {seed}"


@pytest.mark.parametrize("compact", [False, True])
@pytest.mark.parametrize("B,N,M,page,P,reserve", [(40, 60, 300, 2, 12 * 1024, 3), (40, 60, 300, 2, 12 * 1024 + 1, 3), (70, 70, 900, 1, 50021, 0),
                                                  (300, 900, 160, 2, 9000, 5)])
def test_fork_of_large_pools(B, N, M, page, P, reserve, compact):
    """As many pages as one workgroup's LDS has owners for, and more; more entries than it goes through."""
    r = random.Random(P + N)
    table, lens, parents = _case(r, B, N, M, page, P, False)
    rows, new_lens, pairs = fork_books(table, lens, parents, page, P, reserve, compact)
    pools = _pools(0, P, 1, page, 16, E4, seed=P)
    want = _moved(pools, pairs, 0)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    got = _ops().kv_cache_fork(pools[0], pools[1], i32(table), i32(lens), i32(parents), pools[2], pools[3], reserve=reserve, compact=compact)
    assert torch.equal(got[0].cpu(), torch.tensor(rows, dtype=torch.int32)) and got[1].tolist() == new_lens
    # fresh pages hold whatever they held: all pages are compared, since copies alone write
    assert _same(pools, want)


@pytest.mark.parametrize("compact", [False, True])
def test_fork_of_many(compact):
    """More sequences and pages than one workgroup has threads."""
    ops = _ops()
    r = random.Random(3)
    B, N, M, page, P = 1500, 2100, 4, 2, 9000
    table, lens, parents = _case(r, B, N, M, page, P, False)
    pools = _pools(0, P, 1, page, 16, E4)
    rows, new_lens, pairs = fork_books(table, lens, parents, page, P, 1, compact)
    want = _moved(pools, pairs, 0)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    got = ops.kv_cache_fork(pools[0], pools[1], i32(table), i32(lens), i32(parents), pools[2], pools[3], reserve=1, compact=compact)
    assert got[0].tolist() == rows and got[1].tolist() == new_lens and _same(pools, want)


def test_fork_of_one_long_sequence():
    """A table row of many pages, shared by all."""
    ops = _ops()
    P, M, page = 5000, 4500, 3
    order = random.Random(1).sample(range(P), P)
    table, lens, parents = [order[:M]], [M * page - 1], [0] * 7
    pools = _pools(0, P, 1, page, 16, BF)
    for compact in (False, True):
        rows, new_lens, pairs = fork_books(table, lens, parents, page, P, 4, compact)
        want = _moved(pools, pairs, 0)
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        got = ops.kv_cache_fork(pools[0], pools[1], i32(table), i32(lens), i32(parents), reserve=4, compact=compact)
        assert got[0].tolist() == rows and got[1].tolist() == new_lens and _same(pools, want)


def test_fork_without_parents_sequences_or_pages():
    ops = _ops()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    pools = _pools(0, 10, 2, 4, 16, E4)
    table, lens = i32([7, 2, -1], [9, 3, -1]), i32(6, 3)
    got = ops.kv_cache_fork(pools[0], pools[1], table, lens, None, pools[2], pools[3], reserve=3)
    assert got[0].tolist() == [[7, 2, 0], [9, 1, -1]] and got[1].tolist() == [6, 3]
    got = ops.kv_cache_fork(pools[0], pools[1], table, lens, i32(), pools[2], pools[3])
    assert got[0].shape == (0, 3) and got[1].shape == (0,)
    none = torch.empty((0, 3), dtype=torch.int32, device="cuda")
    got = ops.kv_cache_fork(pools[0], pools[1], none, i32(), i32(0, 5), pools[2], pools[3], reserve=2)
    assert got[0].tolist() == [[-1] * 3] * 2 and got[1].tolist() == [0, 0]
    e = _pools(0, 0, 2, 4, 16, E4)
    got = ops.kv_cache_fork(e[0], e[1], table, lens, None, e[2], e[3], reserve=0)
    assert got[0].tolist() == [[7, 2, -1], [9, -1, -1]] and got[1].tolist() == [6, 3]  # pages outside the pool stay
    got = ops.kv_cache_fork(pools[0], pools[1], table[:, :0], lens, None, pools[2], pools[3], reserve=9)
    assert got[0].shape == (2, 0) and got[1].tolist() == [6, 3]


def test_fork_of_a_sequence_without_pages():
    """Pages run out for one sequence; what goes on from it gets none either, and takes none from the others."""
    ops = _ops()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    pools = _pools(0, 3, 2, 4, 16, BF)
    table, lens = ops.kv_cache_fork(pools[0], pools[1], i32([0, -1], [1, -1]), i32(2, 2), i32(0, 0, 1, 1))
    assert table.tolist() == [[0, -1], [2, -1], [1, -1], [-1, -1]] and lens.tolist() == [2, 2, 2, -1]
    for compact in (False, True):
        got = ops.kv_cache_fork(pools[0], pools[1], table, lens, i32(3, 0), reserve=6, compact=compact)
        assert got[0].tolist() == [[-1, -1], [0, 1]] and got[1].tolist() == [-1, 2]


def test_fork_other_stream_and_captured():
    ops = _ops()
    r = random.Random(8)
    B, N, M, page, P = 12, 16, 5, 4, 120
    pools = _pools(2, P, 2, page, 32, E4, ranges=True)
    start = [None if t is None else t.clone() for t in pools]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    cases = [_case(r, B, N, M, page, P, False) for _ in range(5)]
    table, lens, parents = (i32(x) for x in cases[0])

    def call(p):
        return ops.kv_cache_fork(p[0], p[1], table, lens, parents, p[2], p[3], key_ranges=p[4], reserve=2, compact=True)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = call(pools)
    torch.cuda.current_stream().wait_stream(s)
    rows, new_lens, pairs = fork_books(*cases[0], page, P, 2, True)
    assert got[0].tolist() == rows and got[1].tolist() == new_lens and _same(pools, _moved(start, pairs, 2))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call(pools)
    for case in cases[1:]:
        for t, x in zip((table, lens, parents), case):
            t.copy_(i32(x))
        for t, x in zip(pools, start):
            t.view(torch.uint8).copy_(x.view(torch.uint8))
        graph.replay()
        torch.cuda.synchronize()
        rows, new_lens, pairs = fork_books(*case, page, P, 2, True)
        assert held[0].tolist() == rows and held[1].tolist() == new_lens and _same(pools, _moved(start, pairs, 2))
