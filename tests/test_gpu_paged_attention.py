"""paged_attention against the plain 64-bit attention of serving_helpers, element
by element within the bounds of the kernels' arithmetic."""

import pytest
import torch

from serving_helpers import FP8_MAX, attention, within

pytestmark = pytest.mark.gpu

E4, E5, BF, FH = torch.float8_e4m3fn, torch.float8_e5m2, torch.bfloat16, torch.float16


def _ops():
    import primus_turbo.pytorch as turbo

    return turbo.ops


def make(new, lens, Hq, Hkv, D, page, cache, dtype, seed=0, spare=2, spread=0.0):
    """q, pools with scales, table, cu, lens (CPU): pages in random order, what no key needs holds NaN."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-max(n, 0) // page) for n in lens]
    P, M = sum(need) + spare, max(need + [1])
    order = torch.randperm(P, generator=g).to(torch.int32)
    table = torch.full((len(lens), M), -1, dtype=torch.int32)
    pools, scales = [], []
    for _ in range(2):
        x = torch.randn(P, Hkv, page, D, generator=g) * torch.exp(spread * torch.randn(P, Hkv, page, 1, generator=g))
        if cache in FP8_MAX:
            s = x.abs().amax(-1) / FP8_MAX[cache]
            pools.append((x / s[..., None]).clamp(-FP8_MAX[cache], FP8_MAX[cache]).to(cache))
            scales.append(s)
        else:
            pools.append(x.to(cache))
            scales.append(None)
    used = torch.zeros(P, page, dtype=torch.bool)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        for j in range(n):
            used[order[at + j], :min(page, lens[b] - j * page)] = True
        at += n
    for x, s in zip(pools, scales):
        bad = ~used[:, None, :].expand(P, Hkv, page)
        raw = x.view(torch.uint8) if cache in FP8_MAX else x
        raw[bad] = 0x7F if cache in FP8_MAX else float("nan")
        if s is not None:
            s[bad] = float("nan")
    cu = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32)
    q = torch.randn(sum(new), Hq, D, generator=g).to(dtype)
    return q, pools, scales, table, cu, torch.tensor(lens, dtype=torch.int32)


def check(case, window=None, sinks=0, scale=None):
    q, (kc, vc), (ks, vs), table, cu, lens = case
    dev = [None if t is None else t.cuda() for t in (q, kc, vc, table, cu, lens, ks, vs)]
    out, lse = _ops().paged_attention(*dev, window_size=window, num_sinks=sinks, softmax_scale=scale, return_lse=True)
    clean = [None if s is None else torch.nan_to_num(s) for s in (ks, vs)]
    want, wlse, b_out, b_lse = attention(q, *(torch.nan_to_num(c.float()).to(torch.float64) for c in (kc, vc)), *clean, table,
                                         cu, lens, q.shape[2] ** -0.5 if scale is None else scale, window, sinks)
    assert out.dtype == q.dtype and out.shape == q.shape and lse.dtype == torch.float32
    within(out, want, b_out, "out")
    within(lse, wlse, b_lse, "lse")
    again = _ops().paged_attention(*dev, window_size=window, num_sinks=sinks, softmax_scale=scale)
    assert torch.equal(again.view(torch.int16), out.view(torch.int16)), "two calls differ"
    return out, lse


KINDS = [(E4, BF), (E4, FH), (E5, BF), (E5, FH), (BF, BF), (FH, FH)]


@pytest.mark.parametrize("cache,dtype", KINDS)
@pytest.mark.parametrize("D", [16, 48, 64, 80, 128, 192, 256])
@pytest.mark.parametrize("kind", ["decode", "chunk"])
def test_types_and_head_sizes(cache, dtype, D, kind):
    new, lens = ([1, 1, 1], [1, 70, 333]) if kind == "decode" else ([70, 1, 130], [70, 129, 300])
    check(make(new, lens, 4, 2, D, 16, cache, dtype, seed=D))


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (3, 1), (7, 7), (8, 1), (20, 4), (64, 2)])
@pytest.mark.parametrize("new,lens", [([1, 1], [5, 200]), ([40, 3], [40, 90])])
def test_head_layouts(Hq, Hkv, new, lens):
    check(make(new, lens, Hq, Hkv, 64, 32, E4, BF, seed=Hq))


@pytest.mark.parametrize("page", [1, 7, 16, 48, 64, 100, 512])
@pytest.mark.parametrize("new", [[1, 1, 1, 1], [33, 1, 64, 65]])
def test_page_sizes(page, new):
    check(make(new, [33, 127, 128, 257], 4, 2, 64, page, E4, BF, seed=page))


@pytest.mark.parametrize("kind", ["decode", "chunk"])
@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257])
def test_lengths_at_the_tiles_edges(kind, length):
    new = [1] if kind == "decode" else [length]
    check(make(new, [length], 8, 2, 64, 16, E4, BF, seed=length))
    if kind == "chunk":
        check(make([max(1, length // 2)], [length], 2, 2, 128, 16, BF, BF, seed=length))


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 0), (64, 4), (100, 130), (63, 64), (1000, 4)])
@pytest.mark.parametrize("new,lens", [([1, 1, 1], [1, 150, 400]), ([64, 200, 1], [64, 390, 77])])
@pytest.mark.parametrize("cache", [E4, BF])
def test_window_and_sinks(window, sinks, new, lens, cache):
    check(make(new, lens, 4, 2, 64, 16, cache, BF, seed=window), window, sinks)


def test_empty_sequences_and_rows_without_keys():
    """Lengths of zero, sequences without new tokens, more new tokens than the length
    says (the first see nothing), a page table without columns."""
    for n in (1, 40):
        out, lse = check(make([n, 0, n, 1, 0], [0, 50, 5 if n > 5 else 1, 9, 0], 4, 2, 64, 16, E4, BF))
        assert not bool(out[:n].any()) and bool((lse[:n] == float("-inf")).all())
    q, pools, scales, table, cu, lens = make([2, 1], [0, 0], 4, 2, 64, 16, E4, BF)
    out, lse = check((q, pools, scales, table[:, :0], cu, lens + 7))
    assert not bool(out.any()) and bool((lse == float("-inf")).all())


def test_lengths_past_the_table_and_pages_outside_the_pool():
    q, pools, scales, table, cu, lens = make([1, 20], [60, 64], 4, 2, 64, 16, E4, BF, spare=0)
    lens = torch.tensor([1 << 30, 64], dtype=torch.int32)  # the table ends at 64 tokens
    table[0, 3] = table[0, 0]
    check((q, pools, scales, table, cu, lens))
    table[1, 1], table[1, 2] = 10 ** 6, -5  # read as zeros
    check((q, pools, scales, table, cu, lens))


@pytest.mark.parametrize("cache,dtype", [(E4, BF), (E4, FH), (E5, FH)])
def test_scales_over_many_binades(cache, dtype):
    """Rows whose scales differ by factors of thousands; tiny values in fp16."""
    for n, L in ((1, 300), (90, 300)):
        case = make([n], [L], 4, 2, 64, 16, cache, dtype, spread=2.5)
        check(case, scale=0.02)
        q, pools, (ks, vs), *rest = case
        check((q, pools, (ks, vs * 1e-6), *rest), scale=0.02)
        check((q, pools, (ks, vs * 0), *rest), scale=0.02)


def test_large_logits():
    """One key far above the others; logits of hundreds."""
    case = make([1, 50], [200, 180], 2, 1, 64, 16, BF, BF)
    check(case, scale=8.0)


@pytest.mark.parametrize("cache,dtype", KINDS)
@pytest.mark.parametrize("n,D,window,sinks", [(8, 64, None, 0), (8, 128, 30, 2), (10, 64, None, 0), (10, 128, 30, 2), (150, 64, None, 0), (150, 128, 40, 3), (100, 256, None, 0)])
def test_infinities_and_nan_reach_the_rows_that_see_them(cache, dtype, n, D, window, sinks):
    """Values and a key that are NaN or infinite: rows that do not see the token keep
    their finite results, the others get what the formula gives."""
    L = 2 * n + 60
    q, (kc, vc), (ks, vs), table, cu, lens = make([n, 1], [L, 5], 4, 2, D, 16, cache, dtype, seed=n)
    inf = torch.tensor(float("-inf"))

    def put(pool, j, d, x):
        pool[int(table[0, j // 16]), :, j % 16, d] = x

    nan = torch.tensor(float("nan")).to(cache)
    put(vc, L - n // 2, 3, nan)
    put(vc, L - n // 3, D - 1, nan if cache == E4 else inf.to(cache))
    put(vc, L - n // 4, 8, nan if cache == E4 else (-inf).to(cache))
    put(kc, L - 2, 9, nan)
    put(vc, 1, 5, nan)  # seen as a sink, or until the window has passed it
    dev = [t if t is None else t.cuda() for t in (q, kc, vc, table, cu, lens, ks, vs)]
    got = _ops().paged_attention(*dev, window_size=window, num_sinks=sinks).cpu().double()
    args = (table, cu, lens, D ** -0.5, window, sinks)
    raw = attention(q, kc.double(), vc.double(), ks, vs, *args)[0]
    zero = lambda c: torch.nan_to_num(c.double(), 0.0, 0.0, 0.0)  # noqa: E731
    want, _, bound, _ = attention(q, zero(kc), zero(vc), *(s if s is None else torch.nan_to_num(s) for s in (ks, vs)), *args)
    fin = torch.isfinite(raw)
    assert bool((~fin).any()) and torch.equal(torch.isnan(got), torch.isnan(raw))
    assert torch.equal(got[torch.isinf(raw)], raw[torch.isinf(raw)])
    within(torch.where(fin, got, 0.0), torch.where(fin, want, 0.0), bound, "finite results")


@pytest.mark.parametrize("cache", [E4, BF])
@pytest.mark.parametrize("new,lens,Hq,Hkv", [([1] * 3, [9000, 20, 5000], 8, 1), ([100, 1], [6000, 300], 2, 1), ([17], [20000], 1, 1)])
def test_long_contexts_split_over_workgroups(cache, new, lens, Hq, Hkv):
    check(make(new, lens, Hq, Hkv, 64, 64, cache, BF))
    check(make(new, lens, Hq, Hkv, 128, 64, cache, BF), 4096, 4)


@pytest.mark.parametrize("cache", [E4, BF])
def test_row_tiles_with_waves_that_have_no_rows(cache):
    """Row tiles of 8, 40 and 72 rows of 128: waves without rows run ahead of the
    others, which must not change what those read, in this call or in the next."""
    case = make([121, 17, 37, 181], [1183, 700, 900, 1435], 32, 4, 128, 128, cache, BF)
    out, _ = check(case)
    q, pools, scales, table, cu, lens = case
    dev = [None if t is None else t.cuda() for t in (q, *pools, table, cu, lens, *scales)]
    for _ in range(20):
        assert torch.equal(_ops().paged_attention(*dev), out)


def test_many_sequences():
    """More sequences than a workgroup has threads, some without tokens or keys."""
    g = torch.Generator().manual_seed(5)
    new = torch.randint(0, 3, (700,), generator=g).tolist()
    lens = [max(n, x) if x else 0 for n, x in zip(new, torch.randint(0, 40, (700,), generator=g).tolist())]
    check(make(new, lens, 2, 1, 16, 16, E4, BF))


def test_strided_queries_and_table():
    q, pools, scales, table, cu, lens = make([3, 1], [50, 70], 4, 2, 64, 16, E4, BF)
    dev = lambda *x: [None if t is None else t.cuda() for t in x]  # noqa: E731
    ops = _ops()
    want = ops.paged_attention(*dev(q, *pools, table, cu, lens, *scales))
    wide = torch.zeros(4, 8, 64, dtype=BF)
    wide[:, 2:6] = q
    tab = torch.full((2, table.shape[1] + 3), -7, dtype=torch.int32)
    tab[:, 1:1 + table.shape[1]] = table
    odd = torch.zeros(4 * 4 * 64 + 1, dtype=BF)
    odd[1:] = q.reshape(-1)
    for qq in (wide.cuda()[:, 2:6], q.permute(2, 0, 1).contiguous().cuda().permute(1, 2, 0), odd.cuda()[1:].view(4, 4, 64)):
        got = ops.paged_attention(qq, *dev(*pools), tab.cuda()[:, 1:1 + table.shape[1]], *dev(cu, lens, *scales))
        assert torch.equal(got, want)


def test_no_tokens():
    q, pools, scales, table, cu, lens = make([0, 0], [5, 0], 4, 2, 64, 16, E4, BF)
    out, lse = _ops().paged_attention(*[t.cuda() for t in (q, *pools, table, cu, lens, *scales)], return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)


def test_offsets_past_32_bits():
    """Pools of more than 2^32 bytes, the sequence's pages at their end."""
    P, page, D = 4200, 512, 256
    for n in (1, 80):
        q, (kc, vc), (ks, vs), table, cu, lens = make([n], [600], 8, 8, D, page, E4, BF, spare=0)
        big = [torch.zeros((P, 8, page, D), dtype=torch.uint8, device="cuda") for _ in range(2)]
        sc = [torch.zeros((P, 8, page), device="cuda") for _ in range(2)]
        for x, y, s, t in zip(big, (kc, vc), sc, (ks, vs)):
            x[P - 2:] = y.view(torch.uint8).cuda()
            s[P - 2:] = t.cuda()
        args = [x.cuda() for x in (cu, lens)]
        got = _ops().paged_attention(q.cuda(), big[0].view(E4), big[1].view(E4), (table + P - 2).cuda(), *args, *sc)
        want = _ops().paged_attention(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), *args, ks.cuda(), vs.cuda())
        assert torch.equal(got, want)
        del big, sc


@pytest.mark.parametrize("new,lens", [([1, 1, 1], [700, 3, 90]), ([70, 1, 9], [700, 3, 90])])
def test_graph_replay_with_new_lengths(new, lens):
    """Captured once; every replay reads the lengths, pages and queries that are there
    then, and equals the eager call, with eager work in between."""
    q, pools, scales, table, cu, ln = make(new, lens, 4, 2, 64, 16, E4, BF)
    dev = [t.cuda() for t in (q, *pools, table, cu, ln, *scales)]
    ops = _ops()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.paged_attention(*dev)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.paged_attention(*dev)
    for i in range(4):
        dev[0].copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(i)).to(BF))
        dev[5].copy_(torch.tensor([max(n, x - 7 * i) for n, x in zip(new, lens)], dtype=torch.int32))
        want = ops.paged_attention(*dev).clone()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), f"replay {i}"


def test_written_tokens_are_attended():
    """kv_cache_write and paged_attention together: a prompt in one chunk gives what
    the same prompt gives in chunks and token by token, up to the order of sums."""
    ops = _ops()
    T, Hq, Hkv, D, page = 75, 4, 2, 64, 16
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(T, h, D, generator=g).to(BF).cuda() for h in (Hq, Hkv, Hkv))
    table = torch.tensor([[4, 0, 3, 1, 2]], dtype=torch.int32, device="cuda")
    pos = torch.arange(T, device="cuda")
    slots = table[0, pos // page].long() * page + pos % page
    outs = []
    for cuts in ([0, 75], [0, 30, 31, 75], list(range(76))):
        c = [torch.zeros(5, Hkv, page, D, dtype=torch.uint8, device="cuda").view(E4) for _ in range(2)]
        s = [torch.zeros(5, Hkv, page, device="cuda") for _ in range(2)]
        parts = []
        for a, b in zip(cuts, cuts[1:]):
            ops.kv_cache_write(k[a:b], v[a:b], *c, slots[a:b], *s)
            i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
            parts.append(ops.paged_attention(q[a:b], *c, table, i32(0, b - a), i32(b), *s))
        outs.append(torch.cat(parts))
    want, _, bound, _ = attention(q, *c, *s, table, torch.tensor([0, T]), torch.tensor([T]), D ** -0.5, None, 0)
    for o in outs:
        within(o, want, bound, "chunks")


@pytest.mark.parametrize("cache,dtype", [(E4, BF), (E5, FH)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("n,L,j,window,sinks", [(1, 300, 7, None, 0), (8, 76, 72, None, 0), (8, 76, 70, 30, 2), (150, 360, 3, None, 0),
                                                (150, 360, 285, None, 0), (150, 360, 285, 40, 3), (150, 360, 1, 40, 3)])
def test_broken_value_scales_reach_the_rows_that_see_them(cache, dtype, bad, n, L, j, window, sinks):
    """A value scale that is NaN (or infinite, beside elements of 0): NaN for the rows
    that see its token, as fp8 * scale_inv gives it, and finite results for the others."""
    q, (kc, vc), (ks, vs), table, cu, lens = make([n, 1], [L, 5], 4, 2, 64, 16, cache, dtype, seed=n)
    clean = vs.clone()
    page = int(table[0, j // 16])
    vs[page, :, j % 16] = bad
    vc.view(torch.uint8)[page, :, j % 16] = 0
    dev = [t.cuda() for t in (q, kc, vc, table, cu, lens, ks, vs)]
    got, lse = (x.cpu().double() for x in _ops().paged_attention(*dev, window_size=window, num_sinks=sinks, return_lse=True))
    args = (table, cu, lens, 64 ** -0.5, window, sinks)
    zero = lambda c: torch.nan_to_num(c.double(), 0.0, 0.0, 0.0)  # noqa: E731
    raw = attention(q, zero(kc), zero(vc), torch.nan_to_num(ks), vs, *args)[0]
    want, wlse, bound, b_lse = attention(q, zero(kc), zero(vc), *(torch.nan_to_num(s) for s in (ks, clean)), *args)
    nan = torch.isnan(raw)
    assert bool(nan.any()) and not bool(nan.all()) and torch.equal(torch.isnan(got), nan)
    within(torch.where(nan, 0.0, got), torch.where(nan, 0.0, want), bound, "rows that do not see it")
    seen = nan.any(2)
    within(torch.where(seen, 0.0, lse), torch.where(seen, 0.0, wlse), b_lse, "their lse")


@pytest.mark.parametrize("cache,dtype", [(E5, BF), (E5, FH), (BF, BF), (FH, FH)])
@pytest.mark.parametrize("n,L,count", [(1, 1, 1), (1, 40, 40), (1, 9000, 9000), (1, 300, 299), (8, 8, 5), (150, 150, 70), (150, 400, 330), (17, 5000, 5000)])
def test_rows_whose_visible_logits_are_all_minus_infinity(cache, dtype, n, L, count):
    """The first `count` keys give logits of -inf: a row that sees no other gets what the
    formula gives, 0 / 0 and -inf, unlike a row that sees no key; the rest ignore them."""
    q, (kc, vc), scales, table, cu, lens = make([n, 1], [L, 0], 4, 2, 64, 16, cache, dtype, seed=L)
    q[..., 9] = q[..., 9].abs() + 1
    low = kc.clone()
    # logits below -250 in place of -inf have a weight of 0 beside the others, in 64 bits too
    for pool, x in ((kc, float("-inf")), (low, -2000.0)):
        for j in range(count):
            pool[int(table[0, j // 16]), :, j % 16, 9] = torch.tensor(x).to(cache)
    dev = [None if t is None else t.cuda() for t in (q, kc, vc, table, cu, lens, *scales)]
    got, lse = (x.cpu().double() for x in _ops().paged_attention(*dev, return_lse=True))
    if cache in FP8_MAX:
        scales[0][:] = torch.nan_to_num(scales[0])
        scales[1][:] = torch.nan_to_num(scales[1])
        low = low.double() * scales[0][..., None]
        for j in range(count):
            low[int(table[0, j // 16]), :, j % 16, 9] = -2000.0
    zero = lambda c: torch.nan_to_num(c.double(), 0.0, 0.0, 0.0)  # noqa: E731
    want, wlse, bound, b_lse = attention(q, zero(low), zero(vc), None, scales[1], table, cu, lens, 64 ** -0.5, None, 0)
    pos = torch.arange(n) + L - n
    none = torch.cat([pos < count, torch.tensor([False])])[:, None].expand(n + 1, 4)  # the last token sees no key
    assert torch.equal(torch.isnan(got).all(2), none) and torch.equal(torch.isnan(got).any(2), none)
    assert bool((lse[none] == float("-inf")).all())
    within(torch.where(none[..., None], 0.0, got), torch.where(none[..., None], 0.0, want), bound, "out")
    within(torch.where(none, 0.0, lse), torch.where(none, 0.0, wlse), b_lse, "lse")


@pytest.mark.parametrize("new,lens,Hq,Hkv", [([1, 1, 1], [70, 300, 5], 4, 2), ([150], [400], 4, 2), ([150, 1, 0, 3], [400, 90, 7, 3], 4, 2),
                                             ([40, 1], [90, 5000], 20, 1), ([0, 0], [9, 0], 4, 2)])
def test_tokens_of_no_sequence(new, lens, Hq, Hkv):
    """Rows ahead of the first sequence and behind the last (a batch padded to a fixed
    size) become zeros and -inf, in a replayed graph too, whatever was there before."""
    front, back = 3, 70
    q, pools, scales, table, cu, ln = make(new, lens, Hq, Hkv, 64, 16, E4, BF)
    q = torch.randn(front + len(q) + back, Hq, 64, generator=torch.Generator().manual_seed(1)).to(BF)
    cu += front
    junk = [torch.full(q.shape, float("nan"), dtype=BF, device="cuda"), torch.full(q.shape[:2], float("nan"), device="cuda")]
    del junk  # its memory is the outputs' now
    out, lse = check((q, pools, scales, table, cu, ln))
    own = slice(front, front + sum(new))
    for x, y in ((out, 0.0), (lse, float("-inf"))):
        x[own] = y
        assert bool((x == y).all())
    dev = [t.cuda() for t in (q, *pools, table, cu, ln, *scales)]
    ops = _ops()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.paged_attention(*dev, return_lse=True)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = ops.paged_attention(*dev, return_lse=True)
    for i in range(4):  # a different first row, and the first sequence shorter
        fewer = torch.tensor([max(0, new[0] - i), *new[1:]])
        dev[4][0] = i
        dev[4][1:] = i + fewer.cumsum(0)
        want, wlse = ops.paged_attention(*dev, return_lse=True)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(lse, wlse), f"replay {i}"
        end = i + int(fewer.sum())
        for a, b in ((0, i), (end, len(q))):
            assert not bool(out[a:b].any()) and bool((lse[a:b] == float("-inf")).all()), f"replay {i}"


@pytest.mark.parametrize("cache,dtype", [(E4, BF), (FH, FH)])
@pytest.mark.parametrize("new,lens,Hq,Hkv", [([300, 2, 1, 5], [300, 9000, 7000, 40], 12, 4), ([200, 1], [5000, 6000], 16, 1),
                                             ([30, 1, 1, 2, 16], [700, 3000, 5, 900, 2000], 2, 2)])
def test_few_rows_beside_prompts_over_long_contexts(cache, dtype, new, lens, Hq, Hkv):
    """Sequences of up to 16 rows whose keys are split, in a batch with longer chunks."""
    check(make(new, lens, Hq, Hkv, 64, 64, cache, dtype, seed=Hq))


@pytest.mark.parametrize("cache,dtype", [(E4, BF), (FH, FH)])
def test_split_row_tiles_of_many_sequences(cache, dtype):
    """More sequences than a workgroup has threads, with split row tiles among the first
    256, the next and the last, one sequence of two tiles, one that is not split."""
    new, lens = [1] * 600, [3 + i % 90 for i in range(600)]
    for i, n, L in ((5, 40, 3000), (6, 9, 20), (255, 20, 1500), (256, 33, 2000), (300, 100, 2500), (599, 17, 700)):
        new[i], lens[i] = n, L
    check(make(new, lens, 4, 2, 32, 64, cache, dtype))
