"""kv_page_ranges, select_pages and sparse_paged_attention against 64 bits."""

import math
import random

import pytest
import torch

from paged_ops_helpers import choose, page_ranges
from serving_helpers import F32, ROUND, values, within

pytestmark = pytest.mark.gpu

E4, E5, BF, FH = torch.float8_e4m3fn, torch.float8_e5m2, torch.bfloat16, torch.float16


def _ops():
    import primus_turbo.pytorch as turbo

    return turbo.ops


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _batch(new, lens, Hq, Hkv, D, page, dtype, cache, seed=0, spare=2, width=None):
    """(q, pools, scales, table, cu, lens) with pages in any order."""
    g = torch.Generator().manual_seed(seed + 7 * Hq + D)
    need = [-(-n // page) for n in lens]
    P, M = sum(need) + spare, width or max(need + [1])
    kc, vc = (torch.randn(P, Hkv, page, D, generator=g) * torch.exp(torch.randn(1, Hkv, 1, D, generator=g) * 0.5) for _ in range(2))
    ks = vs = None
    if cache in (E4, E5):
        ks, vs = (torch.rand(P, Hkv, page, generator=g) * 0.02 + 0.002 for _ in range(2))
        kc, vc = ((x / s[..., None]).clamp(-240, 240).to(cache) for x, s in ((kc, ks), (vc, vs)))
        ks, vs = ks.cuda(), vs.cuda()
    else:
        kc, vc = kc.to(cache), vc.to(cache)
    order = torch.randperm(P, generator=g).tolist()
    table = []
    for n in need:
        table.append([order.pop() for _ in range(n)] + [-1] * (M - n))
    cu = [sum(new[:b]) for b in range(len(new) + 1)]
    q = torch.randn(cu[-1], Hq, D, generator=g).to(dtype).cuda()
    return q, kc.cuda(), vc.cuda(), ks, vs, _i32(table).view(len(new), M), _i32(cu), _i32(lens)


def _all_ranges(kc, ks, table, lens, page):
    """Ranges of every page of every sequence, and NaN elsewhere (what is not read)."""
    P, H, _, D = kc.shape
    out = torch.full((P, H, 2, D), float("nan"), dtype=BF)
    x = values(kc, ks).float() if ks is None else kc.cpu().float() * ks.cpu()[..., None]
    for row, L in zip(table.tolist(), lens.tolist()):
        for j in range(-(-min(L, len(row) * page) // page)):
            if 0 <= row[j] < P:
                for h in range(H):
                    out[row[j], h] = page_ranges(x[row[j], h, :min(page, L - j * page)])
    return out


def _attention(q, kc, vc, ks, vs, ranges, table, cu, lens, scale, take, first, last):
    """(out, lse, their bounds, pages, keys seen): the bounds are those of serving_helpers.attention."""
    q, K, V, table, ranges = q.cpu(), values(kc, ks), values(vc, vs), table.cpu(), ranges.cpu()
    P, Hkv, page, D = K.shape
    T, Hq, _ = q.shape
    G, u, M = Hq // Hkv, ROUND[q.dtype], table.shape[1]
    out, lse = torch.zeros(q.shape, dtype=torch.float64), torch.full((T, Hq), -math.inf, dtype=torch.float64)
    b_out, b_lse = torch.zeros_like(out), torch.zeros_like(lse)
    pages, seen = torch.full((T, Hkv, min(take, M)), -1, dtype=torch.int32), torch.zeros(T, dtype=torch.int32)
    cu, lens = cu.tolist(), lens.tolist()
    for b in range(len(lens)):
        n, L = cu[b + 1] - cu[b], min(max(lens[b], 0), M * page)
        for i in range(n):
            t, at = L - n + i, cu[b] + i
            if t < 0:
                continue
            for h in range(Hkv):
                js = choose(q[at, h * G:(h + 1) * G], ranges[:, h], table[b], t, page, take, first, last)
                ids = [int(table[b, j]) for j in js]
                pages[at, h, :len(ids)] = torch.tensor(ids, dtype=torch.int32)
                k, v = (torch.cat([X[p, h] if 0 <= p < P else torch.zeros(page, D, dtype=torch.float64) for p in ids]) for X in (K, V))
                see = (len(js) - 1) * page + t % page + 1
                seen[at] = see
                k, v = k[:see], v[:see]
                for g in range(h * G, (h + 1) * G):
                    qq = q[at, g].double()
                    s = (k @ qq) * scale
                    e = (D + 8) * F32 * float(((k.abs() @ qq.abs()) * scale).max()) + 2.0 ** -21
                    p = torch.softmax(s, 0)
                    out[at, g] = p @ v
                    lse[at, g] = torch.logsumexp(s, 0)
                    b_out[at, g] = (p @ v.abs()) * (u + 3 * e + see * F32) + u * out[at, g].abs() + 2.0 ** -30
                    if q.dtype == FH:
                        b_out[at, g] += see * 2.0 ** -25 * float(v.abs().max()) + 2.0 ** -25
                    b_lse[at, g] = 2 * e + see * F32 + 2.0 ** -20 * lse[at, g].abs() + 2.0 ** -20
    return out, lse, b_out, b_lse, pages, seen


def _check(case, take, first, last, scale=None):
    ops = _ops()
    q, kc, vc, ks, vs, table, cu, lens = case
    page = kc.shape[2]
    ranges = _all_ranges(kc, ks, table, lens, page).cuda()
    out, lse, b_out, b_lse, pages, seen = _attention(q, kc, vc, ks, vs, ranges, table, cu, lens, scale or q.shape[2] ** -0.5, take, first, last)
    sel, n = ops.select_pages(q, ranges, table, cu, lens, page, num_selected=take, num_first=first, num_last=last)
    assert torch.equal(sel.cpu(), pages) and torch.equal(n.cpu(), seen)
    o, l = ops.sparse_paged_attention(q, kc, vc, ranges, table, cu, lens, ks, vs, num_selected=take, num_first=first, num_last=last,
                                      softmax_scale=scale, return_lse=True)
    within(o, out, b_out, "out")
    within(l, lse, b_lse, "lse")
    assert torch.equal(o, ops.sparse_paged_attention(q, kc, vc, ranges, table, cu, lens, ks, vs, num_selected=take, num_first=first,
                                                     num_last=last, softmax_scale=scale))


@pytest.mark.parametrize("cache,dtype", [(E4, BF), (E5, FH), (BF, BF), (FH, FH), (E4, FH)])
@pytest.mark.parametrize("Hq,Hkv,D,page,take,first,last", [(4, 2, 64, 16, 4, 1, 2), (8, 1, 128, 7, 5, 0, 1), (3, 3, 80, 32, 3, 1, 1),
                                                           (16, 4, 256, 5, 9, 2, 4), (20, 1, 16, 1, 30, 0, 2)])
def test_mixed_batch(cache, dtype, Hq, Hkv, D, page, take, first, last):
    """Single tokens, chunks, empty sequences, one shorter than its new tokens."""
    new, lens = [1, 0, 9, 1, 4, 1, 1], [page * 12 + 3, page * 5, page * 6 + 2, 1, 2, page * take, page * take + 1]
    _check(_batch(new, lens, Hq, Hkv, D, page, dtype, cache), take, first, last)


@pytest.mark.parametrize("take,first,last", [(1, 0, 1), (3, 2, 1), (6, 0, 6), (500, 3, 2)])
def test_first_and_last_alone_and_all(take, first, last):
    _check(_batch([1, 3, 1], [400, 333, 16], 8, 2, 64, 16, BF, E4, seed=2), take, first, last, scale=0.3)


@pytest.mark.parametrize("L", [16 * 64 + 5, 3000, 64 * 130])
def test_long_contexts(L):
    """Keys split over workgroups, tables of hundreds of pages."""
    _check(_batch([1], [L], 16, 2, 128, 16, BF, E4, seed=L), 40, 1, 2)


@pytest.mark.parametrize("Hq,Hkv,D,page,take,new,lens", [
    (4, 1, 64, 4, 20, [37, 2], [4 * 300 + 1, 4 * 1000]),      # tiles of four tokens, more pages than a wave's first hundreds
    (3, 3, 80, 16, 5, [33], [16 * 40 + 7]),                   # a head of its own for each query, sixteen tokens
    (6, 2, 128, 33, 6, [3, 3, 3, 3, 11], [700, 5, 33 * 12, 34, 400]),  # several sequences in a tile, three query heads: a row too few
    (8, 1, 256, 8, 12, [9, 2], [8 * 60, 8 * 70 + 3]),         # two tokens
    (2, 1, 64, 1, 50, [3, 17], [1999, 2048]),                 # more pages than a lane has sixteen scores for
    (1, 1, 16, 1, 9, [18], [2048]), (2, 2, 16, 1, 9, [18], [2049]),  # the most pages of a tile, and one more
    (16, 2, 64, 1, 3, [5, 40], [5, 64])])
def test_chunks(Hq, Hkv, D, page, take, new, lens):
    """Tokens that share their pages' reads, each with its own pages and position."""
    for dtype, cache in ((BF, E4), (FH, FH)):
        _check(_batch(new, lens, Hq, Hkv, D, page, dtype, cache, seed=3), take, 1, 2)


@pytest.mark.parametrize("page", [16, 32])
@pytest.mark.parametrize("Hq,Hkv,new,pages", [(2, 2, [40], [30]), (4, 2, [3, 2, 35], [30, 30, 30]), (3, 3, [7, 20, 9], [30, 29, 30])])
def test_chunks_whose_lists_are_full(Hq, Hkv, new, pages, page):
    """Every token takes all of its sequence's pages: lists as long as their sequences' rows of the table."""
    _check(_batch(new, [page * n for n in pages], Hq, Hkv, 64, page, BF, E4, seed=6), 30, 1, 2)


def test_chunk_with_special_values():
    """Infinities and NaN of keys that only some of a tile's tokens take or see."""
    ops = _ops()
    page, take = 16, 4
    q, kc, vc, ks, vs, table, cu, lens = _batch([8], [16 * 30], 4, 1, 64, page, BF, BF, seed=11)
    ranges = _all_ranges(kc, ks, table, lens, page).cuda()
    sel, _ = ops.select_pages(q, ranges, table, cu, lens, page, num_selected=take)
    call = lambda: ops.sparse_paged_attention(q, kc, vc, ranges, table, cu, lens, num_selected=take)  # noqa: E731
    want = call()
    # a page that some take and some do not
    count = {int(p): [int(p) in sel[t, 0].tolist() for t in range(8)] for p in table[0].tolist()}
    p, takers = next((p, x) for p, x in count.items() if 0 < sum(x) < 8)
    for bad in (float("nan"), float("inf")):
        keep = vc[p, 0, 3].clone()
        vc[p, 0, 3] = bad
        got = call()
        for t in range(8):
            if takers[t]:
                assert not bool(got[t].isfinite().any())
            else:
                assert torch.equal(got[t], want[t])
        vc[p, 0, 3] = keep
    # the last token's own key: the ones before do not see it
    vc[table[0, 29], 0, 15] = float("nan")
    kc[table[0, 29], 0, 15] = float("nan")
    got = call()
    assert torch.equal(got[:7], want[:7]) and bool(got[7].isnan().all())


@pytest.mark.parametrize("cache,dtype", [(E4, BF), (E5, FH), (BF, BF), (FH, FH)])
@pytest.mark.parametrize("Hq,Hkv,D,page", [(4, 1, 64, 64), (8, 2, 128, 32), (4, 2, 256, 96), (2, 2, 16, 32), (12, 4, 112, 64), (6, 1, 48, 32)])
def test_chunks_over_pages_of_whole_runs(cache, dtype, Hq, Hkv, D, page):
    """Pages of 32 tokens or a multiple, some of them none of the pool's, lengths that end anywhere in a page."""
    case = list(_batch([19, 1, 4], [page * 9 + 5, page * 4, page * 6 - 31], Hq, Hkv, D, page, dtype, cache, seed=page))
    _check(case, 5, 1, 2)
    table = case[5]
    table[0, 3], table[0, 8], table[1, 0], table[2, 2] = -1, case[1].shape[0], 10 ** 9, -7
    _check(case, 5, 1, 2)
    case[7] = _i32([10 ** 9, -4, 3])
    _check(case, 4, 0, 1)


@pytest.mark.parametrize("cache,dtype", [(E4, BF), (E5, FH), (BF, BF), (FH, FH)])
@pytest.mark.parametrize("D,page", [(128, 32), (64, 64), (128, 16)])
def test_chunk_over_special_values(cache, dtype, D, page):
    """Special values of a page that a part of a tile's tokens takes reach those alone, whose other elements hold."""
    ops = _ops()
    q, kc, vc, ks, vs, table, cu, lens = _batch([12], [page * 20], 4, 1, D, page, dtype, cache, seed=5)
    ranges = _all_ranges(kc, ks, table, lens, page).cuda()
    call = lambda: ops.sparse_paged_attention(q, kc, vc, ranges, table, cu, lens, ks, vs, num_selected=5)  # noqa: E731
    sel, _ = ops.select_pages(q, ranges, table, cu, lens, page, num_selected=5)
    want = call()
    count = {int(p): [int(p) in sel[t, 0].tolist() for t in range(12)] for p in table[0].tolist()}
    p, takers = next((p, x) for p, x in count.items() if 0 < sum(x[:4]) < 4)
    for bad in (float("nan"),) if cache == E4 else (float("nan"), float("inf"), -float("inf")):
        x = vc[p, 0, 3].float().cpu()
        keep = x.clone()
        x[7] = bad
        vc[p, 0, 3] = x.to(cache).cuda()
        got = call()
        vc[p, 0, 3] = keep.to(cache).cuda()
        other = [d for d in range(D) if d != 7]
        for t in range(12):
            if not takers[t]:
                assert torch.equal(got[t], want[t])
            else:
                assert torch.equal(got[t, :, other], want[t, :, other])
                assert bool(got[t, :, 7].isnan().all()) if math.isnan(bad) else bool((got[t, :, 7] == bad).all())


def test_chunks_of_several_slices():
    """More scores than are held at once: tiles of five tokens on both sides of where a slice ends,
    against the same tokens by themselves."""
    ops = _ops()
    Hkv, M, take, n = 8, 2048, 12, 1100
    q, kc, vc, ks, vs, table, cu, lens = _batch([n, n], [M, M], 3 * Hkv, Hkv, 16, 1, BF, E4, seed=9)
    lo, hi = torch.sort(torch.randn(2, kc.shape[0], Hkv, 16, generator=torch.Generator().manual_seed(3)), dim=0)[0]
    ranges = torch.stack((lo, hi), dim=2).to(BF).cuda()
    step = (256 << 20) // (Hkv * M * 8) // 5 * 5
    assert n < step < 2 * n
    o, l = ops.sparse_paged_attention(q, kc, vc, ranges, table, cu, lens, ks, vs, num_selected=take, return_lse=True)
    at = [0, n - 1, n, *range(step - 6, step + 6), 2 * n - 1]
    rows = _i32([t // n for t in at]).long()
    one = (q[at], kc, vc, ks, vs, ranges, table[rows], _i32(list(range(len(at) + 1))), _i32([M - n + t % n + 1 for t in at]), 0.25, take, 1, 2)
    out, lse, b_out, b_lse, pages, _ = _attention(*one)
    within(o[at], out, b_out, "out")
    within(l[at], lse, b_lse, "lse")
    sel, _ = ops.select_pages(q, ranges, table, cu, lens, 1, num_selected=take)
    assert torch.equal(sel[at].cpu(), pages)


def test_no_more_pages_than_selected_is_paged_attention():
    ops = _ops()
    q, kc, vc, ks, vs, table, cu, lens = _batch([1, 5, 1], [100, 90, 1], 8, 4, 128, 32, BF, E4)
    ranges = torch.full((kc.shape[0], 4, 2, 128), float("nan"), dtype=BF, device="cuda")  # not read
    a, la = ops.sparse_paged_attention(q, kc, vc, ranges, table, cu, lens, ks, vs, num_selected=4, return_lse=True)
    b, lb = ops.paged_attention(q, kc, vc, table, cu, lens, ks, vs, return_lse=True)
    assert bool(((a.double() - b.double()).abs() <= 2.0 ** -6 * b.double().abs() + 2.0 ** -7).all()) and bool(((la - lb).abs() <= 1e-4).all())


def test_padded_batch_and_strides():
    """Rows that no sequence owns, queries inside a projection, rows of a wider table."""
    ops = _ops()
    q, kc, vc, ks, vs, table, cu, lens = _batch([2, 1], [200, 130], 4, 2, 64, 16, BF, E4)
    ranges = _all_ranges(kc, ks, table, lens, 16).cuda()
    out, lse, b_out, b_lse, _, _ = _attention(q, kc, vc, ks, vs, ranges, table, cu, lens, 64 ** -0.5, 5, 1, 2)
    wide = torch.full((8, 3, 4, 64), float("nan"), dtype=BF, device="cuda")
    wide[2:5, 1] = q
    t2 = torch.full((2, table.shape[1] + 3), 10 ** 9, dtype=torch.int32, device="cuda")
    t2[:, :table.shape[1]] = table
    got = ops.sparse_paged_attention(wide[:, 1], kc, vc, ranges, t2[:, :table.shape[1]], cu + 2, lens, ks, vs, num_selected=5, return_lse=True)
    # more rows may take another form, whose sums have another order: within the bounds, not the same bits
    within(got[0][2:5], out, b_out, "out")
    within(got[1][2:5], lse, b_lse, "lse")
    pad = torch.tensor([0, 1, 5, 6, 7], device="cuda")
    assert not bool(got[0][pad].any()) and bool((got[1][pad] == -math.inf).all())
    sel, n = ops.select_pages(wide[:, 1], ranges, table, cu + 2, lens, 16, num_selected=5)
    assert bool((sel[pad] == -1).all()) and not bool(n[pad].any())


def test_pages_outside_the_pool_lengths_past_the_table():
    case = list(_batch([1, 2, 1], [16 * 9 + 3, 16 * 7, 16 * 8], 4, 2, 64, 16, BF, E4))
    table = case[5]
    table[0, 2], table[0, 5], table[1, 6], table[2, 0] = -1, case[1].shape[0], 10 ** 9, -5
    _check(case, 4, 1, 1)
    case[7] = _i32([10 ** 9, -4, 16 * 10 + 1])  # lengths that the table cannot hold, or below 0
    case[5] = torch.where(table < 0, 0, table)
    _check(case, 4, 1, 1)


def test_chunks_over_bad_pages_and_lengths():
    """The same of tiles of tokens: pages outside the pool are zeros that every token sees."""
    case = list(_batch([6, 5, 4], [16 * 9 + 3, 16 * 7, 16 * 8], 4, 2, 64, 16, BF, E4))
    table = case[5]
    table[0, 2], table[0, 5], table[1, 6], table[2, 0], table[2, 7] = -1, case[1].shape[0], 10 ** 9, -5, -1
    _check(case, 4, 1, 1)
    case[7] = _i32([10 ** 9, -4, 2])  # past the table, below 0, fewer than the new tokens
    _check(case, 4, 1, 1)


def test_ranges_and_attention_past_32_bits():
    """Pools of more than 2^32 bytes: the last pages are where they belong."""
    ops = _ops()
    P, H, page, D = 4200, 8, 512, 256  # 4.4e9 bytes a pool
    g = torch.Generator().manual_seed(1)
    kc, vc = (torch.zeros((P, H, page, D), dtype=torch.uint8, device="cuda").view(E4) for _ in range(2))
    ks, vs = (torch.ones((P, H, page), device="cuda") for _ in range(2))
    ids = [P - 1, 7, P - 2, P // 2, P - 5]
    small = [torch.randn(5, H, page, D, generator=g).to(E4) for _ in range(2)]
    for t, x in zip((kc, vc), small):
        t.view(torch.uint8)[ids] = x.view(torch.uint8).cuda()
    q = torch.randn(2, 8, D, generator=g).to(BF).cuda()
    ranges = torch.zeros((P, H, 2, D), dtype=BF, device="cuda")
    table, cu, lens = _i32([ids]), _i32([0, 2]), _i32([5 * page - 3])
    ops.kv_page_ranges(kc, table, _i32([0, 5 * page - 3]), lens, ranges, ks)
    near = [x.cuda() for x in small] + [torch.ones((5, H, page), device="cuda") for _ in range(2)]
    r2 = torch.zeros((5, H, 2, D), dtype=BF, device="cuda")
    t2 = _i32([[0, 1, 2, 3, 4]])
    ops.kv_page_ranges(near[0], t2, _i32([0, 5 * page - 3]), lens, r2, near[2])
    assert torch.equal(ranges[ids], r2)
    a = ops.sparse_paged_attention(q, kc, vc, ranges, table, cu, lens, ks, vs, num_selected=3)
    b = ops.sparse_paged_attention(q, near[0], near[1], r2, t2, cu, lens, near[2], near[3], num_selected=3)
    assert torch.equal(a, b) and bool(a.any())


def test_no_tokens_no_pages():
    ops = _ops()
    q, kc, vc, ks, vs, table, cu, lens = _batch([1, 1], [40, 3], 4, 2, 64, 16, BF, E4)
    ranges = torch.zeros((kc.shape[0], 2, 2, 64), dtype=BF, device="cuda")
    o, l = ops.sparse_paged_attention(q[:0], kc, vc, ranges, table, cu * 0, lens, ks, vs, num_selected=3, return_lse=True)
    assert o.shape == (0, 4, 64) and l.shape == (0, 4)
    o, l = ops.sparse_paged_attention(q, kc, vc, ranges, table[:, :0], cu, lens, ks, vs, num_selected=3, return_lse=True)
    assert not bool(o.any()) and bool((l == -math.inf).all())
    o, l = ops.sparse_paged_attention(q, kc, vc, ranges, table, cu, lens * 0, ks, vs, num_selected=3, return_lse=True)
    assert not bool(o.any()) and bool((l == -math.inf).all())
    e = [t[:0] for t in (kc, vc, ranges, ks, vs)]
    o = ops.sparse_paged_attention(q, e[0], e[1], e[2], table, cu, lens, e[3], e[4], num_selected=3)
    assert not bool(o.any())
    ops.kv_page_ranges(e[0], table, cu, lens, e[2], e[3])
    ops.kv_page_ranges(kc, table[:0], cu[:1], lens[:0], ranges, ks)
    ops.kv_page_ranges(kc, table[:, :0], cu, lens, ranges, ks)
    assert not bool(ranges.any())


# ---------------------------------------------------------------------------
# the choice alone
# ---------------------------------------------------------------------------
def _choice(q, ranges, row, pos, page, take, first, last):
    """All tokens and heads at once: numbers of the pages, -1 behind the last."""
    T, Hq, D = q.shape
    Hkv = ranges.shape[1]
    x = q.double().view(T, Hkv, Hq // Hkv, D)
    up, down = x.clamp(min=0).sum(2), x.clamp(max=0).sum(2)
    r = ranges[row.long()].double()  # [M, Hkv, 2, D]
    out = torch.full((T, Hkv, take), -1, dtype=torch.int64, device=q.device)
    j, own = torch.arange(row.numel(), device=q.device), pos // page
    for h in range(Hkv):
        s = up[:, h].contiguous() @ r[:, h, 1].t().contiguous() + down[:, h].contiguous() @ r[:, h, 0].t().contiguous()
        s = torch.where((j < first) | (own[:, None] - j < last), math.inf, s)
        s = torch.where(j > own[:, None], -math.inf, s)
        best = torch.sort(s, dim=1, descending=True, stable=True)[1][:, :take]
        best = torch.where(best <= own[:, None], best, 10 ** 9).sort(dim=1)[0]
        out[:, h, :best.shape[1]] = torch.where(best < 10 ** 9, best, -1)
    return out


@pytest.mark.parametrize("T,M,Hq,Hkv,D,take", [(5, 40, 4, 2, 64, 7), (300, 256, 8, 8, 16, 33), (70, 257, 8, 2, 128, 64), (3, 1024, 4, 1, 256, 100),
                                               (9, 1500, 16, 4, 48, 20), (2, 4097, 8, 2, 32, 17), (40, 9000, 4, 4, 16, 1000), (620, 8192, 8, 8, 16, 12)])
def test_choice_among_many_pages(T, M, Hq, Hkv, D, take):
    """Keys in a wave, in several, in more than a workgroup holds; more than one slice of tokens."""
    g = torch.Generator("cuda").manual_seed(M)
    row = torch.randperm(M + 3, generator=g, device="cuda")[:M].to(torch.int32)
    lo, hi = torch.sort(torch.randn(2, M + 3, Hkv, D, generator=g, device="cuda"), dim=0)[0]
    ranges = torch.stack((lo, hi), dim=2).to(BF)
    q = torch.randn(T, Hq, D, generator=g, device="cuda").to(BF)
    L = M  # pages of one token
    sel, n = _ops().select_pages(q, ranges, row[None], _i32([0, T]), _i32([L]), 1, num_selected=take, num_first=1, num_last=2)
    pos = torch.arange(L - T, L, device="cuda")
    want = _choice(q, ranges, row, pos, 1, take, 1, 2)
    assert torch.equal(sel.long(), torch.where(want >= 0, row[want.clamp(min=0)].long(), -1))
    assert torch.equal(n.long(), (pos + 1).clamp(0, take))  # more tokens than the length says see nothing


def test_ties_go_to_the_lower_page():
    ops = _ops()
    for M in (50, 300, 1100, 5000):
        for Hkv, take in ((1, 10), (3, 33)):
            ranges = torch.ones(M, Hkv, 2, 32, dtype=BF, device="cuda")
            ranges[M // 2, :, 1] = 2.0  # one better page
            q = torch.ones(2, Hkv * 2, 32, dtype=FH, device="cuda")
            row = torch.arange(M, device="cuda").to(torch.int32)[None]
            sel, _ = ops.select_pages(q, ranges, row, _i32([0, 2]), _i32([M]), 1, num_selected=take, num_first=0, num_last=1)
            for t, own in ((0, M - 2), (1, M - 1)):
                rest = [j for j in range(M) if j not in (M // 2, own)]
                assert sel[t].tolist() == [sorted(rest[:take - 2] + [M // 2, own])] * Hkv
    # zeros of either sign are equal
    ranges = torch.zeros(20, 1, 2, 16, dtype=BF, device="cuda")
    ranges[::2] = -0.0
    q = torch.ones(1, 1, 16, dtype=BF, device="cuda")
    sel, _ = ops.select_pages(q, ranges, torch.arange(20, device="cuda").to(torch.int32)[None], _i32([0, 1]), _i32([20]), 1, num_selected=6,
                              num_first=0, num_last=1)
    assert sel.flatten().tolist() == [0, 1, 2, 3, 4, 19]


def test_infinities_and_nan_in_ranges_and_queries():
    ops = _ops()
    M, inf = 30, float("inf")
    row = torch.arange(M, device="cuda").to(torch.int32)[None]
    ranges = torch.randn(M, 1, 2, 16, generator=torch.Generator().manual_seed(0)).to(BF).cuda()
    ranges[4, 0, 1, 3], ranges[9, 0, 0, 2], ranges[11, 0, 1], ranges[13, 0, 1, 0] = float("nan"), float("nan"), inf, -inf
    q = torch.ones(1, 2, 16, dtype=BF, device="cuda")
    for x in (q, -q, q * 0):
        for take in (3, 5, 8):
            sel, _ = ops.select_pages(x, ranges, row, _i32([0, 1]), _i32([M]), 1, num_selected=take, num_first=0, num_last=1)
            up, down = x[0].double().clamp(min=0).sum(0), x[0].double().clamp(max=0).sum(0)
            s = (up * ranges[:, 0, 1].double() + down * ranges[:, 0, 0].double()).sum(1)
            s = torch.where(s.isnan(), inf, s)
            want = sorted(sorted(range(M - 1), key=lambda j: (-s[j].item(), j))[:take - 1] + [M - 1])
            assert sel.flatten().tolist() == want
    q[0, 0, 0] = float("nan")  # every score is NaN: the first pages
    sel, _ = ops.select_pages(q, ranges, row, _i32([0, 1]), _i32([M]), 1, num_selected=4, num_first=0, num_last=1)
    assert sel.flatten().tolist() == [0, 1, 2, M - 1]


# ---------------------------------------------------------------------------
# ranges
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("cache", [E4, E5, BF, FH])
@pytest.mark.parametrize("H,D,page", [(1, 16, 1), (2, 64, 16), (3, 80, 7), (8, 128, 64), (2, 256, 130)])
def test_ranges(cache, H, D, page):
    """Of the pages that hold new tokens, over the tokens that the sequence has; no others."""
    new, lens = [1, 0, page + 3, 1, 2 * page, 5], [3 * page + 1, 2 * page, 4 * page, 1, 2 * page, 2]
    _, kc, _, ks, _, table, cu, lens = _batch(new, lens, H, H, D, page, BF, cache, spare=3)
    before = torch.randn(kc.shape[0], H, 2, D, generator=torch.Generator().manual_seed(1)).to(BF).cuda()
    got = before.clone()
    _ops().kv_page_ranges(kc, table, cu, lens, got, ks)
    want, every = before.cpu().clone(), _all_ranges(kc, ks, table, lens, page)
    for row, n, L in zip(table.tolist(), new, lens.tolist()):
        for j in range(max(0, L - n) // page, -(-L // page) if n else 0):
            want[row[j]] = every[row[j]]
    assert torch.equal(got.cpu().view(torch.int16), want.view(torch.int16))


def test_ranges_of_special_values_and_bad_pages():
    ops = _ops()
    kc = torch.randn(4, 1, 8, 32, generator=torch.Generator().manual_seed(2)).to(BF)
    kc[0, 0, 3, 5], kc[0, 0, 2, 6], kc[0, 0, 7, 7], kc[1, 0, 6, 0] = float("nan"), float("inf"), -float("inf"), float("nan")
    kc = kc.cuda()
    r = torch.zeros(4, 1, 2, 32, dtype=BF, device="cuda")
    # page 1's NaN lies behind the length
    ops.kv_page_ranges(kc, _i32([[0, 1, -1, 9], [-3, 4, 3, 2]]), _i32([0, 14, 50]), _i32([14, 2 ** 31 - 1]), r)
    assert r[0, 0, :, 5].isnan().all() and r[0, 0, 1, 6] == math.inf and r[0, 0, 0, 7] == -math.inf
    assert not bool(r[1].isnan().any()) and torch.equal(r[1, 0], page_ranges(kc[1, 0, :6].float()))
    assert torch.equal(r[3, 0], page_ranges(kc[3, 0].float())) and torch.equal(r[2, 0], page_ranges(kc[2, 0].float()))


def test_infinite_keys_and_values_as_paged_attention_has_them():
    """A page with NaN is taken, and shows in the rows that see it."""
    ops = _ops()
    q, kc, vc, ks, vs, table, cu, lens = _batch([1, 1], [16 * 10, 16 * 10], 4, 2, 64, 16, BF, BF)
    kc[table[0, 4].item(), 1, 3, 7] = float("nan")
    ranges = _all_ranges(kc, ks, table, lens, 16).cuda()
    o = ops.sparse_paged_attention(q, kc, vc, ranges, table, cu, lens, num_selected=4)
    assert bool(o[0, 2:].isnan().all()) and not bool(o[0, :2].isnan().any()) and not bool(o[1].isnan().any())


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
def test_served_steps():
    """A prompt in chunks, then single tokens, forked in between: norm, rotation and write, ranges, pages, attention."""
    ops = _ops()
    Hq, Hkv, D, page, P, M, take = 8, 2, 64, 16, 60, 12, 4
    g = torch.Generator().manual_seed(4)
    f = 10000.0 ** (-torch.arange(D // 2, dtype=torch.float64) * 2 / D)
    a = torch.arange(M * page, dtype=torch.float64)[:, None] * f
    cos, sin = a.cos().float().cuda(), a.sin().float().cuda()
    wq, wk = ((1 + 0.2 * torch.randn(D, generator=g)).to(BF).cuda() for _ in range(2))
    kc, vc = (torch.zeros(P, Hkv, page, D, dtype=torch.uint8, device="cuda").view(E4) for _ in range(2))
    ks, vs = (torch.zeros(P, Hkv, page, device="cuda") for _ in range(2))
    ranges = torch.zeros(P, Hkv, 2, D, dtype=BF, device="cuda")
    table, lens = torch.full((2, M), -1, dtype=torch.int32, device="cuda"), _i32([0, 0])
    parents, new = [0, 1], [37, 90]
    for step in range(6):
        if step == 2:
            parents = [1, 0, 1, 1, 0]  # several answers to each prompt
        if step == 4:
            parents = [3, 3, 0]        # the best go on
        if step > 1:
            new = [1] * len(parents)
        table, lens = ops.kv_cache_fork(kc, vc, table, lens, _i32(parents), ks, vs, key_ranges=ranges, reserve=max(new), compact=step % 2 == 1)
        old = lens.tolist()
        lens = lens + _i32(new)
        T = sum(new)
        pos = torch.tensor([L + i for L, n in zip(old, new) for i in range(n)], device="cuda")
        seq = torch.tensor([b for b, n in enumerate(new) for _ in range(n)], device="cuda")
        slots = table[seq, pos // page].long() * page + pos % page
        cu = _i32([sum(new[:b]) for b in range(len(new) + 1)])
        qkv = torch.randn(T, Hq + 2 * Hkv, D, generator=g).to(BF).cuda()
        q, k, v = qkv.split([Hq, Hkv, Hkv], dim=1)
        q = ops.qk_norm_rope_cache_write(q, k, v, cos, sin, pos, kc, vc, slots, ks, vs, q_weight=wq, k_weight=wk)
        ops.kv_page_ranges(kc, table, cu, lens, ranges, ks)
        every = _all_ranges(kc, ks, table, lens, page)
        held = ~every.isnan()
        assert torch.equal(ranges.cpu()[held], every[held]), f"step {step}"
        used = [u for row, L in zip(table.tolist(), lens.tolist()) for u in row[:-(-L // page)]]
        assert min(used) >= 0 and len(set(slots.tolist())) == T
        o, l = ops.sparse_paged_attention(q, kc, vc, ranges, table, cu, lens, ks, vs, num_selected=take, return_lse=True)
        out, lse, b_out, b_lse, _, _ = _attention(q, kc, vc, ks, vs, ranges, table, cu, lens, D ** -0.5, take, 1, 2)
        within(o, out, b_out, f"step {step}")
        within(l, lse, b_lse, f"step {step}")
        parents = list(range(len(new)))


def test_captured_decoding_step():
    ops = _ops()
    q, kc, vc, ks, vs, table, cu, lens = _batch([1] * 6, [300, 17, 160, 1, 299, 64], 8, 2, 64, 16, BF, E4, width=20)
    ranges = _all_ranges(kc, ks, table, lens, 16).cuda()
    ranges = torch.where(ranges.isnan(), 0, ranges)
    full = [list(range(b * 19, b * 19 + 19)) + [-1] for b in range(6)]
    kc, vc, ks, vs, ranges = (t.view(torch.uint8).repeat(6, *[1] * (t.dim() - 1))[:114].contiguous().view(t.dtype) for t in (kc, vc, ks, vs, ranges))
    table.copy_(_i32(full))

    def step():
        ops.kv_page_ranges(kc, table, cu, lens, ranges, ks)
        return ops.sparse_paged_attention(q, kc, vc, ranges, table, cu, lens, ks, vs, num_selected=5, return_lse=True)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    r = random.Random(0)
    for n in range(4):
        lens.copy_(_i32([r.randint(0, 300) for _ in range(6)]))
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(n)).to(BF))
        before = ranges.clone()
        graph.replay()
        torch.cuda.synchronize()
        got, after = [t.clone() for t in held], ranges.clone()
        ranges.copy_(before)
        want = step()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(after.view(torch.int16), ranges.view(torch.int16))


def test_other_stream_and_two_calls_at_once():
    ops = _ops()
    cases = [_batch([1] * 5, [700, 33, 500, 640, 2], 8, 2, 128, 16, BF, E4, seed=s) for s in (1, 2)]
    rs = [_all_ranges(c[1], c[3], c[5], c[7], 16).cuda() for c in cases]
    call = lambda c, r: ops.sparse_paged_attention(c[0], c[1], c[2], r, c[5], c[6], c[7], c[3], c[4], num_selected=6)  # noqa: E731
    want = [call(c, r) for c, r in zip(cases, rs)]
    streams = [torch.cuda.Stream() for _ in cases]
    got = []
    for s, c, r in zip(streams, cases, rs):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append([call(c, r) for _ in range(10)])
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(o, w) for outs, w in zip(got, want) for o in outs)
