"""Plain 64-bit implementations of the operators around the paged cache, with the
error bounds of the kernels' arithmetic, for the tests."""

from __future__ import annotations

import math

import torch

F32 = 2.0 ** -24
#: largest relative error of a rounding to the type, and its smallest half step
ROUND = {torch.bfloat16: (2.0 ** -8, 2.0 ** -134), torch.float16: (2.0 ** -11, 2.0 ** -25), torch.float32: (2.0 ** -24, 2.0 ** -150)}
FP8 = {torch.float8_e4m3fn: (448.0, 2.0 ** -4, 2.0 ** -10), torch.float8_e5m2: (57344.0, 2.0 ** -3, 2.0 ** -17)}


def angles(positions, rot, base=10000.0, device="cuda"):
    f = base ** (-torch.arange(rot // 2, dtype=torch.float64, device=device) * 2 / rot)
    a = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * f
    return a.cos().float(), a.sin().float()


def turn(x, c, s, interleaved):
    """Pairs of the first elements of x [..., H, D] turned by c, s [..., R / 2]."""
    R = 2 * c.shape[-1]
    c, s = c.unsqueeze(-2), s.unsqueeze(-2)
    y = x.clone()
    if interleaved:
        a, b = x[..., 0:R:2], x[..., 1:R:2]
        y[..., 0:R:2], y[..., 1:R:2] = a * c - b * s, a * s + b * c
    else:
        a, b = x[..., :R // 2], x[..., R // 2:R]
        y[..., :R // 2], y[..., R // 2:R] = a * c - b * s, a * s + b * c
    return y


def norm_rope(x, w, cos, sin, pos, eps, interleaved):
    """(y, bound of the error before the last rounding) in 64 bits.

    r is a sum of D squares (D + 2 roundings, halved by the root) and a root of two
    steps; n takes two products; a turned element two products and a sum.
    """
    x, D = x.double(), x.shape[-1]
    ok = (pos >= 0) & (pos < cos.shape[0])
    p = torch.where(ok, pos, 0).long()
    c, s = cos.double()[p], sin.double()[p]
    n = x if w is None else x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * w.double()
    e = 4 if w is None else D / 2 + 12
    y = turn(n, c, s, interleaved)
    size = turn_size(n, c, s, interleaved)
    ok = ok[..., None, None]
    return torch.where(ok, y, 0.0), torch.where(ok, size, 0.0) * (e * F32)


def turn_size(x, c, s, interleaved):
    """|a cos| + |b sin| and so on."""
    R = 2 * c.shape[-1]
    x, c, s = x.abs(), c.abs().unsqueeze(-2), s.abs().unsqueeze(-2)
    y = x.clone()
    if interleaved:
        a, b = x[..., 0:R:2], x[..., 1:R:2]
        y[..., 0:R:2], y[..., 1:R:2] = a * c + b * s, a * s + b * c
    else:
        a, b = x[..., :R // 2], x[..., R // 2:R]
        y[..., :R // 2], y[..., R // 2:R] = a * c + b * s, a * s + b * c
    return y


def norm_rope_grads(x, w, cos, sin, pos, eps, interleaved, g):
    """((dx, bound before its rounding), (dw, bound before its rounding)) in 64 bits; dw None without w."""
    x, g, D = x.double(), g.double(), x.shape[-1]
    ok = (pos >= 0) & (pos < cos.shape[0])
    p = torch.where(ok, pos, 0).long()
    c, s = cos.double()[p], sin.double()[p]
    t, G = turn(g, c, -s, interleaved), turn_size(g, c, s, interleaved)
    ok = ok[..., None, None]
    t, G = torch.where(ok, t, 0.0), torch.where(ok, G, 0.0)
    if w is None:
        return (t, G * (4 * F32)), None
    w = w.double()
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    h = x * r
    er = (D / 2 + 8) * F32  # relative error of h
    dot = (t * w * h).mean(-1, keepdim=True)
    A = (G * w.abs() * h.abs()).mean(-1, keepdim=True)
    dx = r * (t * w - h * dot)
    # g' w: 4 + 1 roundings; the dot's D sums, its factors' errors, the product with h
    e = r * (G * w.abs() * (6 * F32) + h.abs() * A * ((D + 12) * F32 + 3 * er)) + (er + 2 * F32) * r * (G * w.abs() + h.abs() * A)
    rows = x.numel() // D
    dw = (t * h).flatten(0, -2).sum(0)
    ew = (G * h.abs()).flatten(0, -2).sum(0) * ((rows + 64) * F32 + er + 6 * F32)
    return (dx, e), (dw, ew)


def close(got, want, bound, what):
    """got is want, computed within bound and rounded once to its type."""
    u, least = ROUND[got.dtype]
    want, bound, got = want.to(got.device), bound.to(got.device), got.double()
    bad = ~((got - want).abs() <= bound + u * (want.abs() + bound) + least)
    assert not bool(bad.any()), (
        f"{what}: {int(bad.sum())} of {bad.numel()} outside, first at {torch.nonzero(bad)[0].tolist()}: "
        f"{got[bad][0].item()} for {want[bad][0].item()} within {bound[bad][0].item()}"
    )


# ---------------------------------------------------------------------------
# pages: the books of a host
# ---------------------------------------------------------------------------
def fork_books(table, lens, parents, page, P, reserve, compact):
    """(rows, lengths, copies [(from, to)]) of new sequences, one after the other."""
    B, M = len(table), len(table[0]) if table else 0
    seqs = []
    for p in parents:
        if not 0 <= p < B:
            seqs.append(None)
            continue
        n = min(max(lens[p], 0), M * page)
        seqs.append((p, n // page, -(-n // page), min(M, -(-(n + reserve) // page)) if lens[p] >= 0 else 0))
    inside = lambda u: 0 <= u < P  # noqa: E731
    full = {u for s in seqs if s for u in table[s[0]][:s[1]] if inside(u)}
    keeper = {}
    for i, s in enumerate(seqs):
        if s and s[2] > s[1] and inside(table[s[0]][s[1]]) and table[s[0]][s[1]] not in full:
            keeper.setdefault(table[s[0]][s[1]], i)
    used = sorted(full | set(keeper))
    free = [u for u in range(P) if u not in full and u not in keeper]
    need = []
    for i, s in enumerate(seqs):
        if s is None:
            need.append((0, False))
            continue
        last = table[s[0]][s[1]] if s[2] > s[1] else -1
        copy = inside(last) and keeper.get(last) != i
        need.append((s[3] - s[2] + copy, copy))
    move = {}
    if compact:
        bound = len(used) + min(len(free), sum(n for n, _ in need))
        move = dict(zip([u for u in used if u >= bound], free))
    spare = free[len(move):]
    rows, new_lens, copies, at = [], [], list(move.items()), 0
    for s, (n, copy) in zip(seqs, need):
        row = []
        if s is None:
            new_lens.append(0)
        elif n and at + n > len(free):
            new_lens.append(-1)
        else:
            row = [move.get(u, u) for u in table[s[0]][:s[2] - copy]]
            if copy:
                copies.append((table[s[0]][s[1]], spare[at]))
            row += spare[at:at + n]
            new_lens.append(lens[s[0]])
        at += n
        rows.append(row + [-1] * (M - len(row)))
    return rows, new_lens, copies


# ---------------------------------------------------------------------------
# attention through selected pages
# ---------------------------------------------------------------------------
def page_ranges(keys):
    """Smallest and largest of keys [n, D] (fp32), rounded outward: [2, D] bfloat16."""
    out = []
    for x, up in ((keys.amin(0), False), (keys.amax(0), True)):
        y = x.to(torch.bfloat16)
        off = (y.float() < x) if up else (y.float() > x)
        z = torch.nextafter(y, torch.full_like(y, math.inf if up else -math.inf))
        out.append(torch.where(off, z, y))
    return torch.stack(out)


def choose(q, ranges, row, pos, page, take, first, last):
    """Numbers, within the sequence, of the pages that a token takes: q [G, D] of one cache
    head, ranges [P, 2, D] of it, row: the sequence's pages."""
    own = pos // page
    n = own + 1
    if n <= take:
        return list(range(n))
    q, ids = q.double(), row[:n].long()
    ok = (ids >= 0) & (ids < ranges.shape[0])
    r = torch.where(ok[:, None, None], ranges[ids.clamp(0, ranges.shape[0] - 1)].double(), 0.0)
    up, down = torch.where(q > 0, q, 0.0).sum(0), torch.where(q < 0, q, 0.0).sum(0)
    score = (up * r[:, 1] + down * r[:, 0]).sum(1)
    score = torch.where(score.isnan(), math.inf, score)
    always = [j for j in range(n) if j < first or own - j < last]
    rest = sorted((j for j in range(n) if j not in always), key=lambda j: (-score[j].item(), j))
    return sorted(always + rest[:take - len(always)])
