"""Plain 64-bit implementations of the serving operators, with the error bounds
of the kernels' arithmetic, for the tests (CPU)."""

from __future__ import annotations

import math

import torch

FP8_MAX = {torch.float8_e4m3fn: 448.0, torch.float8_e5m2: 57344.0}
#: largest relative error of a rounding to the type
ROUND = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
F32 = 2.0 ** -24


def values(cache, scale):
    """A pool's values in 64 bits."""
    x = cache.cpu().to(torch.float64)
    return x if scale is None else x * scale.cpu().double()[..., None]


def attention(q, kc, vc, ks, vs, table, cu, lens, scale, window, sinks):
    """(out, lse, bound of out's error, bound of lse's) in 64 bits, token by token.

    The bounds follow the kernels' arithmetic: products of 16-bit values are exact,
    a logit is a sum of D of them in fp32 and two more fp32 operations; P and the
    output are rounded once to 16 bits (fp16: with an absolute part for P, whose
    largest is 1); sums over the keys are fp32.
    """
    q, K, V = q.cpu(), values(kc, ks), values(vc, vs)
    Hkv, page, D = K.shape[1:]
    Hq, G = q.shape[1], q.shape[1] // Hkv
    u = ROUND[q.dtype]
    out = torch.zeros(q.shape, dtype=torch.float64)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64)
    b_out, b_lse = torch.zeros_like(out), torch.zeros_like(lse)
    cu, lens, table = cu.tolist(), lens.tolist(), table.cpu()
    for b in range(len(lens)):
        n, L = cu[b + 1] - cu[b], min(lens[b], table.shape[1] * page)
        j = torch.arange(L)
        pg = table[b, j // page].long() if L else j
        ok = (pg >= 0) & (pg < K.shape[0])
        k = K[pg.clamp(0, K.shape[0] - 1), :, j % page] * ok[:, None, None] if L else None  # [L, Hkv, D]
        v = V[pg.clamp(0, K.shape[0] - 1), :, j % page] if L else None
        if L:
            k, v = torch.where(ok[:, None, None], k, 0.0), torch.where(ok[:, None, None], v, 0.0)
        for i in range(n):
            t = L - n + i
            see = [x for x in range(min(t + 1, L)) if not window or t - x < window or x < sinks]
            if not see:
                continue
            kk, vv = k[see].repeat_interleave(G, dim=1), v[see].repeat_interleave(G, dim=1)  # [S, Hq, D]
            qq = q[cu[b] + i].double()
            s = (kk * qq).sum(2) * scale
            e = (D + 8) * F32 * float(((kk.abs() * qq.abs()).sum(2) * abs(scale)).max()) + 2.0 ** -21
            p = torch.softmax(s, dim=0)
            a = (p[..., None] * vv.abs()).sum(0)
            at = cu[b] + i
            out[at] = (p[..., None] * vv).sum(0)
            lse[at] = torch.logsumexp(s, dim=0)
            b_out[at] = a * (u + 3 * e + len(see) * F32) + u * out[at].abs() + 2.0 ** -30
            if q.dtype == torch.float16:
                b_out[at] += len(see) * 2.0 ** -25 * float(vv.abs().max()) + 2.0 ** -25
            b_lse[at] = 2 * e + len(see) * F32 + 2.0 ** -20 * lse[at].abs() + 2.0 ** -20
    return out, lse, b_out, b_lse


def spread(w, s):
    """Scales of any layout as one for each element of w [E, N, K], in 64 bits."""
    s = s.cpu().double()
    E, N, K = w.shape
    if s.numel() == 1:
        return s.reshape(1, 1, 1)
    if tuple(s.shape) == (E, N, 1):
        return s
    return s.repeat_interleave(128, 1)[:, :N].repeat_interleave(128, 2)[:, :, :K]


def experts(x, w1, w2, idx, probs, s1=None, s2=None):
    """(y, bound of its error) in 64 bits, expert by expert."""
    x, idx, probs = x.cpu(), idx.cpu(), probs.cpu().double()
    u, X = ROUND[x.dtype], x.double()
    W1, W2 = (w.cpu().double() if s is None else w.cpu().double() * spread(w, s) for w, s in ((w1, s1), (w2, s2)))
    E, H, I = W2.shape
    y, bound = torch.zeros_like(X), torch.zeros_like(X)
    for e in range(E):
        p = torch.where(idx == e, probs, 0.0).sum(1, keepdim=True)
        t = (idx == e).any(1)
        if not bool(t.any()):
            continue
        h, ha = X[t] @ W1[e].T, X[t].abs() @ W1[e].abs().T * ((H + 8) * F32)  # sums and their fp32 errors
        g, up = h[:, :I], h[:, I:]
        sg = g / (1 + torch.exp(-g))
        a = sg * up * p[t]
        # silu' is below 1.1; a handful of fp32 operations; one rounding to 16 bits
        da = p[t].abs() * (1.1 * ha[:, :I] * up.abs() + sg.abs() * ha[:, I:] + ha[:, :I] * ha[:, I:])
        da = da + a.abs() * (u + 16 * F32 + 2.0 ** -22 * g.abs())
        if x.dtype == torch.float16:
            da = da + 2.0 ** -25
        y[t] += a @ W2[e].T
        bound[t] += (da + a.abs() * ((I + E + 8) * F32)) @ W2[e].abs().T
    bound += u * (y.abs() + bound) + (2.0 ** -25 if x.dtype == torch.float16 else 2.0 ** -60)
    return y, bound


def within(got, want, bound, what):
    got = got.cpu().double()
    bad = ~((got - want).abs() <= bound) & ~(got == want)
    assert not bool(bad.any()), (
        f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst {float(((got - want).abs() / bound).nan_to_num(9e9)[bad].max()):.3g} "
        f"times the bound at {torch.nonzero(bad)[0].tolist()}"
    )
