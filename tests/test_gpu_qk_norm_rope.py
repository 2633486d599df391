"""qk_norm_rope and qk_norm_rope_cache_write against 64 bits, within bounds that
follow the kernels' arithmetic; gradients against the formula's and differences."""

import pytest
import torch

from paged_ops_helpers import F32, FP8, angles, close, norm_rope, norm_rope_grads

pytestmark = pytest.mark.gpu

E4, E5, BF, FH, FF = torch.float8_e4m3fn, torch.float8_e5m2, torch.bfloat16, torch.float16, torch.float32
EPS = 1e-5


def _ops():
    import primus_turbo.pytorch as turbo

    return turbo.ops


def _inputs(T, Hq, Hkv, D, rot, dtype, norm=True, seed=0, extra=0, wdtype=None):
    """Queries, keys and values as parts of one projection, weights, tables, positions."""
    g = torch.Generator().manual_seed(seed + 31 * T + D)
    row = torch.randn(T, (Hq + 2 * Hkv) * D + extra, generator=g).to(dtype).cuda()
    x = row[:, extra:].view(T, Hq + 2 * Hkv, D) if extra == 0 else row[:, extra:].unflatten(1, (Hq + 2 * Hkv, D))
    q, k, v = x.split([Hq, Hkv, Hkv], dim=1)
    w = [(1 + 0.3 * torch.randn(D, generator=g)).to(wdtype or dtype).cuda() if norm else None for _ in range(2)]
    cos, sin = angles(97, rot)
    pos = torch.randint(0, 97, (T,), generator=g).cuda()
    return q, k, v, w[0], w[1], cos, sin, pos


SHAPES = [(1, 1, 1, 2, 2), (3, 2, 1, 6, 4), (7, 3, 2, 10, 10), (33, 4, 2, 16, 16), (19, 5, 5, 64, 64), (64, 12, 12, 80, 32),
          (41, 6, 2, 96, 24), (65, 32, 8, 128, 128), (30, 3, 1, 128, 50), (17, 4, 4, 250, 100), (29, 8, 2, 256, 64), (5, 2, 2, 256, 256)]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("dtype", [BF, FH, FF])
@pytest.mark.parametrize("T,Hq,Hkv,D,rot", SHAPES)
def test_forward_and_backward(T, Hq, Hkv, D, rot, dtype, norm, interleaved):
    q, k, _, wq, wk, cos, sin, pos = _inputs(T, Hq, Hkv, D, rot, dtype, norm)
    leaves = [None if t is None else t.detach().requires_grad_() for t in (q, k, wq, wk)]
    out = _ops().qk_norm_rope(leaves[0], leaves[1], cos, sin, pos, leaves[2], leaves[3], eps=EPS, interleaved=interleaved)
    gs = [torch.randn(o.shape, generator=torch.Generator().manual_seed(5)).to(dtype).cuda() for o in out]
    torch.autograd.backward(out, gs)
    for n, x, w, y, g, lx, lw in zip("qk", (q, k), (wq, wk), out, gs, leaves[:2], leaves[2:]):
        assert y.dtype == dtype and y.shape == x.shape and y.is_contiguous()
        close(y.detach(), *norm_rope(x, w, cos, sin, pos, EPS, interleaved), n)
        dx, dw = norm_rope_grads(x, w, cos, sin, pos, EPS, interleaved, g)
        close(lx.grad, *dx, "d" + n)
        if w is not None:
            assert lw.grad.dtype == w.dtype
            close(lw.grad, *dw, "dw" + n)


@pytest.mark.parametrize("T,Hq,Hkv,D,rot,dtype", [(4133, 32, 8, 128, 128, BF), (9001, 16, 4, 64, 32, FH), (2500, 32, 4, 256, 128, BF), (3001, 24, 8, 80, 80, FF)])
def test_many_rows(T, Hq, Hkv, D, rot, dtype):
    """Several heads a lane, several runs of a workgroup."""
    q, k, _, wq, wk, cos, sin, pos = _inputs(T, Hq, Hkv, D, rot, dtype, wdtype=FF)
    leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
    out = _ops().qk_norm_rope(leaves[0], leaves[1], cos, sin, pos, leaves[2], leaves[3], eps=EPS)
    gs = [torch.randn(o.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(5)).to(dtype) for o in out]
    grads = torch.autograd.grad(out, leaves, gs, retain_graph=True)
    for n, x, w, y, g, gx, gw in zip("qk", (q, k), (wq, wk), out, gs, grads[:2], grads[2:]):
        close(y.detach(), *norm_rope(x, w, cos, sin, pos, EPS, False), n)
        dx, dw = norm_rope_grads(x, w, cos, sin, pos, EPS, False, g)
        close(gx, *dx, "d" + n)
        close(gw, *dw, "dw" + n)
    again = torch.autograd.grad(out, leaves, gs)
    assert all(torch.equal(a, b) for a, b in zip(grads, again)), "the same call has other bits"


@pytest.mark.parametrize("extra", [1, 2, 4, 8])
@pytest.mark.parametrize("dtype", [BF, FF])
def test_alignments_and_layouts(extra, dtype):
    """Rows that begin anywhere, heads ahead of tokens, a last dimension that is not contiguous, leading dimensions."""
    ops = _ops()
    q, k, _, wq, wk, cos, sin, pos = _inputs(24, 4, 2, 64, 32, dtype, extra=extra)
    assert not q.is_contiguous()
    want = ops.qk_norm_rope(q.contiguous(), k.contiguous(), cos, sin, pos, wq, wk)
    # another alignment is another split of the row's sum: within the bound, which goes by
    # |a cos| + |b sin| (the two may cancel), not the same bits
    for a, x, w in zip(ops.qk_norm_rope(q, k, cos, sin, pos, wq, wk), (q, k), (wq, wk)):
        close(a, *norm_rope(x, w, cos, sin, pos, 1e-6, False), "strided")
    turned = [x.permute(2, 1, 0).contiguous().permute(2, 1, 0) for x in (q, k)]
    for a, b in zip(ops.qk_norm_rope(*turned, cos, sin, pos, wq, wk), want):
        assert torch.equal(a, b)
    ahead = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k)]
    for a, b in zip(ops.qk_norm_rope(*ahead, cos, sin, pos, wq, wk), want):
        assert torch.equal(a, b)
    more = [x.contiguous().view(2, 3, 4, *x.shape[1:]) for x in (q, k)]
    got = ops.qk_norm_rope(*more, cos, sin, pos.view(2, 3, 4).to(torch.int32), wq, wk)
    for a, b in zip(got, want):
        assert torch.equal(a.view(b.shape), b)
    one = ops.qk_norm_rope(q[3].contiguous(), k[3].contiguous(), cos, sin, pos[3], wq, wk)
    assert torch.equal(one[0], want[0][3]) and torch.equal(one[1], want[1][3])


def test_tables_that_begin_anywhere():
    """cos and sin off a 16-byte boundary, an odd number of angles."""
    ops = _ops()
    for rot in (64, 6):
        q, k, _, wq, wk, cos, sin, pos = _inputs(9, 2, 1, 64, rot, BF)
        off = [torch.cat((t.new_zeros(1), t.flatten()))[1:].view(t.shape) for t in (cos, sin)]
        for a, x, w in zip(ops.qk_norm_rope(q, k, *off, pos, wq, wk), (q, k), (wq, wk)):
            close(a, *norm_rope(x, w, cos, sin, pos, 1e-6, False), "off")


def test_positions_outside_the_tables():
    ops = _ops()
    q, k, v, wq, wk, cos, sin, pos = _inputs(12, 4, 2, 128, 128, BF)
    pos[2], pos[5], pos[7], pos[11] = -1, 97, 2 ** 40, -(2 ** 40)
    out_of = torch.tensor([2, 5, 7, 11], device="cuda")
    q[2], k[5] = float("nan"), float("inf")  # padding may hold anything
    leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
    out = ops.qk_norm_rope(leaves[0], leaves[1], cos, sin, pos, leaves[2], leaves[3])
    grads = torch.autograd.grad(out, leaves, [torch.ones_like(o) for o in out])
    for t in (*out, *grads[:2]):
        assert not bool(t[out_of].any()) and bool(t[0].any()) and not bool(t.isnan().any())
    keep = torch.ones(12, dtype=torch.bool, device="cuda")
    keep[out_of] = False
    same = [t.detach().requires_grad_() for t in (q[keep], k[keep], wq, wk)]
    o2 = ops.qk_norm_rope(same[0], same[1], cos, sin, pos[keep], same[2], same[3])
    g2 = torch.autograd.grad(o2, same, [torch.ones_like(o) for o in o2])
    for a, b in zip(out, o2):
        assert torch.equal(a[keep], b)
    for x, w, g in ((q, wq, grads[2]), (k, wk, grads[3])):
        close(g, *norm_rope_grads(x[keep], w, cos, sin, pos[keep], 1e-6, False, torch.ones_like(x[keep]))[1], "dw")
    assert torch.equal(g2[0], grads[0][keep])


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("D,rot,dtype", [(128, 128, BF), (80, 32, FH), (10, 6, FF)])
def test_positions_outside_the_tables_beside_weights_that_are_not_finite(D, rot, dtype, bad):
    """Zeros and no gradient are what padding gets, whatever the weights hold."""
    ops = _ops()
    q, k, v, wq, wk, cos, sin, pos = _inputs(9, 4, 2, D, rot, dtype)
    pos[1], pos[4], pos[8] = -1, 97, -7
    pad = torch.tensor([1, 4, 8], device="cuda")
    gs = [torch.randn(x.shape, generator=torch.Generator().manual_seed(1)).to(dtype).cuda() for x in (q, k)]

    def run(wq, wk):
        leaves = [t.detach().clone().requires_grad_() for t in (q, k, wq, wk)]
        out = ops.qk_norm_rope(leaves[0], leaves[1], cos, sin, pos, leaves[2], leaves[3])
        return [o.detach() for o in out] + list(torch.autograd.grad(out, leaves, gs))

    w2 = [w.clone() for w in (wq, wk)]
    w2[0][0] = w2[1][D - 1] = bad
    want, got = run(wq, wk), run(*w2)
    for t in got[:4]:
        assert not bool(t[pad].any()) and bool(t[0].isnan().any() or t[0].isinf().any())
    for a, b in zip(got[4:], want[4:]):  # the weights' gradients do not depend on the weights
        assert torch.equal(a, b)
    if D % 16 or dtype == FF:
        return
    slots = torch.arange(9, device="cuda")
    for kind in (E4, dtype):
        kc, vc, ks, vs = _cache(1, 2, 16, D, kind)
        o = ops.qk_norm_rope_cache_write(q, k, v, cos, sin, pos, kc, vc, slots, ks, vs, q_weight=w2[0], k_weight=w2[1])
        assert not bool(o[pad].any()) and not bool(_rows(kc, pad, 16).any())
        assert ks is None or bool(ks.isfinite().all(0).all(0)[pad].all())


def test_gradient_against_differences():
    ops = _ops()
    q, k, _, wq, wk, cos, sin, pos = _inputs(6, 3, 2, 32, 16, FF)
    leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
    out = ops.qk_norm_rope(leaves[0], leaves[1], cos, sin, pos, leaves[2], leaves[3], eps=EPS)
    gs = [torch.randn_like(o) for o in out]
    grads = torch.autograd.grad(out, leaves, gs)

    def f(*a):
        return sum((norm_rope(x, w, cos, sin, pos, EPS, False)[0] * g.double()).sum() for x, w, g in zip(a[:2], a[2:], gs))

    base = [t.double() for t in (q, k, wq, wk)]
    for n in range(4):
        d = torch.randn(base[n].shape, generator=torch.Generator().manual_seed(n)).cuda().double()
        h = 1e-5
        up, down = (f(*[b + s * h * d if i == n else b for i, b in enumerate(base)]) for s in (1, -1))
        diff = (up - down) / (2 * h)
        got = (grads[n].double() * d).sum()
        # differences: h^2 times the third derivative (of order 10^2 here) and 1e-16 / h of rounding; the
        # kernel: its bound, summed
        side = norm_rope_grads((q, k)[n % 2], (wq, wk)[n % 2], cos, sin, pos, EPS, False, gs[n % 2])
        bound = (side[n // 2][1] + 2.0 ** -24 * side[n // 2][0].abs()) * d.abs()
        assert abs(float(got - diff)) <= float(bound.sum()) + 1e-6


def test_only_what_is_asked_for():
    """One side's gradients, a weight alone, an output that nothing depends on, a gradient that is expanded."""
    ops = _ops()
    q, k, _, wq, wk, cos, sin, pos = _inputs(10, 4, 2, 64, 64, BF)
    ones = torch.ones_like
    for pick in ([0], [1], [2], [3], [0, 3], [1, 2]):
        leaves = [t.detach().clone().requires_grad_(i in pick) for i, t in enumerate((q, k, wq, wk))]
        out = ops.qk_norm_rope(leaves[0], leaves[1], cos, sin, pos, leaves[2], leaves[3])
        (out[0].float().sum() + out[1].float().sum()).backward()
        for i, (x, w) in enumerate(((q, wq), (k, wk))):
            dx, dw = norm_rope_grads(x, w, cos, sin, pos, 1e-6, False, ones(x))
            if i in pick:
                close(leaves[i].grad, *dx, "x")
            if i + 2 in pick:
                close(leaves[i + 2].grad, *dw, "w")
        assert all((t.grad is not None) == (i in pick) for i, t in enumerate(leaves))
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, wq, wk)]
    ops.qk_norm_rope(leaves[0], leaves[1], cos, sin, pos, leaves[2], leaves[3])[0].sum().backward()
    assert bool(leaves[0].grad.any()) and not bool(leaves[1].grad.any()) and not bool(leaves[3].grad.any())
    # expanded: sum()'s gradient has strides of zero
    close(leaves[0].grad, *norm_rope_grads(q, wq, cos, sin, pos, 1e-6, False, ones(q))[0], "expanded")


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("wdtype", [BF, FF])
def test_a_norm_of_one_side(which, wdtype):
    """A weight for the queries or for the keys alone: the other side is only turned."""
    ops = _ops()
    q, k, v, wq, wk, cos, sin, pos = _inputs(21, 6, 2, 64, 32, BF, wdtype=wdtype)
    w = [wq, None] if which == 0 else [None, wk]
    leaves = [None if t is None else t.detach().clone().requires_grad_() for t in (q, k, *w)]
    out = ops.qk_norm_rope(leaves[0], leaves[1], cos, sin, pos, leaves[2], leaves[3], eps=EPS)
    gs = [torch.randn(o.shape, generator=torch.Generator().manual_seed(5)).to(BF).cuda() for o in out]
    torch.autograd.backward(out, gs)
    for n, x, y, g, lx, lw, wx in zip("qk", (q, k), out, gs, leaves[:2], leaves[2:], w):
        close(y.detach(), *norm_rope(x, wx, cos, sin, pos, EPS, False), n)
        dx, dw = norm_rope_grads(x, wx, cos, sin, pos, EPS, False, g)
        close(lx.grad, *dx, "d" + n)
        if wx is not None:
            close(lw.grad, *dw, "dw")
    kc, vc, _, _ = _cache(2, 2, 16, 64, BF)
    slots = torch.arange(21, device="cuda")
    o = ops.qk_norm_rope_cache_write(q, k, v, cos, sin, pos, kc, vc, slots, q_weight=w[0], k_weight=w[1], eps=EPS)
    assert torch.equal(o, out[0]) and torch.equal(_rows(kc, slots, 16), out[1])


def test_no_tokens_no_heads():
    ops = _ops()
    q, k, v, wq, wk, cos, sin, pos = _inputs(4, 2, 1, 32, 32, BF)
    leaves = [t.detach().requires_grad_() for t in (q[:0], k[:0], wq, wk)]
    out = ops.qk_norm_rope(leaves[0], leaves[1], cos, sin, pos[:0], leaves[2], leaves[3])
    assert out[0].shape == (0, 2, 32)
    g = torch.autograd.grad(out, leaves, [torch.ones_like(o) for o in out])
    assert not bool(g[2].any()) and not bool(g[3].any()), "a sum over no tokens is 0"
    a, b = ops.qk_norm_rope(q, k[:, :0], cos, sin, pos, wq, wk)
    assert b.shape == (4, 0, 32) and torch.equal(a, ops.qk_norm_rope(q, k, cos, sin, pos, wq, wk)[0])
    none = [t[:0] for t in (cos, sin)]
    assert not bool(ops.qk_norm_rope(q, k, *none, pos, wq, wk)[0].any())


def test_infinities_and_nan_stay_in_their_rows():
    ops = _ops()
    q, k, _, wq, wk, cos, sin, pos = _inputs(8, 4, 2, 64, 64, BF)
    want = ops.qk_norm_rope(q, k, cos, sin, pos, wq, wk)
    q2 = q.clone()
    q2[3, 1, 5] = float("nan")
    q2[5, 0, 9] = float("inf")
    got = ops.qk_norm_rope(q2, k, cos, sin, pos, wq, wk)
    assert bool(got[0][3, 1].isnan().all()) and bool(got[0][5, 0].isnan().any())
    same = torch.ones(8, 4, dtype=torch.bool, device="cuda")
    same[3, 1] = same[5, 0] = False
    assert torch.equal(got[0][same], want[0][same]) and torch.equal(got[1], want[1])
    zero = torch.zeros_like(q)
    assert not bool(ops.qk_norm_rope(zero, k, cos, sin, pos, wq, wk)[0].any())


def _bits(x):
    return x.contiguous().view(torch.int32 if x.element_size() == 4 else torch.int16)


# runs of 8, 4, 2 and 1 elements
PARTLY = [(128, 64), (256, 128), (80, 24), (64, 4), (10, 6)]


def _partner(j, rot, interleaved):
    """The element that is turned with element j; j itself beyond the turned ones."""
    if j >= rot:
        return j
    return j ^ 1 if interleaved else (j + rot // 2) % rot


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF, FH, FF])
@pytest.mark.parametrize("D,rot", PARTLY)
def test_special_values_reach_their_pair_alone(D, rot, dtype, interleaved):
    """Without a norm an element depends on its pair, and beyond the turned ones on nothing else:
    outputs, gradients, and keys in a cache."""
    ops = _ops()
    q, k, v, _, _, cos, sin, pos = _inputs(6, 3, 2, D, rot, dtype, norm=False)
    gs = [torch.randn(x.shape, generator=torch.Generator().manual_seed(1)).to(dtype).cuda() for x in (q, k)]
    cached = dtype != FF and D % 16 == 0
    slots = torch.arange(6, device="cuda")

    def run(k, gk):
        leaves = [t.detach().clone().requires_grad_() for t in (q, k)]
        out = ops.qk_norm_rope(leaves[0], leaves[1], cos, sin, pos, interleaved=interleaved)
        res = [out[1].detach(), torch.autograd.grad(out, leaves, (gs[0], gk))[1]]
        if cached:
            kc, vc, _, _ = _cache(2, 2, 4, D, dtype)
            ops.qk_norm_rope_cache_write(q, k, v, cos, sin, pos, kc, vc, slots, interleaved=interleaved)
            res.append(_rows(kc, slots, 4))
        return res

    want = run(k, gs[1])
    for j in sorted({0, rot - 1, rot, (rot + D) // 2, D - 1}):
        p = _partner(j, rot, interleaved)
        other = [d for d in range(D) if d not in (j, p)]
        for bad in (float("inf"), -float("inf"), float("nan")):
            k2, g2 = k.clone(), gs[1].clone()
            k2[2, 1, j] = g2[2, 1, j] = bad
            for got, ref in zip(run(k2, g2), want):
                rows = torch.ones(6, 2, dtype=torch.bool, device="cuda")
                rows[2, 1] = False
                assert torch.equal(_bits(got[rows]), _bits(ref[rows]))
                assert torch.equal(_bits(got[2, 1, other]), _bits(ref[2, 1, other])), f"element {j} is {bad}"
                if j >= rot:
                    assert bool(got[2, 1, j].isnan()) if bad != bad else got[2, 1, j].item() == bad


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF, FH, FF])
@pytest.mark.parametrize("D,rot", PARTLY)
def test_special_values_of_normed_rows(D, rot, dtype, interleaved):
    """A norm joins a row's elements: an infinity makes zeros of the others, as the formula does.
    One of a gradient's reaches its own channel of the weight's gradient, and no unrelated one."""
    ops = _ops()
    q, k, _, wq, wk, cos, sin, pos = _inputs(6, 3, 2, D, rot, dtype)
    gs = [torch.randn(x.shape, generator=torch.Generator().manual_seed(1)).to(dtype).cuda() for x in (q, k)]

    def run(k, gk):
        leaves = [t.detach().clone().requires_grad_() for t in (q, k, wq, wk)]
        out = ops.qk_norm_rope(leaves[0], leaves[1], cos, sin, pos, leaves[2], leaves[3], eps=EPS, interleaved=interleaved)
        return [out[1].detach(), *torch.autograd.grad(out, leaves, (gs[0], gk))]

    want = run(k, gs[1])
    for j in sorted({rot, (rot + D) // 2, D - 1}):
        other = [d for d in range(D) if d != j]
        for bad in (float("inf"), -float("inf")):
            k2 = k.clone()
            k2[2, 1, j] = bad
            y = run(k2, gs[1])[0]
            assert bool(y[2, 1, j].isnan()) and not bool(y[2, 1, other].any()), f"element {j} is {bad}"
            g2 = gs[1].clone()
            g2[2, 1, j] = bad
            _, _, dk, _, dw = run(k, g2)
            assert torch.equal(_bits(dw[other]), _bits(want[4][other])) and not bool(dw[j].isfinite()), f"gradient {j} is {bad}"
            ref = norm_rope_grads(k, wk, cos, sin, pos, EPS, interleaved, g2)[0][0]
            assert torch.equal(dk.isnan(), ref.isnan())
            assert torch.equal(dk.isinf(), ref.isinf()) and bool((dk.sign() == ref.sign())[ref.isinf()].all())


def test_offsets_past_32_bits():
    """More than 2^32 bytes of queries, forward and backward: the last tokens' rows are where they belong."""
    ops = _ops()
    T, Hq, D = 540000, 32, 128  # 4.4e9 bytes
    _, k, _, wq, wk, cos, sin, _ = _inputs(6, Hq, 1, D, 128, BF)
    q, g = (torch.empty(T, Hq, D, dtype=BF, device="cuda") for _ in range(2))
    for t in (q, g):
        for i in range(0, T, 90000):
            t[i:i + 90000].normal_()
    k = k[:1].expand(T, 1, D).contiguous()
    pos = torch.arange(T, device="cuda") % 97
    q.requires_grad_()
    y, _ = ops.qk_norm_rope(q, k, cos, sin, pos, wq, wk)
    (dq,) = torch.autograd.grad(y, q, g)
    at = torch.tensor([0, T // 2, T - 3, T - 1], device="cuda")
    x = q.detach()[at].requires_grad_()
    y2, _ = ops.qk_norm_rope(x, k[at], cos, sin, pos[at], wq, wk)
    (dx,) = torch.autograd.grad(y2, x, g[at])
    assert torch.equal(y[at], y2) and torch.equal(dq[at], dx)


def test_no_second_derivative_and_changed_inputs():
    ops = _ops()
    q, k, _, wq, wk, cos, sin, pos = _inputs(3, 2, 1, 32, 32, FF)
    x = q.detach().clone().requires_grad_()
    y = ops.qk_norm_rope(x, k, cos, sin, pos, wq, wk)[0]
    (g,) = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable|differentiate twice"):
        g.sum().backward()
    x = q.detach().clone().requires_grad_()
    z = x * 1
    y = ops.qk_norm_rope(z, k, cos, sin, pos, wq, wk)[0]
    z.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_captured_training_step():
    """Forward and backward in a graph, replayed with new values in place, between eager work."""
    ops = _ops()
    q, k, _, wq, wk, cos, sin, pos = _inputs(130, 8, 2, 128, 64, BF)
    st = [t.detach().clone().requires_grad_() for t in (q, k, wq, wk)]
    gs = [torch.randn(130, h, 128, device="cuda").to(BF) for h in (8, 2)]

    def step():
        out = ops.qk_norm_rope(st[0], st[1], cos, sin, pos, st[2], st[3])
        return [o.detach() for o in out] + list(torch.autograd.grad(out, st, gs))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for n in range(4):
        with torch.no_grad():
            for t in (*st, *gs):
                t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(n)).to(t.dtype))
            pos.copy_(torch.randint(-1, 97, (130,), generator=torch.Generator().manual_seed(n)))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        fresh = [t.detach().clone().requires_grad_() for t in st]
        out = ops.qk_norm_rope(fresh[0], fresh[1], cos, sin, pos, fresh[2], fresh[3])
        want = [o.detach() for o in out] + list(torch.autograd.grad(out, fresh, gs))
        assert all(torch.equal(a, b) for a, b in zip(got, want)), f"replay {n}"


# ---------------------------------------------------------------------------
# into the cache
# ---------------------------------------------------------------------------
def _cache(P, H, page, D, dtype):
    kv = [torch.full((P, H, page, D), 3.0, device="cuda").to(dtype) for _ in range(2)]
    sc = [torch.full((P, H, page), 7.0, device="cuda") for _ in range(2)] if dtype in FP8 else [None, None]
    return kv + sc


def _rows(pool, slots, page):
    x = pool.view(torch.uint8) if pool.element_size() == 1 else pool
    return x[slots // page, :, slots % page]


@pytest.mark.parametrize("norm,interleaved", [(True, False), (False, True), (True, True)])
@pytest.mark.parametrize("dtype", [BF, FH])
@pytest.mark.parametrize("cache", [E4, E5, None])
@pytest.mark.parametrize("T,Hq,Hkv,D,rot,page", [(1, 32, 8, 128, 128, 64), (5, 3, 3, 48, 10, 7), (70, 4, 1, 64, 64, 16), (33, 6, 2, 256, 64, 5),
                                                 (6007, 8, 2, 128, 128, 32), (19, 16, 1, 80, 32, 1)])
def test_cache_write(T, Hq, Hkv, D, rot, page, cache, dtype, norm, interleaved):
    ops = _ops()
    q, k, v, wq, wk, cos, sin, pos = _inputs(T, Hq, Hkv, D, rot, dtype, norm)
    kind = cache or dtype
    P = -(-T // page) + 2
    slots = torch.randperm(P * page, generator=torch.Generator().manual_seed(T))[:T].cuda()
    has = torch.ones(T, dtype=torch.bool, device="cuda")
    if T > 4:
        slots[1], slots[3], has[1], has[3] = -1, P * page, False, False
        pos[2] = -1
    kc, vc, ks, vs = _cache(P, Hkv, page, D, kind)
    out = ops.qk_norm_rope_cache_write(q, k, v, cos, sin, pos, kc, vc, slots, ks, vs, q_weight=wq, k_weight=wk, eps=EPS, interleaved=interleaved)
    close(out, *norm_rope(q, wq, cos, sin, pos, EPS, interleaved), "q")
    at = slots[has]
    # values are what kv_cache_write writes, byte for byte; what has no slot stays
    k2, v2, ks2, vs2 = _cache(P, Hkv, page, D, kind)
    both = ops.qk_norm_rope(q, k, cos, sin, pos, wq, wk, eps=EPS, interleaved=interleaved)
    ops.kv_cache_write(both[1], v, k2, v2, slots, ks2, vs2)
    assert torch.equal(vc.view(torch.uint8), v2.view(torch.uint8)) and (vs is None or torch.equal(vs, vs2))
    rest = torch.ones(P * page, dtype=torch.bool, device="cuda")
    rest[at] = False
    assert bool((kc.float().permute(0, 2, 1, 3).reshape(P * page, Hkv, D)[rest] == 3.0).all())
    want, bound = norm_rope(k[has], wk, cos, sin, pos[has], EPS, interleaved)
    if cache is None:
        assert torch.equal(kc.view(torch.uint8), k2.view(torch.uint8))
        close(_rows(kc, at, page), want, bound, "k")
        return
    most, u, least = FP8[cache]
    amax = want.abs().amax(-1)
    inv = _rows(ks[..., None], at, page)[..., 0].double()
    e = bound.amax(-1)
    # max / amax and 1 / that are two roundings, and 1e-12, where a row is below it, is rounded itself
    amax = amax.clamp(min=1e-12)
    assert bool(((inv - amax / most).abs() <= e / most + 4 * F32 * (amax + e) / most + 1e-45).all())
    got = _rows(kc, at, page).view(cache).double() * inv[..., None]
    # a scaled value carries the key's error and two roundings, then the fp8 one
    assert bool(((got - want).abs() <= bound + e[..., None] + (u + 8 * F32) * (want.abs() + 2 * e[..., None]) + least * inv[..., None]).all())


@pytest.mark.parametrize("cache", [E4, E5])
def test_cache_write_without_norm_or_angle_is_kv_cache_write(cache):
    ops = _ops()
    q, k, v, _, _, cos, sin, pos = _inputs(53, 4, 2, 128, 64, BF, norm=False)
    k = k.clone()
    k[0, 0] = 0
    k[1, 1] = 1e-30
    cos, sin, slots = torch.ones_like(cos), torch.zeros_like(sin), torch.arange(53, device="cuda").to(torch.int32)
    a, b = _cache(4, 2, 16, 128, cache), _cache(4, 2, 16, 128, cache)
    out = ops.qk_norm_rope_cache_write(q, k, v, cos, sin, pos.to(torch.int32), a[0], a[1], slots, a[2], a[3])
    ops.kv_cache_write(k, v, b[0], b[1], slots, b[2], b[3])
    assert torch.equal(out, q) and all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a, b))


@pytest.mark.parametrize("cache", [E4, E5])
@pytest.mark.parametrize("interleaved", [False, True])
def test_cache_write_of_special_values_that_are_not_turned(cache, interleaved):
    ops = _ops()
    q, k, v, _, _, cos, sin, pos = _inputs(6, 4, 2, 128, 64, BF, norm=False)
    k = k.clone()
    k[0, 0, 64], k[1, 1, 127], k[2, 0, 100], k[3, 1, 96] = float("inf"), -float("inf"), float("nan"), float("inf")
    cos, sin, slots = torch.ones_like(cos), torch.zeros_like(sin), torch.arange(6, device="cuda")
    a, b = _cache(1, 2, 16, 128, cache), _cache(1, 2, 16, 128, cache)
    ops.qk_norm_rope_cache_write(q, k, v, cos, sin, pos, a[0], a[1], slots, a[2], a[3], interleaved=interleaved)
    ops.kv_cache_write(k, v, b[0], b[1], slots, b[2], b[3])
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a, b))


def test_cache_write_offsets_past_32_bits_and_no_pages():
    ops = _ops()
    P, H, page, D = 4200, 8, 512, 256  # 4.4e9 bytes a pool
    kc, vc = (torch.zeros((P, H, page, D), dtype=torch.uint8, device="cuda").view(E4) for _ in range(2))
    ks, vs = (torch.ones((P, H, page), device="cuda") for _ in range(2))
    slots = torch.tensor([P * page - 1, (P - 1) * page, 5, (P // 2) * page + 3], device="cuda")
    q, k, v, wq, wk, cos, sin, pos = _inputs(4, 8, 8, 256, 256, BF)
    ops.qk_norm_rope_cache_write(q, k, v, cos, sin, pos, kc, vc, slots, ks, vs, q_weight=wq, k_weight=wk)
    rk, rv = ops.kv_cache_read(kc, vc, slots, ks, vs, out_dtype=FF)
    want, _ = norm_rope(k, wk, cos, sin, pos, 1e-6, False)
    for y, x in ((rk, want), (rv, v.double())):
        assert bool(((y - x).abs() <= 2.0 ** -4 * 1.001 * x.abs().amax(-1, keepdim=True)).all())
    e = _cache(0, 8, 4, 256, E4)
    out = ops.qk_norm_rope_cache_write(q, k, v, cos, sin, pos, e[0], e[1], slots, e[2], e[3])
    assert torch.equal(out, ops.qk_norm_rope(q, k, cos, sin, pos)[0])


def test_cache_write_other_stream_and_captured():
    ops = _ops()
    q, k, v, wq, wk, cos, sin, pos = _inputs(40, 8, 2, 128, 128, BF)
    slots = torch.arange(40, device="cuda")
    want = _cache(3, 2, 16, 128, E4)
    out = ops.qk_norm_rope_cache_write(q, k, v, cos, sin, pos, want[0], want[1], slots, want[2], want[3], q_weight=wq, k_weight=wk)
    s = torch.cuda.Stream()
    got = _cache(3, 2, 16, 128, E4)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        q2 = q * 1
        o2 = ops.qk_norm_rope_cache_write(q2, k, v, cos, sin, pos, got[0], got[1], slots, got[2], got[3], q_weight=wq, k_weight=wk)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(out, o2) and all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, want))
    held = _cache(3, 2, 16, 128, E4)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o3 = ops.qk_norm_rope_cache_write(q, k, v, cos, sin, pos, held[0], held[1], slots, held[2], held[3], q_weight=wq, k_weight=wk)
    for n in range(3):
        slots.copy_(torch.randperm(48, generator=torch.Generator().manual_seed(n))[:40])
        pos.copy_(torch.randint(0, 97, (40,), generator=torch.Generator().manual_seed(n)))
        graph.replay()
        torch.cuda.synchronize()
        eager = [t.clone() for t in held]
        for t in eager:
            t.view(torch.uint8).zero_()
        o4 = ops.qk_norm_rope_cache_write(q, k, v, cos, sin, pos, eager[0], eager[1], slots, eager[2], eager[3], q_weight=wq, k_weight=wk)
        assert torch.equal(o3, o4)
        for a, b in zip(held, eager):
            assert torch.equal(_rows(a if a.dim() == 4 else a[..., None], slots, 16), _rows(b if b.dim() == 4 else b[..., None], slots, 16))
