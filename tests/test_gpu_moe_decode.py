"""moe_decode against the plain 64-bit experts of serving_helpers, element by
element within the bounds of the kernels' arithmetic."""

import pytest
import torch

from serving_helpers import experts, within

pytestmark = pytest.mark.gpu

E4, E5, BF, FH = torch.float8_e4m3fn, torch.float8_e5m2, torch.bfloat16, torch.float16
GRANS = ["TENSORWISE", "ROWWISE", "BLOCKWISE", "NONE"]


def _ops():
    import primus_turbo.pytorch as turbo

    return turbo.ops


def weights(E, I, H, gran, fmt, dtype, seed):
    """Random fp8 (or 16-bit) weights [E, 2I, H], [E, H, I] and their scales, on the GPU."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for N, K in ((2 * I, H), (H, I)):
        w = torch.randn(E, N, K, generator=g) * K ** -0.5
        if gran == "NONE":
            out += [w.to(dtype).cuda(), None]
            continue
        shape = {"TENSORWISE": (), "ROWWISE": (E, N, 1), "BLOCKWISE": (E, -(-N // 128), -(-K // 128))}[gran]
        s = torch.exp(torch.randn(shape, generator=g)) * 0.01
        out += [(w * 100).to(fmt).cuda(), s.cuda()]
    w1, s1, w2, s2 = out
    return w1, w2, s1, s2


def routing(T, E, k, seed, away=0):
    g = torch.Generator().manual_seed(seed)
    top, idx = torch.topk(torch.randn(T, E, generator=g), k, dim=1)
    idx = torch.where(idx < E - away, idx, torch.full_like(idx, -1))
    return idx.cuda(), torch.softmax(top, 1).cuda()


def check(x, w, idx, probs):
    w1, w2, s1, s2 = w
    y = _ops().moe_decode(x, w1, w2, idx, probs, s1, s2)
    want, bound = experts(x, w1, w2, idx, probs, s1, s2)
    assert y.dtype == x.dtype and y.shape == x.shape
    within(y, want, bound, "y")
    assert torch.equal(_ops().moe_decode(x, w1, w2, idx, probs, s1, s2), y), "two calls differ"
    return y


def tokens(T, H, dtype, seed=0):
    return torch.randn(T, H, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


@pytest.mark.parametrize("gran", GRANS)
@pytest.mark.parametrize("dtype,fmt", [(BF, E4), (FH, E4), (BF, E5), (FH, E5)])
@pytest.mark.parametrize("T", [1, 7, 33])
def test_types_and_scales(gran, dtype, fmt, T):
    if gran == "NONE" and fmt == E5:
        pytest.skip("16-bit weights have no fp8 format")
    E, k, I, H = 6, 2, 144, 272
    check(tokens(T, H, dtype), weights(E, I, H, gran, fmt, dtype, T), *routing(T, E, k, T))


@pytest.mark.parametrize("I,H", [(16, 16), (16, 256), (128, 128), (48, 400), (272, 144), (256, 512), (528, 1040)])
@pytest.mark.parametrize("gran", ["BLOCKWISE", "ROWWISE", "NONE"])
def test_sizes(I, H, gran):
    check(tokens(5, H, BF), weights(4, I, H, gran, E4, BF, I), *routing(5, 4, 2, H))


@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 32, 33, 48, 63, 64, 65, 130])
@pytest.mark.parametrize("E,k", [(1, 1), (4, 2), (8, 8), (64, 1)])
def test_token_and_expert_counts(T, E, k):
    check(tokens(T, 64, BF, T), weights(E, 32, 64, "ROWWISE", E4, BF, E), *routing(T, E, k, T * E))


@pytest.mark.parametrize("T,E,k", [(1, 300, 32), (9, 1024, 6), (64, 160, 6)])
def test_many_experts(T, E, k):
    check(tokens(T, 32, BF, T), weights(E, 16, 32, "TENSORWISE", E4, BF, E), *routing(T, E, k, T + E))


@pytest.mark.parametrize("T,E", [(3, 16), (20, 4)])
def test_indices_outside_twice_and_none(T, E):
    """Entries of other ranks, an expert named twice by a token, int32 indices, a
    token without experts, nobody routed at all."""
    w = weights(E, 48, 80, "BLOCKWISE", E4, BF, 1)
    idx, probs = routing(T, E, 4, 3)
    idx[0] = torch.tensor([2, -1, E, 2])
    idx[1] = -1
    idx[2, 3] = 2 ** 40
    y = check(tokens(T, 80, BF), w, idx, probs)
    assert not bool(y[1].any())
    short = torch.where((idx >= 0) & (idx < E), idx, -7).to(torch.int32)
    assert torch.equal(check(tokens(T, 80, BF), w, short, probs), y)
    assert not bool(check(tokens(T, 80, BF), w, torch.full_like(idx, -1), probs).any())


def test_all_tokens_to_one_expert():
    w = weights(8, 64, 128, "BLOCKWISE", E4, BF, 2)
    idx = torch.full((64, 1), 5, device="cuda")
    check(tokens(64, 128, BF), w, idx, torch.rand(64, 1, generator=torch.Generator().manual_seed(0)).cuda())


@pytest.mark.parametrize("gran,fmt", [("ROWWISE", E5), ("NONE", E4)])
@pytest.mark.parametrize("T", [3, 40])
@pytest.mark.parametrize("which", ["up", "down"])
def test_infinite_weights_give_infinite_outputs(gran, fmt, T, which):
    """An infinity at the begin of rows that end inside a step of the contraction."""
    E, k, I, H = 4, 2, 48, 80
    w = weights(E, I, H, gran, fmt, BF, 7)
    inf = torch.tensor(float("inf")).to(w[0].dtype).cuda()
    w[0 if which == "up" else 1][1, I + 5 if which == "up" else 5, 0] = inf
    x, (idx, probs) = tokens(T, H, BF), routing(T, E, k, T)
    y = _ops().moe_decode(x, w[0], w[1], idx, probs, w[2], w[3]).cpu().double()
    want = experts(x, w[0], w[1], idx, probs, w[2], w[3])[0]
    assert bool(torch.isinf(want).any()) and not bool(torch.isnan(want).any())
    assert torch.equal(torch.isnan(y), torch.isnan(want))
    assert torch.equal(y[torch.isinf(want)], want[torch.isinf(want)]) and bool(torch.isfinite(y[torch.isfinite(want)]).all())


@pytest.mark.parametrize("T", [2, 40])
def test_broken_experts_reach_their_tokens_alone(T):
    """NaN in one expert's weights stays with the tokens that go to it."""
    w1, w2, s1, s2 = weights(8, 48, 64, "ROWWISE", E4, BF, 4)
    idx, probs = routing(T, 8, 2, 5)
    idx[0] = torch.tensor([3, 1])
    idx[1:] = torch.where(idx[1:] == 3, 2, idx[1:])
    w1.view(torch.uint8)[3] = 0x7F
    w2.view(torch.uint8)[3] = 0x7F
    y = _ops().moe_decode(tokens(T, 64, BF), w1, w2, idx, probs, s1, s2)
    assert bool(y[0].isnan().all())
    want, bound = experts(tokens(T, 64, BF)[1:], w1, w2, idx[1:], probs[1:], s1, s2)
    within(y[1:], want, bound, "other tokens")


@pytest.mark.parametrize("gran", ["TENSORWISE", "ROWWISE", "BLOCKWISE"])
def test_quantized_tensors_and_the_grouped_layer(gran):
    """Weights from create_quantized_weight, and the same layer by grouped GEMMs'
    dequantized weights."""
    from primus_turbo.pytorch.core.low_precision import Float8QuantConfig, ScalingGranularity
    from primus_turbo.pytorch.core.quantized_tensor import create_quantized_weight

    g = ScalingGranularity[gran]
    cfg = Float8QuantConfig(granularity=g, block_size=128 if gran == "BLOCKWISE" else None)
    hp = [torch.randn(s, generator=torch.Generator().manual_seed(7)).to(BF).cuda() * 0.05 for s in ((4, 512, 256), (4, 256, 256))]
    q1, q2 = (create_quantized_weight(w, E4, cfg)[0] for w in hp)
    x = tokens(6, 256, BF)
    idx, probs = routing(6, 4, 2, 1)
    y = _ops().moe_decode(x, q1, q2, idx, probs)
    assert torch.equal(y, _ops().moe_decode(x, q1.qdata, q2.qdata, idx, probs, q1.scale_inv, q2.scale_inv))
    want, bound = experts(x, q1.qdata, q2.qdata, idx, probs, q1.scale_inv, q2.scale_inv)
    within(y, want, bound, "y")


def test_strides_streams_and_no_tokens():
    w = weights(4, 32, 64, "ROWWISE", E4, BF, 1)
    idx, probs = routing(5, 4, 2, 1)
    x = tokens(5, 64, BF)
    want = check(x, w, idx, probs)
    wide = torch.zeros(5, 200, dtype=BF, device="cuda")
    for off in (8, 3):
        wide[:, off:off + 64] = x
        assert torch.equal(_ops().moe_decode(wide[:, off:off + 64], w[0], w[1], idx, probs, w[2], w[3]), want)
    two = torch.stack([idx, idx], 2)[:, :, 0], torch.stack([probs, probs], 2)[:, :, 1]
    assert torch.equal(_ops().moe_decode(x, w[0], w[1], *two, w[2], w[3]), want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = _ops().moe_decode(x * 1, w[0], w[1], idx, probs, w[2], w[3])
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(y, want)
    assert _ops().moe_decode(x[:0], w[0], w[1], idx[:0], probs[:0], w[2], w[3]).shape == (0, 64)


def test_graph_replay_with_new_routing():
    w = weights(8, 64, 128, "BLOCKWISE", E4, BF, 3)
    for T in (2, 24):
        x = tokens(T, 128, BF)
        idx, probs = routing(T, 8, 2, 0)
        call = lambda: _ops().moe_decode(x, w[0], w[1], idx, probs, w[2], w[3])  # noqa: E731
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            call()
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        for i in range(4):
            a, b = routing(T, 8, 2, i + 1, away=i % 2)
            idx.copy_(a)
            probs.copy_(b)
            x.copy_(tokens(T, 128, BF, i))
            want = call().clone()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want), f"replay {i}"


@pytest.mark.parametrize("T,E,k", [(65, 256, 3), (130, 6, 4), (200, 1024, 2), (129, 300, 8), (1000, 16, 2)])
def test_several_groups_of_tokens(T, E, k):
    """More tokens than a pass takes, whose rows between the products lie close together:
    experts that nobody reaches, entries of other ranks, an expert named twice by a token."""
    idx, probs = routing(T, E, k, T, away=E // 5)
    idx[1, k - 1] = idx[1, 0]
    idx[T - 1, 0] = idx[T - 1, 1]
    idx[64:, :][idx[64:, :] == E // 2] = -1
    idx[5] = -1
    check(tokens(T, 48, BF, T), weights(E, 32, 48, "ROWWISE", E4, BF, E), idx, probs)
