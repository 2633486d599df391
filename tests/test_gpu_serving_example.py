"""The serving example: every operator call that it makes is checked against the
plain 64-bit implementations, on the inputs of that call."""

import importlib.util
import os

import pytest
import torch

from serving_helpers import attention, experts, within

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(__file__), "..", "primus-turbo_amd", "examples", "serve_moe_layer.py")


class Checked:
    """turbo.ops whose serving operators are checked as they are called."""

    def __init__(self):
        import primus_turbo.pytorch as turbo

        self.ops, self.calls = turbo.ops, []

    def __getattr__(self, name):
        self.calls.append(name)
        return getattr(self.ops, name)

    def kv_cache_write(self, k, v, kc, vc, slots, ks, vs):
        self.calls.append("kv_cache_write")
        self.ops.kv_cache_write(k, v, kc, vc, slots, ks, vs)
        for x, got in zip((k, v), self.ops.kv_cache_read(kc, vc, slots, ks, vs, out_dtype=torch.float32)):
            top = x.abs().amax(2, keepdim=True).double().cpu()
            # an e4m3 step is 2^-3 of the binade below: half of it, or half the smallest
            # step at the row's scale; and the fp32 scale's own roundings
            bound = x.abs().double().cpu() * (2.0 ** -4 + 2.0 ** -20) + top / 448 * 2.0 ** -10 * 1.001
            within(got, x.cpu().double(), bound, "cache rows")

    def paged_attention(self, q, kc, vc, table, cu, lens, ks, vs):
        self.calls.append("paged_attention")
        out = self.ops.paged_attention(q, kc, vc, table, cu, lens, ks, vs)
        want, _, bound, _ = attention(q, kc.cpu(), vc.cpu(), ks, vs, table, cu, lens, q.shape[2] ** -0.5, None, 0)
        within(out, want, bound, "attention")
        return out

    def moe_decode(self, x, w1, w2, idx, probs):
        self.calls.append("moe_decode")
        y = self.ops.moe_decode(x, w1, w2, idx, probs)
        want, bound = experts(x, w1.qdata, w2.qdata, idx, probs, w1.scale_inv, w2.scale_inv)
        within(y, want, bound, "experts")
        return y


def test_prompts_chunks_and_single_tokens_together():
    spec = importlib.util.spec_from_file_location("serve_moe_layer", PATH)
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    torch.manual_seed(1)
    ops = Checked()
    layer = ex.ServedLayer(256, 4, 2, 64, 4, 2, 128, ops=ops)
    cache = ex.PagedCache(24, 2, 16, 64)
    a, b, c = (cache.add_sequence() for _ in range(3))
    tok = lambda n: torch.randn(n, 256, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    for seqs, new in (([a, b], [40, 5]), ([a, b, c], [1, 1, 90]), ([b, c], [1, 1]), ([a, b, c], [1, 1, 1])):
        y = layer(tok(sum(new)), cache, seqs, new)
        assert y.shape == (sum(new), 256) and bool(torch.isfinite(y).all())
    assert cache.lens == [42, 8, 92]
    cache.drop_sequence(c)
    assert bool(torch.isfinite(layer(tok(20), cache, [cache.add_sequence()], [20])).all())
    assert {"kv_cache_write", "paged_attention", "moe_decode", "moe_permute", "grouped_gemm_fp8", "moe_unpermute"} <= set(ops.calls)
