"""Argument checks of the serving operators, before any GPU work (CPU), and of
their C entries."""

import ctypes

import pytest
import torch

E4, BF, FH = torch.float8_e4m3fn, torch.bfloat16, torch.float16


def _ops():
    import primus_turbo.pytorch as turbo

    return turbo.ops


def z(*shape, dtype=BF):
    return torch.zeros(shape, dtype=torch.uint8).view(dtype) if dtype == E4 else torch.zeros(shape, dtype=dtype)


def cache_args(**over):
    """A valid kv_cache_write call on CPU tensors, with replacements."""
    a = dict(k=z(3, 2, 32), v=z(3, 2, 32), k_cache=z(4, 2, 8, 32, dtype=E4), v_cache=z(4, 2, 8, 32, dtype=E4),
             slots=z(3, dtype=torch.int64), k_scale_inv=z(4, 2, 8, dtype=torch.float32),
             v_scale_inv=z(4, 2, 8, dtype=torch.float32))
    return a | over


def attn_args(**over):
    a = cache_args()
    a = dict(q=z(3, 4, 32), k_cache=a["k_cache"], v_cache=a["v_cache"], page_table=z(2, 3, dtype=torch.int32),
             cu_seqlens_q=z(3, dtype=torch.int32), seq_lens=z(2, dtype=torch.int32), k_scale_inv=a["k_scale_inv"],
             v_scale_inv=a["v_scale_inv"])
    return a | over


def moe_args(**over):
    a = dict(x=z(3, 64), w_gate_up=z(4, 96, 64, dtype=E4), w_down=z(4, 64, 48, dtype=E4), topk_idx=z(3, 2, dtype=torch.int64),
             topk_probs=z(3, 2, dtype=torch.float32), gate_up_scale_inv=z(4, 96, 1, dtype=torch.float32),
             down_scale_inv=z(4, 64, 1, dtype=torch.float32))
    return a | over


def refused(fn, args, match, error=AssertionError):
    with pytest.raises(error, match=match):
        fn(**args)


def no_gpu(fn, args):
    if torch.cuda.is_available():
        pytest.skip("checks what happens without a GPU")
    refused(fn, args, "need a ROCm GPU", RuntimeError)


@pytest.mark.parametrize("over,match", [
    (dict(k_cache=z(4, 2, 8, 32)), "one type"),
    (dict(k_cache=z(4, 2, 32, dtype=E4)), "num_pages, Hkv"),
    (dict(v_cache=z(4, 2, 4, 32, dtype=E4)), "both alike"),
    (dict(k_scale_inv=None), "needs k_scale_inv"),
    (dict(v_scale_inv=z(4, 2, 7, dtype=torch.float32)), "scale_inv must be"),
    (dict(k=z(3, 2, 16)), "k and v must be"),
    (dict(v=z(3, 2, 32, dtype=FH)), "one type"),
    (dict(slots=z(3, dtype=torch.float32)), "slots must be"),
    (dict(slots=z(2, dtype=torch.int64)), "one slot for each"),
    (dict(k=z(3, 2, 32).requires_grad_()), "no backward"),
    (dict(slots=torch.zeros(3, dtype=torch.int64, device="meta")), "all tensors must be on"),
])
def test_write_refuses(over, match):
    refused(_ops().kv_cache_write, cache_args(**over), match)


def test_cache_layouts_refused():
    ops = _ops()
    t = z(4, 2, 32, 8, dtype=E4).transpose(2, 3)
    refused(ops.kv_cache_write, cache_args(k_cache=t, v_cache=t), "contiguous")
    for D in (8, 24, 272):
        c = z(4, 2, 8, D, dtype=E4)
        refused(ops.kv_cache_write, cache_args(k_cache=c, v_cache=c), "multiple of 16")
    c = z(4, 2, 8, 32)
    refused(ops.kv_cache_write, cache_args(k_cache=c, v_cache=c), "has no scales")
    refused(ops.kv_cache_write, cache_args(k_cache=c, v_cache=c, k_scale_inv=None, v_scale_inv=None, k=z(3, 2, 32, dtype=FH),
                                           v=z(3, 2, 32, dtype=FH)), "values of its type")
    c = z(4, 2, 8, 32, dtype=torch.float32)
    refused(ops.kv_cache_write, cache_args(k_cache=c, v_cache=c), "unsupported cache type")


def test_read_refuses():
    ops = _ops()
    a = {n: x for n, x in cache_args().items() if n not in ("k", "v")}
    refused(ops.kv_cache_read, a | dict(slots=z(3, 1, dtype=torch.int64)), "slots must be")
    refused(ops.kv_cache_read, a | dict(slots=z(6, dtype=torch.int64)[::2]), "contiguous")
    refused(ops.kv_cache_read, a | dict(out_dtype=torch.int32), "unsupported", TypeError)
    c = z(4, 2, 8, 32)
    refused(ops.kv_cache_read, a | dict(k_cache=c, v_cache=c, k_scale_inv=None, v_scale_inv=None, out_dtype=FH), "read back as it is")
    no_gpu(ops.kv_cache_read, a)


@pytest.mark.parametrize("over,match", [
    (dict(q=z(3, 4, 16)), "q must be"),
    (dict(q=z(3, 4, 32, dtype=torch.float32)), "bfloat16 or float16"),
    (dict(q=z(3, 3, 32)), "multiple of cache heads"),
    (dict(seq_lens=z(2, dtype=torch.int64)), "seq_lens must be"),
    (dict(cu_seqlens_q=z(2, dtype=torch.int32)), "cu_seqlens_q must be"),
    (dict(page_table=z(1, 3, dtype=torch.int32)), "page_table must be"),
    (dict(page_table=z(2, 6, dtype=torch.int32)[:, ::2]), "rows of page_table"),
    (dict(window_size=0), "window_size must be"),
    (dict(window_size=8, num_sinks=-1), "num_sinks"),
    (dict(softmax_scale=float("inf")), "finite"),
    (dict(q=z(3, 4, 32).requires_grad_()), "no backward"),
    (dict(page_table=z(0, 3, dtype=torch.int32), seq_lens=z(0, dtype=torch.int32), cu_seqlens_q=z(1, dtype=torch.int32)),
     "without a sequence"),
])
def test_attention_refuses(over, match):
    refused(_ops().paged_attention, attn_args(**over), match)


@pytest.mark.parametrize("over,match", [
    (dict(x=z(3, 64, dtype=torch.float32)), "x must be"),
    (dict(w_gate_up=z(4, 64, 64, dtype=E4)), "weights must be"),
    (dict(w_down=z(4, 64, 48)), "one kind"),
    (dict(down_scale_inv=None), "one kind"),
    (dict(gate_up_scale_inv=None, down_scale_inv=None), "fp8 with scale_inv"),
    (dict(w_gate_up=z(4, 96, 64), w_down=z(4, 64, 48)), "must be fp8"),
    (dict(gate_up_scale_inv=z(4, 95, 1, dtype=torch.float32)), "scale_inv must be one value"),
    (dict(down_scale_inv=z(1, dtype=torch.float32)), "one granularity"),
    (dict(topk_idx=z(2, 2, dtype=torch.int64)), "topk_idx must be"),
    (dict(topk_probs=z(3, 2)), "topk_probs must be"),
    (dict(topk_idx=z(3, 0, dtype=torch.int64), topk_probs=z(3, 0, dtype=torch.float32)), "1 to 32 experts"),
    (dict(x=z(3, 64).requires_grad_()), "no backward"),
])
def test_moe_refuses(over, match):
    refused(_ops().moe_decode, moe_args(**over), match)


def test_moe_refuses_sizes():
    for I, H in ((40, 64), (48, 72)):
        refused(_ops().moe_decode, moe_args(x=z(3, H), w_gate_up=z(4, 2 * I, H), w_down=z(4, H, I), gate_up_scale_inv=None,
                                            down_scale_inv=None), "multiples of 16")


def test_without_a_gpu():
    no_gpu(_ops().kv_cache_write, cache_args())
    no_gpu(_ops().paged_attention, attn_args())
    no_gpu(_ops().moe_decode, moe_args())


def test_c_entries_refuse():
    from primus_turbo.pytorch import _C

    p = ctypes.c_void_p(256)  # never dereferenced: the checks reject first
    with pytest.raises(RuntimeError, match="multiple of 16"):
        _C.call("pta_kv_cache_write", p, p, 2, 1, 1, 24, 24, 24, 24, 24, p, 0, p, p, 0, 1, 8, p, p, None)
    with pytest.raises(RuntimeError, match="2\\^31 rows"):
        _C.call("pta_kv_cache_write", p, p, 2, 1, 8, 32, 32, 32, 32, 32, p, 0, p, p, 0, 1 << 24, 64, p, p, None)
    with pytest.raises(RuntimeError, match="needs its scales"):
        _C.call("pta_kv_cache_read", p, p, 0, 4, 8, 1, 32, None, p, p, 0, 1, p, p, 2, None)
    with pytest.raises(RuntimeError, match="read back as it is"):
        _C.call("pta_kv_cache_read", p, p, 2, 4, 8, 1, 32, None, None, p, 0, 1, p, p, 0, None)

    def attn(T=4, Hq=4, D=64, st=256, kind=0, Hkv=2, scale=1.0, win=0, q=p, ws=None):
        _C.call("pta_paged_attention", q, 2, T, Hq, D, st, 64, p, p, kind, 8, 16, Hkv, p, p, p, 4, 4, p, p, 2, scale, win, 0,
                p, None, ws, 0, None)

    for kw, match in ((dict(kind=7), "unknown cache kind"), (dict(Hkv=3), "multiple of cache heads"), (dict(D=300), "head_dim"),
                      (dict(st=257), "multiples of 8"), (dict(win=-1), "negative"), (dict(scale=float("nan")), "finite"),
                      (dict(q=None), "null pointer"), (dict(T=1 << 31), "too many tokens")):
        with pytest.raises(RuntimeError, match=match):
            attn(**kw)

    def moe(T=1, E=4, k=2, I=32, H=64, kind=0, gran=2, ws=p, n=1 << 30):
        _C.call("pta_moe_decode", p, 2, T, H, H, p, p, kind, p, p, gran, E, I, p, 1, p, k, p, ws, n, None)

    for kw, match in ((dict(kind=2), "does not fit"), (dict(gran=4), "does not fit"), (dict(E=2000), "num_experts"), (dict(k=33), "topk"),
                      (dict(I=40), "multiples of 16"), (dict(ws=None), "workspace too small"), (dict(n=16), "workspace too small")):
        with pytest.raises(RuntimeError, match=match):
            moe(**kw)


def test_workspace_sizes():
    from primus_turbo.pytorch import _C

    assert _C.query("pta_moe_decode_workspace_size", 0, 8, 2, 64) == 0
    assert _C.query("pta_moe_decode_workspace_size", 3, 8, 2, 64) == 6 * 3 * 64 * 2      # a slot for each entry
    assert _C.query("pta_moe_decode_workspace_size", 64, 8, 2, 64) == 8 * 64 * 64 * 2    # a slot for each expert
    q = lambda *a: _C.query("pta_paged_attention_workspace_size", *a)  # noqa: E731
    assert q(0, 1, 8, 8, 64, 4, 16) == 0
    assert q(1, 1, 8, 8, 64, 1, 16) == 0              # one key tile: nothing to split
    assert q(1, 1, 8, 8, 64, 1000, 16) > 0            # few rows, many keys
    assert q(1 << 16, 1, 64, 8, 64, 1000, 16) == 0    # rows alone fill the chip


def test_cpu_tensors_are_refused_beside_a_gpu(monkeypatch):
    """Where a GPU is there, tensors in host memory must not reach a kernel."""
    from primus_turbo.pytorch import _C

    def launch(name, *args):
        raise RuntimeError(f"{name} was launched on host memory")

    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(_C, "stream", lambda device=None: 0)
    monkeypatch.setattr(_C, "call", launch)
    read = {n: x for n, x in cache_args().items() if n not in ("k", "v")}
    for fn, args in ((_ops().kv_cache_write, cache_args()), (_ops().kv_cache_read, read), (_ops().paged_attention, attn_args()),
                     (_ops().moe_decode, moe_args())):
        refused(fn, args, "must be GPU tensors")


@pytest.mark.parametrize("T,B,Hq,Hkv,D,keys", [(8193, 2, 64, 8, 128, 8192), (16384, 2, 64, 8, 128, 16384), (8193, 2, 64, 1, 128, 32768),
                                               (32769, 2, 8, 1, 128, 32768), (2049, 2, 32, 8, 128, 16384)])
def test_workspace_of_prompts_beside_single_tokens(T, B, Hq, Hkv, D, keys):
    """Long prompts in a batch of several sequences: their rows have no parts among the
    few rows' ones."""
    from primus_turbo.pytorch import _C

    size = _C.query("pta_paged_attention_workspace_size", T, B, Hq, Hkv, D, keys // 64, 64)
    assert size <= max(16 << 20, 2 * T * Hq * D)


def test_workspace_without_few_rows():
    """Beyond 16 query heads to a cache head no token has few rows: its form has no parts."""
    from primus_turbo.pytorch import _C

    q = lambda *a: _C.query("pta_paged_attention_workspace_size", *a)  # noqa: E731
    assert q(8193, 2, 64, 1, 128, 512, 64) == 0   # row tiles alone fill the chip
    assert q(8193, 2, 136, 8, 64, 512, 64) == 0
    assert q(8193, 2, 128, 8, 64, 512, 64) > 0    # 16 heads: a single token is 16 rows


@pytest.mark.parametrize("T,B,Hq,Hkv,D,keys", [(1001, 1000, 16, 16, 256, 4096), (1500, 1000, 16, 16, 256, 4096), (192, 64, 64, 8, 128, 16384),
                                               (3000, 170, 8, 8, 128, 32768), (40, 1, 8, 2, 256, 32768), (300, 16, 16, 16, 64, 4096)])
def test_workspace_of_many_sequences(T, B, Hq, Hkv, D, keys):
    """Parts of 4 D + 8 bytes a row: row tiles of 128 for less than twice the chunks that fill
    256 CUs twice, and at least four of few rows, no more than tokens and what fills the CUs."""
    from primus_turbo.pytorch import _C

    size = _C.query("pta_paged_attention_workspace_size", T, B, Hq, Hkv, D, keys // 64, 64)
    rows = 2 * (512 + Hkv) * 128 + 4 * T * Hq + 512 * max(16, Hq // Hkv) + T * Hq
    assert size <= rows * (4 * D + 8) + 16 * (T * Hq // Hkv // 128 + B + 512) + 1024


@pytest.mark.parametrize("T,E,k,I", [(4096, 256, 8, 2048), (512, 256, 8, 2048), (65, 1024, 1, 64), (1000, 8, 2, 1024)])
def test_expert_workspace_of_many_tokens(T, E, k, I):
    """A row of 16 bit for each entry of topk_idx, whatever the number of experts."""
    from primus_turbo.pytorch import _C

    assert _C.query("pta_moe_decode_workspace_size", T, E, k, I) <= T * k * I * 2


def _calls_with_floats():
    """(entry, arguments, name of one floating tensor) for every one of the four calls."""
    h = dict(k_cache=z(4, 2, 8, 32), v_cache=z(4, 2, 8, 32), k_scale_inv=None, v_scale_inv=None)
    w = dict(w_gate_up=z(4, 96, 64), w_down=z(4, 64, 48), gate_up_scale_inv=None, down_scale_inv=None)
    read = {n: x for n, x in cache_args(**h).items() if n not in ("k", "v")}
    ops = _ops()
    out = [(ops.kv_cache_write, cache_args(**h), n) for n in ("k", "v", "k_cache", "v_cache")]
    out += [(ops.kv_cache_read, read, n) for n in ("k_cache", "v_cache")]
    out += [(ops.paged_attention, attn_args(**h), n) for n in ("q", "k_cache", "v_cache")]
    out += [(ops.moe_decode, moe_args(**w), n) for n in ("x", "topk_probs", "w_gate_up", "w_down")]
    out += [(ops.kv_cache_write, cache_args(), "k_scale_inv"), (ops.paged_attention, attn_args(), "v_scale_inv"),
            (ops.moe_decode, moe_args(), "down_scale_inv")]
    return out


def test_gradients_are_refused_not_dropped():
    """16-bit caches and weights that need gradients, as queries and tokens that do."""
    for fn, args, name in _calls_with_floats():
        args = args | {name: args[name].detach().clone().requires_grad_()}
        refused(fn, args, "no backward")
        with torch.no_grad():  # refused for another reason, or not at all
            if not torch.cuda.is_available():
                refused(fn, args, "need a ROCm GPU", RuntimeError)


def test_forward_mode_tangents_are_refused_not_dropped():
    import torch.autograd.forward_ad as fwad

    for fn, args, name in _calls_with_floats():
        with fwad.dual_level(), torch.no_grad():
            t = args[name]
            refused(fn, args | {name: fwad.make_dual(t, torch.ones_like(t))}, "no forward-mode derivative")


def test_quantized_weights_that_need_gradients_are_refused():
    from primus_turbo.pytorch.core.low_precision import ScalingGranularity
    from primus_turbo.pytorch.core.quantized_tensor import QuantizedTensor

    def make(N, K, grad):
        return QuantizedTensor(z(4, N, K, dtype=E4), z(4, N, 1, dtype=torch.float32), shape=(4, N, K), orig_dtype=BF, dest_dtype=E4,
                               granularity=ScalingGranularity.ROWWISE, quantized_axis=2, requires_grad=grad)

    none = dict(gate_up_scale_inv=None, down_scale_inv=None)
    refused(_ops().moe_decode, moe_args(w_gate_up=make(96, 64, False), w_down=make(64, 48, True), **none), "no backward")
    no_gpu(_ops().moe_decode, moe_args(w_gate_up=make(96, 64, False), w_down=make(64, 48, False), **none))


def test_a_written_cache_counts_as_changed(monkeypatch):
    """What autograd has saved of a pool is not used after the pool was written."""
    from primus_turbo.pytorch import _C

    done = []
    monkeypatch.setattr(_C, "stream", lambda device=None: 0)
    monkeypatch.setattr(_C, "call", lambda name, *args: done.append(name))
    a = cache_args()
    pools = [a[n] for n in ("k_cache", "v_cache", "k_scale_inv", "v_scale_inv")]
    before = [p._version for p in pools]
    monkeypatch.setattr(torch.cuda, "is_available", lambda: False)
    _ops().kv_cache_write(**a)
    assert done == ["pta_kv_cache_write"] and all(p._version > b for p, b in zip(pools, before))
    c = z(4, 2, 8, 32)
    w = torch.ones(32, dtype=BF, requires_grad=True)
    y = (w * c).sum()
    _ops().kv_cache_write(**cache_args(k_cache=c, v_cache=z(4, 2, 8, 32), k_scale_inv=None, v_scale_inv=None))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        i = cache_args(**{n: x.clone() for n, x in a.items() if n in ("k_cache", "v_cache", "k_scale_inv", "v_scale_inv")})
    _ops().kv_cache_write(**i)  # inference tensors have no version


def test_fake_tensors_are_refused(monkeypatch):
    """Fake tensors have no memory, and views of them addresses that are not null."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    from primus_turbo.pytorch import _C

    done = []
    monkeypatch.setattr(_C, "stream", lambda device=None: 0)
    monkeypatch.setattr(_C, "call", lambda name, *args: done.append(name))
    read = {n: x for n, x in cache_args().items() if n not in ("k", "v")}
    for fn, args in ((_ops().kv_cache_write, cache_args()), (_ops().kv_cache_read, read), (_ops().paged_attention, attn_args()),
                     (_ops().moe_decode, moe_args())):
        with FakeTensorMode() as mode:
            refused(fn, {n: mode.from_tensor(x) for n, x in args.items()}, "fake tensors")
    assert not done
