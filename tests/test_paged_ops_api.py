"""Argument checks of the operators around the paged cache, before any GPU work
(CPU), and of their C entries."""

import ctypes

import pytest
import torch

from paged_ops_helpers import fork_books

E4, BF, FH, FF = torch.float8_e4m3fn, torch.bfloat16, torch.float16, torch.float32
I32, I64 = torch.int32, torch.int64


def _ops():
    import primus_turbo.pytorch as turbo

    return turbo.ops


def z(*shape, dtype=BF):
    return torch.zeros(shape, dtype=torch.uint8).view(dtype) if dtype == E4 else torch.zeros(shape, dtype=dtype)


def rope_args(**over):
    return dict(q=z(3, 4, 32), k=z(3, 2, 32), cos=z(9, 8, dtype=FF), sin=z(9, 8, dtype=FF), positions=z(3, dtype=I64), q_weight=z(32),
                k_weight=z(32)) | over


def pools():
    return dict(k_cache=z(4, 2, 8, 32, dtype=E4), v_cache=z(4, 2, 8, 32, dtype=E4), k_scale_inv=z(4, 2, 8, dtype=FF),
                v_scale_inv=z(4, 2, 8, dtype=FF))


def enter_args(**over):
    return rope_args() | dict(v=z(3, 2, 32), slots=z(3, dtype=I64)) | pools() | over


def copy_args(**over):
    return pools() | dict(src_pages=z(2, dtype=I32), dst_pages=z(2, dtype=I32)) | over


def fork_args(**over):
    return pools() | dict(page_table=z(2, 3, dtype=I32), seq_lens=z(2, dtype=I32), parents=z(3, dtype=I64)) | over


def ranges_args(**over):
    return dict(k_cache=z(4, 2, 8, 32, dtype=E4), page_table=z(2, 3, dtype=I32), cu_seqlens_q=z(3, dtype=I32), seq_lens=z(2, dtype=I32),
                key_ranges=z(4, 2, 2, 32), k_scale_inv=z(4, 2, 8, dtype=FF)) | over


def sparse_args(**over):
    return ranges_args() | pools() | dict(q=z(3, 4, 32), num_selected=4) | over


def select_args(**over):
    return dict(q=z(3, 4, 32), key_ranges=z(4, 2, 2, 32), page_table=z(2, 3, dtype=I32), cu_seqlens_q=z(3, dtype=I32),
                seq_lens=z(2, dtype=I32), page_size=8, num_selected=4) | over


def _all():
    o = _ops()
    return ((o.qk_norm_rope, rope_args()), (o.qk_norm_rope_cache_write, enter_args()), (o.kv_cache_copy, copy_args()),
            (o.kv_cache_fork, fork_args()), (o.kv_page_ranges, ranges_args()), (o.select_pages, select_args()),
            (o.sparse_paged_attention, sparse_args()))


def refused(fn, args, match, error=AssertionError):
    with pytest.raises(error, match=match):
        fn(**args)


@pytest.mark.parametrize("over,match,error", [
    (dict(q=z(3, 4, 30)), "same tokens and D", AssertionError),
    (dict(k=z(2, 2, 32)), "same tokens and D", AssertionError),
    (dict(k=z(3, 2, 32, dtype=FH)), "one type", AssertionError),
    (dict(q=z(3, 4, 32, dtype=torch.float64), k=z(3, 2, 32, dtype=torch.float64)), "unsupported type", TypeError),
    (dict(q=z(32), k=z(32)), "heads, D", AssertionError),
    (dict(q=z(3, 4, 33), k=z(3, 2, 33)), "even", AssertionError),
    (dict(q=z(3, 4, 258), k=z(3, 2, 258)), "at most 256", AssertionError),
    (dict(sin=z(9, 7, dtype=FF)), "both alike", AssertionError),
    (dict(cos=z(9, 8)), "contiguous float32", AssertionError),
    (dict(cos=z(9, 17, dtype=FF), sin=z(9, 17, dtype=FF)), "turn 34 elements", AssertionError),
    (dict(cos=z(9, 0, dtype=FF), sin=z(9, 0, dtype=FF)), "turn 0 elements", AssertionError),
    (dict(positions=z(2, dtype=I64)), "positions must be", AssertionError),
    (dict(positions=z(3, dtype=FF)), "positions must be", AssertionError),
    (dict(q_weight=z(31)), "a weight must be", AssertionError),
    (dict(k_weight=z(64)[::2]), "a weight must be", AssertionError),
    (dict(k_weight=z(32, dtype=I32)), "unsupported weight", TypeError),
    (dict(eps=-1.0), "eps must be", AssertionError),
    (dict(eps=float("nan")), "eps must be", AssertionError),
    (dict(cos=z(9, 8, dtype=FF).requires_grad_()), "no gradients", AssertionError),
    (dict(sin=torch.zeros(9, 8, device="meta")), "all tensors must be on", AssertionError),
])
def test_qk_norm_rope_refuses(over, match, error):
    refused(_ops().qk_norm_rope, rope_args(**over), match, error)


@pytest.mark.parametrize("over,match", [
    (dict(q=z(3, 4, 64)), "q must be"),
    (dict(q=z(6, 32)), "q must be"),
    (dict(k=z(3, 4, 32)), "k and v must be"),
    (dict(v=z(3, 2, 16)), "k and v must be"),
    (dict(q=z(3, 4, 32, dtype=FF)), "bfloat16 or float16"),
    (dict(v=z(3, 2, 32, dtype=FH)), "one type"),
    (dict(k_cache=z(4, 2, 8, 32, dtype=FH), v_cache=z(4, 2, 8, 32, dtype=FH), k_scale_inv=None, v_scale_inv=None), "values of its type"),
    (dict(k_scale_inv=None), "needs k_scale_inv"),
    (dict(slots=z(4, dtype=I64)), "one slot for each"),
    (dict(positions=z(6, dtype=I64)[::2]), "positions must be contiguous"),
    (dict(positions=z(4, dtype=I64)), "positions must be"),
    (dict(q_weight=z(16)), "a weight must be"),
    (dict(cos=z(9, 20, dtype=FF), sin=z(9, 20, dtype=FF)), "turn 40 elements"),
    (dict(eps=float("inf")), "eps must be"),
    (dict(k=z(3, 2, 32).requires_grad_()), "no backward"),
    (dict(k_weight=z(32).requires_grad_()), "no backward"),
    (dict(cos=z(9, 8, dtype=FF).requires_grad_()), "no backward"),
])
def test_cache_write_refuses(over, match):
    refused(_ops().qk_norm_rope_cache_write, enter_args(**over), match)


@pytest.mark.parametrize("over,match", [
    (dict(src_pages=z(3, dtype=I32)), "one type and length"),
    (dict(src_pages=z(2, dtype=I64)), "one type and length"),
    (dict(src_pages=z(2, dtype=FF), dst_pages=z(2, dtype=FF)), "int32 / int64"),
    (dict(src_pages=z(1, 2, dtype=I32), dst_pages=z(1, 2, dtype=I32)), "one-dimensional"),
    (dict(src_pages=z(4, dtype=I32)[::2], dst_pages=z(4, dtype=I32)[::2]), "contiguous"),
    (dict(v_cache=z(3, 2, 8, 32, dtype=E4)), "both alike"),
    (dict(k_cache=z(2, 4, 2, 8, 32, dtype=E4)), "both alike"),
    (dict(k_cache=z(2, 4, 2, 8, 32, dtype=E4), v_cache=z(2, 4, 2, 8, 32, dtype=E4)), "scale_inv must be"),
    (dict(k_cache=z(4, 3, 2, 8, 32, dtype=E4).transpose(0, 1), v_cache=z(4, 3, 2, 8, 32, dtype=E4).transpose(0, 1)), "contiguous"),
    (dict(k_cache=z(2, 4, 2, 8, 24, dtype=E4), v_cache=z(2, 4, 2, 8, 24, dtype=E4)), "multiple of 16"),
    (dict(k_cache=z(2, 4, 2, 8, 32), v_cache=z(2, 4, 2, 8, 32)), "has no scales"),
    (dict(k_cache=z(2, 4, 2, 8, 32, dtype=FF), v_cache=z(2, 4, 2, 8, 32, dtype=FF)), "unsupported cache type"),
    (dict(k_cache=z(2, 4, 2, 8, 32), v_cache=z(2, 4, 2, 8, 32, dtype=FH)), "one type"),
    (dict(k_cache=z(2, 4, 2, 8, 32, dtype=E4), v_cache=z(2, 4, 2, 8, 32, dtype=E4), v_scale_inv=None), "needs k_scale_inv"),
    (dict(k_cache=z(8, 32, dtype=E4), v_cache=z(8, 32, dtype=E4)), "both alike"),
    (dict(key_ranges=z(4, 2, 2, 16)), "key_ranges must be"),
    (dict(key_ranges=z(4, 2, 2, 32, dtype=FH)), "key_ranges must be"),
    (dict(k_scale_inv=z(4, 2, 8, dtype=FF).requires_grad_()), "no backward"),
])
def test_copy_refuses(over, match):
    refused(_ops().kv_cache_copy, copy_args(**over), match)


@pytest.mark.parametrize("over,match", [
    (dict(page_table=z(2, 3, dtype=I64)), "page_table must be"),
    (dict(page_table=z(3, 3, dtype=I32)), "page_table must be"),
    (dict(page_table=z(2, 6, dtype=I32)[:, ::2]), "rows of page_table"),
    (dict(seq_lens=z(2, dtype=I64)), "seq_lens must be"),
    (dict(parents=z(3, dtype=FF)), "parents must be"),
    (dict(parents=z(3, 1, dtype=I32)), "parents must be"),
    (dict(parents=z(6, dtype=I32)[::2]), "parents must be"),
    (dict(reserve=-1), "reserve"),
    (dict(k_cache=z(4, 2, 8, 32), v_cache=z(4, 2, 8, 32), k_scale_inv=None, v_scale_inv=None, key_ranges=z(4, 2, 2, 32).requires_grad_()),
     "no backward"),
])
def test_fork_refuses(over, match):
    refused(_ops().kv_cache_fork, fork_args(**over), match)


@pytest.mark.parametrize("over,match", [
    (dict(key_ranges=z(4, 2, 32)), "key_ranges must be"),
    (dict(key_ranges=z(5, 2, 2, 32)), "key_ranges must be"),
    (dict(k_scale_inv=None), "needs k_scale_inv"),
    (dict(cu_seqlens_q=z(2, dtype=I32)), "cu_seqlens_q must be"),
    (dict(page_table=z(2, 6, dtype=I32)[:, ::2]), "rows of page_table"),
])
def test_ranges_refuse(over, match):
    refused(_ops().kv_page_ranges, ranges_args(**over), match)


@pytest.mark.parametrize("over,match", [
    (dict(q=z(3, 3, 32)), "multiple of cache heads"),
    (dict(q=z(3, 4, 32, dtype=FF)), "bfloat16 or float16"),
    (dict(q=z(3, 4, 16)), "q must be"),
    (dict(key_ranges=z(4, 2, 3, 32)), "key_ranges must be"),
    (dict(num_selected=2), "must hold the first"),
    (dict(num_last=0), "num_last at least 1"),
    (dict(num_first=-1), "num_first"),
    (dict(seq_lens=z(2, dtype=I64)), "seq_lens must be"),
    (dict(page_table=z(0, 3, dtype=I32), seq_lens=z(0, dtype=I32), cu_seqlens_q=z(1, dtype=I32)), "without a sequence"),
    (dict(q=z(3, 4, 32).requires_grad_()), "no backward"),
])
@pytest.mark.parametrize("entry", ["select_pages", "sparse_paged_attention"])
def test_selection_refuses(entry, over, match):
    refused(getattr(_ops(), entry), (select_args if entry == "select_pages" else sparse_args)(**over), match)


def test_sparse_attention_refuses():
    o = _ops()
    for s in (0.0, -1.0, float("inf"), float("nan")):
        refused(o.sparse_paged_attention, sparse_args(softmax_scale=s), "softmax_scale")
    c = z(4, 2, 8, 32, dtype=FH)
    refused(o.sparse_paged_attention, sparse_args(k_cache=c, v_cache=c, k_scale_inv=None, v_scale_inv=None), "queries of its type")
    refused(o.select_pages, select_args(page_size=0), "page_size")
    refused(o.select_pages, select_args(q=z(3, 4, 24), key_ranges=z(4, 2, 2, 24)), "multiple of 16")


def test_without_a_gpu():
    if torch.cuda.is_available():
        pytest.skip("checks what happens without a GPU")
    for fn, args in _all():
        refused(fn, args, "need a ROCm GPU", RuntimeError)


def test_cpu_tensors_are_refused_beside_a_gpu(monkeypatch):
    from primus_turbo.pytorch import _C

    def launch(name, *args):
        raise RuntimeError(f"{name} was launched on host memory")

    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(_C, "stream", lambda device=None: 0)
    monkeypatch.setattr(_C, "call", launch)
    for fn, args in _all():
        refused(fn, args, "must be GPU tensors")


def test_fake_tensors_are_refused(monkeypatch):
    from torch._subclasses.fake_tensor import FakeTensorMode

    from primus_turbo.pytorch import _C

    done = []
    monkeypatch.setattr(_C, "stream", lambda device=None: 0)
    monkeypatch.setattr(_C, "call", lambda name, *args: done.append(name))
    for fn, args in _all():
        with FakeTensorMode() as mode:
            refused(fn, {n: mode.from_tensor(x) if isinstance(x, torch.Tensor) else x for n, x in args.items()}, "fake tensors")
    assert not done


def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fwad

    for fn, args in _all()[1:]:
        name = next(n for n in ("q", "v_scale_inv", "k_scale_inv") if n in args)
        with fwad.dual_level(), torch.no_grad():
            refused(fn, args | {name: fwad.make_dual(args[name], torch.ones_like(args[name]))}, "no forward-mode derivative")


def test_changed_tensors_count_as_changed(monkeypatch):
    from primus_turbo.pytorch import _C

    monkeypatch.setattr(_C, "stream", lambda device=None: 0)
    monkeypatch.setattr(_C, "call", lambda name, *args: None)
    monkeypatch.setattr(torch.cuda, "is_available", lambda: False)
    o = _ops()
    for fn, args, names in ((o.qk_norm_rope_cache_write, enter_args(), list(pools())), (o.kv_cache_copy, copy_args(), list(pools())),
                            (o.kv_cache_fork, fork_args(key_ranges=z(4, 2, 2, 32)), [*pools(), "key_ranges"]),
                            (o.kv_page_ranges, ranges_args(), ["key_ranges"])):
        before = [args[n]._version for n in names]
        fn(**args)
        assert all(args[n]._version > b for n, b in zip(names, before)), fn


def test_launches_go_to_the_tensors_device(monkeypatch):
    """The current device is the tensors' while a size is asked for and a kernel launched."""
    from primus_turbo.pytorch import _C

    class Device:
        current = 0

        def __init__(self, device):
            self.device, self.before = device, Device.current

        def __enter__(self):
            Device.current = self.device.index

        def __exit__(self, *_):
            Device.current = self.before

    seen = []
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(_C, "_cur_device", lambda: Device.current)
    monkeypatch.setattr(_C, "call", lambda name, *args: seen.append((name, Device.current)))
    monkeypatch.setattr(_C, "query", lambda name, *args: seen.append((name, Device.current)))
    for i in (1, 0):
        _C.call_on(torch.device("cuda", i), "launch")
        _C.query_on(torch.device("cuda", i), "size")
    assert seen == [("launch", 1), ("size", 1), ("launch", 0), ("size", 0)] and Device.current == 0


def test_c_entries_refuse():
    from primus_turbo.pytorch import _C

    p = ctypes.c_void_p(256)  # never dereferenced: the checks reject first

    def rope(dt=2, T=3, Hq=2, Hkv=1, D=32, rot=16, n=9, eps=1e-6, q=p, out=p, wdt=2):
        _C.call("pta_qk_norm_rope", q, p, dt, T, Hq, Hkv, D, 64, 32, 32, 32, p, p, n, rot, p, 1, p, wdt, p, 2, eps, 0, out, p, None)

    for kw, match in ((dict(dt=5), "unknown type"), (dict(D=31), "even"), (dict(D=300), "at most 256"), (dict(rot=34), "rotated"), (dict(rot=0), "rotated"),
                      (dict(T=1 << 31), "too many rows"), (dict(T=-1), "bad sizes"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
                      (dict(q=None), "null pointer"), (dict(out=ctypes.c_void_p(8)), "16-byte aligned"), (dict(wdt=9), "weight type")):
        with pytest.raises(RuntimeError, match=match):
            rope(**kw)

    def back(ws=p, n=1 << 30, qw=p, g=p):
        _C.call("pta_qk_norm_rope_backward", g, p, 64, 32, 32, 32, p, p, 2, 3, 2, 1, 32, 64, 32, 32, 32, p, p, 9, 16, p, 1, qw, 2, p, 2, 1e-6, 0,
                p, p, p, p, ws, n, None)

    for kw, match in ((dict(ws=None), "workspace too small"), (dict(n=16), "workspace too small"), (dict(qw=None), "without the weight"),
                      (dict(g=None), "null pointer")):
        with pytest.raises(RuntimeError, match=match):
            back(**kw)

    def enter(dt=2, D=32, kind=0, P=4, page=8, ks=p, slots=p, kc=p):
        _C.call("pta_qk_norm_rope_cache_write", p, p, p, dt, 3, 2, 1, D, 64, 32, 32, 32, 32, 32, p, p, 9, 16, p, 1, p, 2, p, 2, 1e-6, 0, slots, 1, kc, p,
                kind, P, page, ks, p, p, None)

    for kw, match in ((dict(dt=0), "bfloat16 or float16"), (dict(D=24), "multiple of 16"), (dict(kind=4), "unknown cache kind"),
                      (dict(P=1 << 40), "2\\^31 rows"), (dict(ks=None), "needs its scales"), (dict(slots=None), "null pointer"), (dict(kc=None), "null cache")):
        with pytest.raises(RuntimeError, match=match):
            enter(**kw)

    def copy(kind=0, L=1, P=4, D=32, ks=p, n=2, src=p, kc=p):
        _C.call("pta_kv_cache_copy", kc, p, kind, L, P, 2, 8, D, ks, p, None, src, p, 1, n, None)

    for kw, match in ((dict(kind=3), "unknown cache kind"), (dict(L=-1), "bad cache sizes"), (dict(D=8), "multiple of 16"), (dict(ks=None), "needs its scales"),
                      (dict(n=-1), "number of pages"), (dict(src=None), "null page list"), (dict(kc=ctypes.c_void_p(8)), "16-byte aligned"),
                      (dict(L=1 << 31), "too many layers")):
        with pytest.raises(RuntimeError, match=match):
            copy(**kw)

    def fork(M=3, B=2, N=2, reserve=0, ws=p, n=1 << 30, parents=p, lens=p):
        _C.call("pta_kv_cache_fork", p, p, 0, 1, 4, 2, 8, 32, p, p, None, p, 3, M, lens, B, parents, 1, N, reserve, 0, p, p, ws, n, None)

    for kw, match in ((dict(M=-1), "bad sizes"), (dict(reserve=-2), "bad sizes"), (dict(M=1 << 30), "too many entries"), (dict(N=1 << 25), "too many entries"),
                      (dict(N=3, parents=None), "without parents"), (dict(lens=None), "null pointer"), (dict(ws=None), "workspace too small"),
                      (dict(n=16), "workspace too small")):
        with pytest.raises(RuntimeError, match=match):
            fork(**kw)

    def ranges(kind=0, ks=p, D=32, out=p):
        _C.call("pta_kv_page_ranges", p, kind, 0, 4, 8, 2, D, ks, p, 3, 3, p, p, 2, out, None)

    for kw, match in ((dict(kind=9), "unknown cache kind"), (dict(ks=None), "needs its scales"), (dict(D=40), "multiple of 16"), (dict(out=None), "null pointer")):
        with pytest.raises(RuntimeError, match=match):
            ranges(**kw)

    def select(dt=2, T=3, take=4, first=1, last=2, ws=p, n=1 << 30, st=128):
        _C.call("pta_select_pages", p, dt, T, 4, 32, st, 32, p, 4, 8, 2, p, 3, 30, p, p, 2, take, first, last, p, p, ws, n, None)

    def sparse(dt=2, T=3, take=4, first=1, last=2, ws=p, n=1 << 30, st=128, scale=0.1):
        _C.call("pta_sparse_paged_attention", p, dt, T, 4, 32, st, 32, p, p, 0, 4, 8, 2, p, p, p, p, 3, 30, p, p, 2, take, first, last, scale, p, None,
                ws, n, None)

    for kw, match in ((dict(dt=0), "bfloat16 or float16"), (dict(T=-1), "bad sizes"), (dict(take=2), "must hold"), (dict(last=0), "must hold"),
                      (dict(first=-1), "must hold"), (dict(ws=None), "workspace too small"), (dict(n=8), "workspace too small"), (dict(st=129), "multiples of 8")):
        for f in (select, sparse):
            with pytest.raises(RuntimeError, match=match):
                f(**kw)
    with pytest.raises(RuntimeError, match="softmax_scale"):
        sparse(scale=-1.0)


def test_workspaces_stay_small():
    from primus_turbo.pytorch import _C

    # scores of a slice of tokens at most
    assert _C.query("pta_select_pages_workspace_size", 100000, 8, 4096) <= 256 << 20
    assert _C.query("pta_select_pages_workspace_size", 1, 64, 1 << 20) == 64 * 8 << 20  # one token's
    assert _C.query("pta_select_pages_workspace_size", 0, 8, 64) == 0
    # lists of a tile's tokens: 10 bytes for each page that a token takes, 12 a token; parts of tiles
    # that do not fill the chip
    q = lambda *a: _C.query("pta_sparse_paged_attention_workspace_size", *a)  # noqa: E731
    assert q(8192, 1, 32, 8, 128, 256, 64, 16) <= 8192 * 8 * 16 * 10 + 12 * 8192 + (256 << 20) + 4096
    assert q(64, 64, 32, 4, 64, 512, 32, 48) <= 64 * 4 * 48 * 4 + 12 * 64 + max(64 * 4 * 512 * 8, 8 * 64 * 32 * (4 * 64 + 8)) + 4096
    assert q(0, 1, 32, 8, 128, 256, 64, 16) == 0
    # a row for each workgroup that sums
    assert _C.query("pta_qk_norm_rope_backward_workspace_size", 1 << 20, 32, 8, 128) <= (8 * 256 + 2) * 128 * 4
    assert _C.query("pta_qk_norm_rope_backward_workspace_size", 0, 32, 8, 128) == 0


def test_lists_of_tiles_hold_no_page_twice():
    """A list of a tile's pages is no longer than its sequences' rows of the table: sixteen tokens of one
    sequence that take all of its pages have them once (10 bytes each), not sixteen times."""
    from primus_turbo.pytorch import _C

    q = lambda *a: _C.query("pta_sparse_paged_attention_workspace_size", *a)  # noqa: E731
    T, H, M = 8192, 8, 2048  # a query head to each cache head: sixteen tokens a tile
    rest = (256 << 20) + 12 * T + 4 * (T // 16 * H) + 4096  # the scores, the tokens' lengths and positions, the lists' lengths
    assert q(T, 1, H, H, 128, M, 16, M) <= T // 16 * H * M * 10 + rest
    assert q(T, 3, H, H, 128, M, 16, M) <= T // 16 * H * 3 * M * 10 + rest
    # many sequences, or few pages a token: as many as the tokens take
    assert q(T, 4096, H, H, 128, M, 16, 16) <= T // 16 * H * 16 * 16 * 10 + rest


def test_books_by_hand():
    """The oracle's own check: what the documentation says, on cases small enough to follow."""
    # two answers to one prompt of 6 tokens in pages of 4: the full page is shared, the second answer's last page is a copy
    assert fork_books([[7, 2, -1]], [6], [0, 0], 4, 10, 0, False) == ([[7, 2, -1], [7, 0, -1]], [6, 6], [(2, 0)])
    # the same with room for three more tokens each: a page more
    assert fork_books([[7, 2, -1]], [6], [0, 0], 4, 10, 3, False) == ([[7, 2, 0], [7, 1, 3]], [6, 6], [(2, 1)])
    # compacted: pages 7 and 2 and a copy are pages 0 to 2
    assert fork_books([[7, 2, -1]], [6], [0, 0], 4, 10, 0, True) == ([[0, 2, -1], [0, 1, -1]], [6, 6], [(7, 0), (2, 1)])
    # a page that one sequence fills is not another one's to write into
    assert fork_books([[5, 6], [5, -1]], [8, 3], [0, 1], 4, 8, 0, False) == ([[5, 6], [0, -1]], [8, 3], [(5, 0)])
    # too few pages: the first in order get theirs
    assert fork_books([[0, -1], [1, -1]], [2, 2], [0, 0, 1, 1], 4, 3, 0, False) == ([[0, -1], [2, -1], [1, -1], [-1, -1]], [2, 2, 2, -1], [(0, 2)])
    # and one that had none gets none, whatever it is to reserve
    assert fork_books([[0, -1], [-1, -1]], [2, -1], [1, 0, 1], 4, 3, 9, False) == ([[-1, -1], [0, 1], [-1, -1]], [-1, 2, -1], [])
