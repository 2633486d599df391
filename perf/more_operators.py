"""The operators around a paged key / value cache, as cases that can be timed: how
queries, keys and values get ready for it, how sequences share and part its pages,
and how a long context is attended through few of them.

A case is a dict of plain values; ``op`` says which entry points it stands for:

  rope    ops.qk_norm_rope: norms of queries and keys for each head with the
          position rotation, forward and backward, as a training step makes them
  enter   ops.qk_norm_rope_cache_write: the same for new tokens that are served,
          whose keys and values go straight into their cache slots
  copy    ops.kv_cache_copy: pages copied inside the cache, all layers at once
  fork    ops.kv_cache_fork: sequences that go on from others, share their full
          pages and get copies of the partly filled one; with ``compact`` the
          pages in use move to the front of the pool
  sparse  ops.kv_page_ranges and ops.sparse_paged_attention: the ranges of the
          new tokens' keys, then attention over the pages that they select

The plain forms are elementary torch operations in 32 bits; sums over all tokens
and the scores that pages are chosen by are in 64.
"""

import math
import os
import random
import sys

import torch

#: set by whoever measures: whether run() calls the framework's operators
own = False

DEV = "cuda"
EPS = 1e-6
_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4, "e4m3": 1, "e5m2": 1}
_FP8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
_FP8_MAX = {"e4m3": 448.0, "e5m2": 57344.0}


def _ops():
    pkg = os.path.join(os.getcwd(), "primus-turbo_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import primus_turbo.pytorch as turbo

    return turbo.ops


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def _rope(name, B, S, Hq, Hkv, D, rot, dtype="bf16", interleaved=False, norm=True):
    return {"name": name, "op": "rope", "B": B, "S": S, "Hq": Hq, "Hkv": Hkv, "D": D, "rot": rot, "dtype": dtype,
            "interleaved": interleaved, "norm": norm}


def _enter(name, T, Hq, Hkv, D, rot, page, cache="e4m3", dtype="bf16", interleaved=False, norm=True, skip=0):
    return {"name": name, "op": "enter", "T": T, "Hq": Hq, "Hkv": Hkv, "D": D, "rot": rot, "page": page, "cache": cache,
            "dtype": dtype, "interleaved": interleaved, "norm": norm, "skip": skip}


def _copy(name, layers, pages, pairs, Hkv, D, page, cache="e4m3"):
    return {"name": name, "op": "copy", "layers": layers, "pages": pages, "pairs": pairs, "Hkv": Hkv, "D": D, "page": page,
            "cache": cache}


def _fork(name, layers, B, N, ctx, Hkv, D, page, cache="e4m3", compact=False, reserve=1, ranges=False):
    return {"name": name, "op": "fork", "layers": layers, "B": B, "N": N, "ctx": ctx, "Hkv": Hkv, "D": D, "page": page,
            "cache": cache, "compact": compact, "reserve": reserve, "ranges": ranges}


def _sparse(name, B, chunk, ctx, Hq, Hkv, D, page, take, cache="e4m3", dtype="bf16", ragged=True, first=1, last=2):
    return {"name": name, "op": "sparse", "B": B, "chunk": chunk, "ctx": ctx, "Hq": Hq, "Hkv": Hkv, "D": D, "page": page,
            "take": take, "cache": cache, "dtype": dtype, "ragged": ragged, "first": first, "last": last}


def listed():
    return [
        # a training step's attention inputs, four sequences of 2048, grouped heads
        _rope("rope_4x2048_32+8x128", 4, 2048, 32, 8, 128, 128),
        # a head size that is no power of two, of which a part is rotated, neighbours as pairs, odd lengths
        _rope("rope_3x333_12+12x80_rot32_fp16", 3, 333, 12, 12, 80, 32, dtype="fp16", interleaved=True),
        # a small model in 32 bits, one head of keys, rotation alone
        _rope("rope_1x257_8+1x64_fp32", 1, 257, 8, 1, 64, 64, dtype="fp32", norm=False),
        # one sequence answers token by token: latency counts
        _enter("enter_1_32+8x128", 1, 32, 8, 128, 128, 64),
        # the prompt tokens of one step, some of them padding that has no slot
        _enter("enter_8192_32+8x128", 8192, 32, 8, 128, 128, 64, skip=100),
        # one sequence's last page to each of a few others, one layer
        _copy("copy_1x8_of_64", 1, 64, 8, 8, 128, 64),
        # pages moved for a host that keeps its own books, all layers of a small model, 16-bit cache, small pages
        _copy("copy_16x1000_of_4096_bf16", 16, 4096, 1000, 4, 64, 16, cache="bf16"),
        # a step of beam search: 16 prompts of four beams each, every layer's last pages
        _fork("fork_8x64_of_4096", 8, 64, 64, 4096, 8, 128, 64, ranges=True),
        # half of 64 sequences have ended; what the others hold moves to the front
        _fork("compact_2x32_of_64x4096", 2, 64, 32, 4096, 8, 128, 64, compact=True, reserve=0),
        # one long sequence answers token by token through 64 of its 2048 pages
        _sparse("sparse_1x131072_32h8_d128", 1, 1, 131072, 32, 8, 128, 64, 64, ragged=False),
        # a decoding batch over contexts of all lengths, pages of 32 tokens, 16-bit cache
        _sparse("sparse_64x16384_32h4_d64_fp16", 64, 1, 16384, 32, 4, 64, 32, 48, cache="fp16", dtype="fp16"),
        # a chunk of a long prompt, every token with pages of its own
        _sparse("sparse_1024_of_16384_32h8_d128", 1, 1024, 16384, 32, 8, 128, 64, 16, ragged=False),
    ]


def _log(rng, lo, hi, mult=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(mult, int(v / mult + 0.5) * mult)


def _nameless(case):
    return {n: v for n, v in case.items() if n != "name"}


_ROPE = 4 * 2048 * 40 * 128 * 2       # bytes of the largest listed queries and keys
_PAIRS = 1024 * 32 * 16 * 64 * 128    # products of the largest listed chunk's logits
_POOL = 64 * 4096 * 8 * 128           # bytes of a layer's keys in the largest listed pool


def draw(rng):
    op = rng.choice(("rope", "enter", "copy", "fork", "sparse", "sparse"))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    cache = rng.choice(("e4m3", "e4m3", "e5m2", dtype))
    Hkv, D, page = rng.choice((1, 2, 4, 8)), rng.choice((64, 80, 96, 128, 128, 256)), rng.choice((16, 32, 64, 48, 128))
    Hq = Hkv * rng.choice((1, 2, 4, 8))
    rot = rng.choice((D, D, D // 2, 32))
    two, norm = rng.random() < 0.3, rng.random() < 0.7
    if op == "rope":
        dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
        most = _ROPE // ((Hq + Hkv) * D * _SIZE[dtype])
        T = _log(rng, 16, most)
        B = min(T, rng.randint(1, 8))
        return _nameless(_rope("", B, T // B, Hq, Hkv, D, rot, dtype, two, norm))
    if op == "enter":
        T = _log(rng, 1, min(8192, _ROPE // ((Hq + Hkv) * D * 2)))
        return _nameless(_enter("", T, Hq, Hkv, D, rot, page, cache, dtype, two, norm, rng.choice((0, 0, min(3, T - 1)))))
    if op == "copy":
        layers = rng.randint(1, 16)
        most = 1000 * 16 * 4 * 64 * 16 * 2 // (layers * Hkv * D * page * _SIZE[cache])
        pairs = _log(rng, 1, max(2, min(1000, most)))
        return _nameless(_copy("", layers, 2 * pairs + rng.randint(1, 40), pairs, Hkv, D, page, cache))
    if op == "fork":
        while True:
            B, ctx, layers = _log(rng, 1, 64), _log(rng, 16, 8192), rng.randint(1, 8)
            compact = rng.random() < 0.4
            if B * ctx * Hkv * D * _SIZE[cache] * layers <= 2 * _POOL:
                return _nameless(_fork("", layers, B, _log(rng, 1, 64), ctx, Hkv, D, page, cache, compact,
                                       rng.choice((0, 1, 1, 7)), rng.random() < 0.5))
    while True:
        B = _log(rng, 1, 64)
        chunk = 1 if rng.random() < 0.5 else _log(rng, 2, 1024)
        ctx = _log(rng, max(16, chunk), 65536)
        last = rng.choice((1, 2, 4))
        c = _sparse("", B, chunk, ctx, Hq, Hkv, D, page, rng.randint(last + 2, 64), cache, dtype, rng.random() < 0.7,
                    rng.choice((0, 1, 2)), last)
        if (B * chunk * Hq * c["take"] * page * max(D, 128) <= _PAIRS and B * ctx * Hkv * D * _SIZE[cache] <= _POOL
                and B * chunk * Hkv * (ctx // page + 1) * D <= 1024 * 8 * 257 * 128):
            return _nameless(c)


# ---------------------------------------------------------------------------
# what belongs to the case itself, so that its work is known
# ---------------------------------------------------------------------------
def _lengths(case):
    """(new tokens, length with them) of every sequence."""
    B, chunk, ctx = case["B"], case["chunk"], case["ctx"]
    if not case["ragged"]:
        return [chunk] * B, [ctx] * B
    r = random.Random(B * 100003 + ctx)
    new = [max(1, round(chunk ** r.random())) for _ in range(B)]
    new[0] = chunk
    lens = [max(n, int(ctx * (0.1 + 0.9 * r.random()))) for n in new]
    lens[0] = ctx
    return new, lens


def _family(case):
    """(lengths, parents) of a fork: four beams go on from each prompt's best ones, or, where
    pages are compacted, some sequences go on and the others have ended."""
    B, N = case["B"], case["N"]
    r = random.Random(B * 7919 + N)
    lens = [max(1, int(case["ctx"] * (0.1 + 0.9 * r.random()))) for _ in range(B)]
    if case["compact"]:
        return lens, sorted(r.sample(range(B), min(B, N)))
    for b in range(B):
        lens[b] = lens[b // 4 * 4]
    return lens, [min(B - 1, i // 4 * 4 % B + r.randint(0, 3)) for i in range(N)]


def _layer_page(case):
    """Bytes of one page of one layer: keys and values, their scales and ranges."""
    e = _SIZE[case["cache"]]
    row = 2 * (case["D"] * e + (4 if e == 1 else 0))
    return case["Hkv"] * (case["page"] * row + (4 * case["D"] if case.get("ranges") else 0))


def _fork_pages(case):
    """Pages of a fork's pool."""
    lens, _ = _family(case)
    page = case["page"]
    return sum(-(-n // page) + 1 for n in lens) + case["N"] * (1 + -(-case["reserve"] // page)) + 3


def work(case):
    op = case["op"]
    if op == "rope":
        n = case["B"] * case["S"] * (case["Hq"] + case["Hkv"]) * case["D"]
        table = 4 * case["S"] * case["rot"]
        return {"bytes": 5.0 * n * _SIZE[case["dtype"]] + table, "flops": 30.0 * n}
    if op == "enter":
        T, Hq, Hkv, D = case["T"], case["Hq"], case["Hkv"], case["D"]
        rows, e = 2 * (T - case["skip"]) * Hkv, _SIZE[case["cache"]]
        return {"bytes": 4.0 * T * Hq * D + rows * (2 * D + D * e + (4 if e == 1 else 0)) + T * (4 * case["rot"] + 16),
                "flops": 12.0 * T * (Hq + Hkv) * D}
    if op == "copy":
        return {"bytes": 2.0 * case["layers"] * case["pairs"] * _layer_page(case) + 16 * case["pairs"], "flops": 0.0}
    if op == "fork":
        lens, parents = _family(case)
        page = case["page"]
        part = [p for p in parents if lens[p] % page]
        moved = float(len(part) - len(set(part)))
        if case["compact"]:
            # pages in use lie anywhere in the pool
            kept, P = sum(-(-lens[p] // page) for p in set(parents)), _fork_pages(case)
            moved += kept * (1.0 - kept / P)
        tables = 4 * (sum(-(-lens[p] // page) for p in parents) + len(parents))
        return {"bytes": 2.0 * case["layers"] * moved * _layer_page(case) + 2 * tables, "flops": 0.0}
    new, lens = _lengths(case)
    page, D, Hq, Hkv, take = case["page"], case["D"], case["Hq"], case["Hkv"], case["take"]
    row = 2 * (D + 4) if case["cache"] in _FP8 else 4 * D
    ranges = keys = pairs = scored = 0
    for n, L in zip(new, lens):
        pages = -(-L // page)
        ranges += pages
        scored += n * pages
        seen = [min(p + 1, (take - 1) * page + p % page + 1) for p in range(L - n, L)]
        pairs += sum(seen)
        # one token's pages at least; a chunk's tokens need not choose different ones
        keys += seen[-1]
    q = sum(new) * Hq * D
    return {"bytes": 4.0 * Hkv * D * ranges + Hkv * row * keys + 4.0 * q,
            "flops": 4.0 * Hq * D * pairs + 4.0 * Hkv * D * scored}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _randn(shape, g):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32)


def _rows_to_fp8(x, fmt):
    """One scale for each row of the last axis: (fp8, inverse scales)."""
    s = _FP8_MAX[fmt] / x.abs().amax(dim=-1).clamp(min=1e-12)
    return (x * s.unsqueeze(-1)).clamp(-_FP8_MAX[fmt], _FP8_MAX[fmt]).to(_FP8[fmt]), 1.0 / s


def _pool(pages, case, g, layers=0):
    """Cache pages with content: channels of different strength, as keys and values have them."""
    Hkv, page, D = case["Hkv"], case["page"], case["D"]
    strength = torch.exp(0.5 * _randn((1, Hkv, 1, D), g))
    n_all = pages * max(layers, 1)
    x = torch.empty((n_all, Hkv, page, D), dtype=_FP8.get(case["cache"]) or _DT[case["cache"]], device=DEV)
    s = torch.empty((n_all, Hkv, page), dtype=torch.float32, device=DEV) if case["cache"] in _FP8 else None
    step = max(1, (1 << 27) // (Hkv * page * D))
    for p in range(0, n_all, step):
        n = min(step, n_all - p)
        v = _randn((n, Hkv, page, D), g) * strength
        if s is None:
            x[p:p + n] = v.to(x.dtype)
        else:
            x[p:p + n], s[p:p + n] = _rows_to_fp8(v, case["cache"])
    if layers:
        x = x.view(layers, pages, Hkv, page, D)
        s = s if s is None else s.view(layers, pages, Hkv, page)
    return x, s


def _rotation(positions, rot):
    """cos and sin of a rotation's angles, [positions, rot / 2]."""
    f = 10000.0 ** (-torch.arange(rot // 2, device=DEV, dtype=torch.float64) * 2 / rot)
    a = torch.arange(positions, device=DEV, dtype=torch.float64)[:, None] * f
    return a.cos().float(), a.sin().float()


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    st = {"case": case}
    return {"rope": _prepare_rope, "enter": _prepare_enter, "copy": _prepare_copy, "fork": _prepare_fork,
            "sparse": _prepare_sparse}[case["op"]](case, st, g)


def _weights(case, st, g, dt):
    for n in ("wq", "wk"):
        st[n] = (1.0 + 0.2 * _randn((case["D"],), g)).to(dt) if case["norm"] else None


def _prepare_rope(case, st, g):
    B, S, Hq, Hkv, D, dt = (case[n] for n in ("B", "S", "Hq", "Hkv", "D", "dtype"))
    dt = _DT[dt]
    # parts of a projection's output, as a model has them
    qkv = torch.empty((B, S, Hq + 2 * Hkv, D), dtype=dt, device=DEV).copy_(_randn((B, S, Hq + 2 * Hkv, D), g))
    st["q"], st["k"] = qkv[:, :, :Hq].detach().requires_grad_(), qkv[:, :, Hq:Hq + Hkv].detach().requires_grad_()
    _weights(case, st, g, dt)
    for n in ("wq", "wk"):
        if st[n] is not None:
            st[n].requires_grad_()
    st["cos"], st["sin"] = _rotation(S + 7, case["rot"])
    st["pos"] = torch.arange(S, device=DEV).expand(B, S).contiguous()
    st["gq"], st["gk"] = _randn((B, S, Hq, D), g).to(dt), _randn((B, S, Hkv, D), g).to(dt)
    return st


def _prepare_enter(case, st, g):
    T, Hq, Hkv, D, page, dt = (case[n] for n in ("T", "Hq", "Hkv", "D", "page", "dtype"))
    dt = _DT[dt]
    pages = -(-T // page) + 3
    for n in ("k", "v"):
        st[n + "_cache"], st[n + "_scale"] = _pool(pages, case, g)
    at = torch.randperm(pages, generator=g, device=DEV)
    i = torch.arange(T, device=DEV)
    st["slots"] = at[i // page] * page + i % page
    if case["skip"]:
        st["slots"][torch.randperm(T, generator=g, device=DEV)[:case["skip"]]] = -1
    qkv = torch.empty((T, Hq + 2 * Hkv, D), dtype=dt, device=DEV).copy_(_randn((T, Hq + 2 * Hkv, D), g))
    st["q"], st["k"], st["v"] = qkv.split([Hq, Hkv, Hkv], dim=1)
    _weights(case, st, g, dt)
    st["cos"], st["sin"] = _rotation(32768, case["rot"])
    # tokens of prompts that began before
    st["pos"] = (i + torch.randint(0, 32768 - T, (1,), generator=g, device=DEV)).to(torch.int32)
    return st


def _pools(case, st, g, pages):
    for n in ("k", "v"):
        st[n + "_cache"], st[n + "_scale"] = _pool(pages, case, g, case["layers"])
    st["ranges"] = None
    if case.get("ranges"):
        st["ranges"] = _randn((case["layers"], pages, case["Hkv"], 2, case["D"]), g).to(torch.bfloat16)


def _prepare_copy(case, st, g):
    _pools(case, st, g, case["pages"])
    order = torch.randperm(case["pages"], generator=g, device=DEV).to(torch.int32)
    n = case["pairs"]
    st["src"], st["dst"] = order[:n].contiguous(), order[n:2 * n].contiguous()
    return st


def _prepare_fork(case, st, g):
    lens, parents = _family(case)
    page = case["page"]
    most = -(-(max(lens) + case["reserve"]) // page) + 1
    pages = _fork_pages(case)
    _pools(case, st, g, pages)
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((case["B"], most), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(lens):
        full, need = n // page, -(-n // page)
        # beams share their prompt's first half
        shared = 0 if case["compact"] or b % 4 == 0 else full // 2
        if shared:
            table[b, :shared] = table[b // 4 * 4, :shared]
        table[b, shared:need] = order[at:at + need - shared]
        at += need - shared
    st["table"], st["lens"] = table, torch.tensor(lens, dtype=torch.int32, device=DEV)
    st["parents"] = torch.tensor(parents, dtype=torch.int32, device=DEV)
    return st


def _prepare_sparse(case, st, g):
    B, Hq, D, page = case["B"], case["Hq"], case["D"], case["page"]
    new, lens = _lengths(case)
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 1
    for n in ("k", "v"):
        st[n + "_cache"], st[n + "_scale"] = _pool(pages, case, g)
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((B, max(need)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    st["table"], st["lens"] = table, torch.tensor(lens, dtype=torch.int32, device=DEV)
    st["cu"] = torch.tensor([sum(new[:b]) for b in range(B + 1)], dtype=torch.int32, device=DEV)
    st["q"] = _randn((sum(new), Hq, D), g).to(_DT[case["dtype"]])
    # the pages of earlier tokens have their ranges, the new tokens' pages are yet to get them
    st["ranges"] = torch.zeros((pages, case["Hkv"], 2, D), dtype=torch.bfloat16, device=DEV)
    step = max(1, (1 << 26) // (case["Hkv"] * page * D))
    for p in range(0, pages, step):
        x = st["k_cache"][p:p + step].float()
        if st["k_scale"] is not None:
            x = x * st["k_scale"][p:p + step, ..., None]
        st["ranges"][p:p + step] = _range_of(x)
    for b in range(B):
        st["ranges"][table[b, (lens[b] - new[b]) // page:need[b]].long()] = 0
    st["new_list"], st["lens_list"] = new, lens
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(st):
    case, op = st["case"], st["case"]["op"]
    if not own:
        return {"rope": _plain_rope, "enter": _plain_enter, "copy": _plain_copy, "fork": _plain_fork,
                "sparse": _plain_sparse}[op](st)
    ops = _ops()
    if op == "rope":
        q, k = ops.qk_norm_rope(st["q"], st["k"], st["cos"], st["sin"], st["pos"], st["wq"], st["wk"], eps=EPS,
                                interleaved=case["interleaved"])
        to = (st["q"], st["k"], st["wq"], st["wk"]) if case["norm"] else (st["q"], st["k"])
        return (q.detach(), k.detach()) + torch.autograd.grad((q, k), to, (st["gq"], st["gk"]))
    if op == "enter":
        q = ops.qk_norm_rope_cache_write(st["q"], st["k"], st["v"], st["cos"], st["sin"], st["pos"], st["k_cache"],
                                         st["v_cache"], st["slots"], st["k_scale"], st["v_scale"], q_weight=st["wq"],
                                         k_weight=st["wk"], eps=EPS, interleaved=case["interleaved"])
        return {"q": q} | _held(st)
    if op == "copy":
        ops.kv_cache_copy(st["k_cache"], st["v_cache"], st["src"], st["dst"], st["k_scale"], st["v_scale"])
        return _held(st)
    if op == "fork":
        table, lens = ops.kv_cache_fork(st["k_cache"], st["v_cache"], st["table"], st["lens"], st["parents"], st["k_scale"],
                                        st["v_scale"], key_ranges=st["ranges"], reserve=case["reserve"],
                                        compact=case["compact"])
        return {"table": table, "lens": lens} | _held(st)
    ops.kv_page_ranges(st["k_cache"], st["table"], st["cu"], st["lens"], st["ranges"], st["k_scale"])
    out = ops.sparse_paged_attention(st["q"], st["k_cache"], st["v_cache"], st["ranges"], st["table"], st["cu"], st["lens"],
                                     st["k_scale"], st["v_scale"], num_selected=case["take"], num_first=case["first"],
                                     num_last=case["last"])
    return {"out": out, "ranges": st["ranges"]}


def _held(st):
    """What the cache holds."""
    out = {"k": st["k_cache"], "v": st["v_cache"]}
    if st["k_scale"] is not None:
        out |= {"k_scale": st["k_scale"], "v_scale": st["v_scale"]}
    if st.get("ranges") is not None:
        out["ranges"] = st["ranges"]
    return out


def _turn(x, c, s, interleaved):
    """The pairs of the first elements of x turned by (c, s)."""
    rot = 2 * c.shape[-1]
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack((a * c - b * s, a * s + b * c), dim=-1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat((a * c - b * s, a * s + b * c), dim=-1)
    return torch.cat((y, x[..., rot:]), dim=-1)


def _plain_one(x, w, c, s, interleaved):
    x = x.float()
    if w is not None:
        x = x * (x.square().mean(dim=-1, keepdim=True) + EPS).rsqrt() * w.float()
    return _turn(x, c, s, interleaved)


def _plain_back(x, w, c, s, interleaved, g):
    """(gradient of x, gradient of w)."""
    g, y = _turn(g.float(), c, -s, interleaved), x.float()
    if w is None:
        return g.to(x.dtype), None
    r = (y.square().mean(dim=-1, keepdim=True) + EPS).rsqrt()
    y = y * r
    dw = (g * y).flatten(0, -2).sum(dim=0, dtype=torch.float64)
    g = g * w.float()
    return (r * (g - y * (g * y).mean(dim=-1, keepdim=True))).to(x.dtype), dw.to(w.dtype)


def _plain_rope(st):
    two = st["case"]["interleaved"]
    c, s = st["cos"][st["pos"]].unsqueeze(-2), st["sin"][st["pos"]].unsqueeze(-2)
    out, dx, dw = [], [], []
    with torch.no_grad():
        for n in ("q", "k"):
            out.append(_plain_one(st[n], st["w" + n], c, s, two).to(st[n].dtype))
            a, b = _plain_back(st[n], st["w" + n], c, s, two, st["g" + n])
            dx.append(a)
            dw.append(b)
    return tuple(out + dx + [x for x in dw if x is not None])


def _plain_put(x, cache, scale, slots, fmt):
    page = cache.shape[2]
    if scale is None:
        cache[slots // page, :, slots % page] = x.to(cache.dtype)
        return
    q, inv = _rows_to_fp8(x.float(), fmt)
    # torch moves fp8 values through index_put as bytes
    cache.view(torch.uint8)[slots // page, :, slots % page] = q.view(torch.uint8)
    scale[slots // page, :, slots % page] = inv


def _plain_enter(st):
    case, slots = st["case"], st["slots"]
    c, s = st["cos"][st["pos"].long()].unsqueeze(1), st["sin"][st["pos"].long()].unsqueeze(1)
    q = _plain_one(st["q"], st["wq"], c, s, case["interleaved"]).to(st["q"].dtype)
    k, v = _plain_one(st["k"], st["wk"], c, s, case["interleaved"]), st["v"]
    if case["skip"]:
        has = slots >= 0
        slots, k, v = slots[has], k[has], v[has]
    _plain_put(k, st["k_cache"], st["k_scale"], slots, case["cache"])
    _plain_put(v, st["v_cache"], st["v_scale"], slots, case["cache"])
    return {"q": q} | _held(st)


def _plain_move(st, src, dst):
    for n in ("k_cache", "v_cache", "k_scale", "v_scale", "ranges"):
        x = st.get(n)
        if x is not None:
            x = x.view(torch.uint8) if x.element_size() == 1 else x
            x[:, dst] = x[:, src]


def _plain_copy(st):
    _plain_move(st, st["src"].long(), st["dst"].long())
    return _held(st)


def _plain_fork(st):
    case, table, parents = st["case"], st["table"].long(), st["parents"].long()
    page, M, P, N = case["page"], table.shape[1], st["k_cache"].shape[1], parents.shape[0]
    lens = st["lens"][parents]
    rows, j, i = table[parents], torch.arange(M, device=DEV), torch.arange(N, device=DEV)
    full, part = (lens // page).long(), lens % page > 0
    has = full + part.long()
    held, last = j < has[:, None], (full.clamp(max=M - 1)[:, None] == j) & part[:, None]
    # who has a page: everybody (full), or the first sequence that it is the last page of
    owner = torch.full((P + 1,), N, dtype=torch.int64, device=DEV)
    at = torch.where(held & last, rows, P)
    owner.scatter_reduce_(0, at.flatten(), i[:, None].expand(N, M).flatten(), "amin")
    owner[torch.where(held & ~last, rows, P).flatten()] = -1
    mine = owner[rows] == i[:, None]
    fresh = (last & ~mine) | (~held & (j < (-(-(lens.long() + case["reserve"]) // page)).clamp(max=M)[:, None]))
    used = owner[:P] < N
    count = used.sum()
    take = fresh.sum()
    number = fresh.flatten().cumsum(0).view(N, M) - 1
    # free pages in order, and the same list for the pages that move
    page_id = torch.arange(P, device=DEV)
    bound = (count + take).clamp(max=P) if case["compact"] else torch.full_like(count, P)
    free = torch.argsort(used.to(torch.int8), stable=True)
    moves = used & (page_id >= bound)
    n_moves = moves.sum()
    to = torch.where(moves, free[(moves.cumsum(0) - 1).clamp(min=0)], page_id)
    free_id = free[(number + n_moves).clamp(0, P - 1)]
    out = torch.where(fresh, free_id, torch.where(held, to[rows.clamp(min=0)], -1))
    copied = last & ~mine
    src, dst = torch.cat((page_id[moves], rows[copied])), torch.cat((to[moves], free_id[copied]))
    _plain_move(st, src, dst)
    return {"table": out.to(torch.int32), "lens": lens} | _held(st)


def _range_of(x):
    """Smallest and largest of the keys [..., page, D], rounded outward to bf16: [..., 2, D]."""
    lo, hi = x.amin(dim=-2), x.amax(dim=-2)
    out = torch.stack((lo, hi), dim=-2)
    b = out.view(torch.int32)
    away = torch.stack((lo < 0, hi > 0), dim=-2) & ((b & 0xffff) != 0)
    return ((b >> 16) + away).to(torch.int16).view(torch.bfloat16)


def _plain_keys(cache, scale, ids):
    """Pages [..., Hkv, page, D] in 32 bits."""
    x = cache.view(torch.uint8)[ids].view(cache.dtype).float() if cache.element_size() == 1 else cache[ids].float()
    return x if scale is None else x * scale[ids].unsqueeze(-1)


def _plain_sparse(st):
    case, q, table = st["case"], st["q"], st["table"].long()
    Hq, Hkv, D, page, take = (case[n] for n in ("Hq", "Hkv", "D", "page", "take"))
    group = Hq // Hkv
    out = torch.empty_like(q)
    heads = torch.arange(Hkv, device=DEV)
    at = 0
    for b, (n, L) in enumerate(zip(st["new_list"], st["lens_list"])):
        pages = -(-L // page)
        ids = table[b, :pages]
        p0 = (L - n) // page
        x = _plain_keys(st["k_cache"], st["k_scale"], ids[p0:])
        there = torch.arange(p0 * page, pages * page, device=DEV).view(pages - p0, 1, page, 1) < L
        low = _range_of(torch.where(there, x, math.inf))[..., 0, :]
        high = _range_of(torch.where(there, x, -math.inf))[..., 1, :]
        st["ranges"][ids[p0:]] = torch.stack((low, high), dim=-2)
        r = st["ranges"][ids].double().permute(1, 2, 3, 0).contiguous()  # [Hkv, 2, D, pages]
        step = max(1, (1 << 30) // (4 * Hkv * min(take, pages) * page * (D + 2 * group)))
        for i in range(0, n, step):
            m = min(step, n - i)
            x = q[at + i:at + i + m].view(m, Hkv, group, D)
            up, down = x.double().clamp(min=0).sum(dim=2), x.double().clamp(max=0).sum(dim=2)
            score = torch.matmul(up.transpose(0, 1).contiguous(), r[:, 1]) + torch.matmul(down.transpose(0, 1).contiguous(), r[:, 0])
            pos = torch.arange(L - n + i, L - n + i + m, device=DEV)
            mine = (pos // page)[:, None]
            j = torch.arange(pages, device=DEV)
            score = score.transpose(0, 1)  # [m, Hkv, pages]
            score = score.masked_fill(((j < case["first"]) | (j > mine - case["last"]))[:, None], math.inf)
            score = score.masked_fill((j > mine)[:, None], -math.inf)
            best = torch.sort(score, dim=-1, descending=True, stable=True)[1][..., :take]
            best = torch.sort(best, dim=-1)[0]  # [m, Hkv, taken]
            key = best[..., None] * page + torch.arange(page, device=DEV)
            seen = (key <= pos[:, None, None, None]).flatten(2)
            sel = ids[best]
            k, v = (_plain_pick(st[c + "_cache"], st[c + "_scale"], sel, heads).flatten(2, 3) for c in ("k", "v"))
            s = torch.matmul(x.float(), k.transpose(2, 3).contiguous()) * D ** -0.5
            s = s.masked_fill(~seen[:, :, None], -math.inf)
            s = torch.exp(s - s.amax(dim=-1, keepdim=True))
            out[at + i:at + i + m] = (torch.matmul(s, v) / s.sum(dim=-1, keepdim=True)).view(m, Hq, D).to(q.dtype)
        at += n
    return {"out": out, "ranges": st["ranges"]}


def _plain_pick(cache, scale, sel, heads):
    """Every head's own pages: sel [m, Hkv, taken] -> [m, Hkv, taken, page, D] in 32 bits."""
    h = heads[None, :, None]
    x = cache.view(torch.uint8)[sel, h].view(cache.dtype).float() if cache.element_size() == 1 else cache[sel, h].float()
    return x if scale is None else x * scale[sel, h].unsqueeze(-1)


# ---------------------------------------------------------------------------
# what a correct answer is, in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        return {"rope": _exact_rope, "enter": _exact_enter, "copy": _exact_copy, "fork": _exact_fork,
                "sparse": _exact_sparse}[case["op"]](st)


def _exact_angles(st, lead):
    """The rotation as complex numbers, one for each token and pair."""
    pos = st["pos"].long()
    return torch.complex(st["cos"].double()[pos], st["sin"].double()[pos]).reshape(lead + (1, -1))


def _exact_pairs(x, half, interleaved):
    """The rotated elements as complex numbers."""
    x = x[..., :2 * half]
    return torch.view_as_complex(x.reshape(x.shape[:-1] + (half, 2)).contiguous()) if interleaved else \
        torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous())


def _exact_turn(x, z, interleaved):
    half = z.shape[-1]
    y = _exact_pairs(x, half, interleaved) * z
    y = torch.view_as_real(y).flatten(-2) if interleaved else torch.cat((y.real, y.imag), dim=-1)
    return torch.cat((y, x[..., 2 * half:]), dim=-1)


def _exact_norm(x, w):
    """(x / rms, rms) in 64 bits, times the weights."""
    rms = (x.pow(2).sum(dim=-1, keepdim=True) / x.shape[-1] + EPS).sqrt()
    return x / rms * w.double(), rms


def _exact_rope(st):
    case, out, dx, dw = st["case"], [], [], []
    for n in ("q", "k"):
        x, w, g = st[n].double(), st["w" + n], st["g" + n].double()
        z = _exact_angles(st, tuple(x.shape[:-2]))
        g = _exact_turn(g, z.conj(), case["interleaved"])
        if w is None:
            out.append(_exact_turn(x, z, case["interleaved"]))
            dx.append(g)
            continue
        y, rms = _exact_norm(x, w)
        out.append(_exact_turn(y, z, case["interleaved"]))
        h = x / rms
        dw.append((g * h).sum(dim=(0, 1, 2)))
        g = g * w.double()
        # d(x / rms): the part along x goes
        along = (g * h).sum(dim=-1, keepdim=True) / x.shape[-1]
        dx.append((g - h * along) / rms)
    return tuple(out + dx + dw)


def _exact_enter(st):
    """Values of the cache afterwards, fp8 codes as the values they stand for without the scale."""
    case = st["case"]
    fmt, page = case["cache"], case["page"]
    new = {}
    for n in ("q", "k"):
        x = st[n].double()
        if case["norm"]:
            x, _ = _exact_norm(x, st["w" + n])
        new[n] = _exact_turn(x, _exact_angles(st, (case["T"],)), case["interleaved"])
    new["v"] = st["v"].double()
    out = {"q": new["q"]}
    has = torch.nonzero(st["slots"] >= 0).flatten()
    p, o = st["slots"][has] // page, st["slots"][has] % page
    for n in ("k", "v"):
        x, pool = new[n][has], st[n + "_cache"].double()
        if fmt in _FP8:
            scale = _FP8_MAX[fmt] / x.abs().amax(dim=2).clamp(min=1e-12)
            x = (x * scale[:, :, None]).clamp(-_FP8_MAX[fmt], _FP8_MAX[fmt]).to(_FP8[fmt]).double()
            inv = st[n + "_scale"].double()
            inv[p, :, o] = 1.0 / scale
        pool[p, :, o] = x
        out[n] = pool
        if fmt in _FP8:
            out[n + "_scale"] = inv
    return {n: out[n] for n in ("q", "k", "v", "k_scale", "v_scale") if n in out}


def _exact_moved(st, pairs):
    out = {}
    for name, key in (("k", "k_cache"), ("v", "v_cache"), ("k_scale", "k_scale"), ("v_scale", "v_scale"), ("ranges", "ranges")):
        x = st.get(key)
        if x is None:
            continue
        y = x.double()
        for s, d in pairs:
            y[:, d] = x[:, s].double()
        out[name] = y
    return out


def _exact_copy(st):
    return _exact_moved(st, list(zip(st["src"].tolist(), st["dst"].tolist())))


def _exact_fork(st):
    """The books of a host that goes through the sequences one by one."""
    case = st["case"]
    page, table, lens = case["page"], st["table"].tolist(), st["lens"].tolist()
    M, P = len(table[0]), st["k_cache"].shape[1]
    parents = st["parents"].tolist()
    everybodys, firsts = set(), {}
    for i, p in enumerate(parents):
        everybodys.update(table[p][:lens[p] // page])
    for i, p in enumerate(parents):
        if lens[p] % page:
            u = table[p][lens[p] // page]
            if u not in everybodys:
                firsts.setdefault(u, i)
    rows, fresh = [], []
    for i, p in enumerate(parents):
        row = [("page", u) for u in table[p][:lens[p] // page]]
        if lens[p] % page:
            u = table[p][lens[p] // page]
            if firsts.get(u) == i:
                row.append(("page", u))
            else:
                row.append(("new", len(fresh)))
                fresh.append(u)
        while len(row) < min(M, -(-(lens[p] + case["reserve"]) // page)):
            row.append(("new", len(fresh)))
            fresh.append(None)
        rows.append(row)
    used = sorted(everybodys | set(firsts))
    free = [u for u in range(P) if u not in set(used)]
    move = {}
    if case["compact"]:
        bound = len(used) + len(fresh)
        movers = [u for u in used if u >= bound]
        move = dict(zip(movers, free))
        free = free[len(movers):]
    pairs = list(move.items()) + [(u, free[n]) for n, u in enumerate(fresh) if u is not None]
    new = torch.full((len(parents), M), -1, dtype=torch.int32)
    for i, row in enumerate(rows):
        for j, (kind, u) in enumerate(row):
            new[i, j] = move.get(u, u) if kind == "page" else free[u]
    return {"table": new.to(DEV), "lens": torch.tensor([lens[p] for p in parents], dtype=torch.int32, device=DEV)} | \
        _exact_moved(st, pairs)


def _exact_sparse(st):
    """Head by head: which pages every token takes, then the softmax over their keys."""
    case = st["case"]
    page, D, group, take = case["page"], case["D"], case["Hq"] // case["Hkv"], case["take"]
    cu, lens = st["cu"].tolist(), st["lens"].tolist()
    out = torch.empty(st["q"].shape, dtype=torch.float64, device=DEV)
    ranges = st["ranges"].double()
    for b, L in enumerate(lens):
        n, pages = cu[b + 1] - cu[b], -(-L // page)
        ids = st["table"][b, :pages].long()
        pos = torch.arange(L - n, L, device=DEV)
        own_page, j = pos // page, torch.arange(pages, device=DEV)
        for h in range(case["Hkv"]):
            kv = []
            for name in ("k", "v"):
                x = st[name + "_cache"][:, h].view(torch.uint8)[ids].view(st[name + "_cache"].dtype).double()
                if st[name + "_scale"] is not None:
                    x = x * st[name + "_scale"][ids, h].double()[..., None]
                kv.append(x.reshape(-1, D)[:L].contiguous())
            for p in range((L - n) // page, pages):
                x = kv[0][p * page:(p + 1) * page].float()  # a key is a 32-bit product
                lo, hi = x.amin(dim=0), x.amax(dim=0)
                ranges[ids[p], h, 0], ranges[ids[p], h, 1] = _exact_outward(lo, -1), _exact_outward(hi, 1)
            q = st["q"][cu[b]:cu[b + 1], h * group:(h + 1) * group].double()
            r = ranges[ids, h]  # [pages, 2, D]
            # the largest that a key within the page's ranges could give, heads together
            score = torch.zeros((n, pages), dtype=torch.float64, device=DEV)
            for one in q.unbind(1):
                score += one.clamp(min=0) @ r[:, 1].t().contiguous() - (-one).clamp(min=0) @ r[:, 0].t().contiguous()
            past = j[None] > own_page[:, None]
            always = (j[None] < case["first"]) | (own_page[:, None] - j[None] < case["last"])
            score[always] = math.inf
            score[past] = -math.inf
            order = torch.sort(score, dim=1, descending=True, stable=True)[1]
            chosen = torch.zeros_like(past).scatter_(1, order[:, :take], True) & ~past
            hidden = ~chosen.repeat_interleave(page, dim=1)[:, :L] | (torch.arange(L, device=DEV)[None] > pos[:, None])
            kt = kv[0].t().contiguous()
            for i in range(group):
                logits = q[:, i].contiguous() @ kt / math.sqrt(D)
                logits[hidden] = -math.inf
                out[cu[b]:cu[b + 1], h * group + i] = torch.softmax(logits, dim=1) @ kv[1]
    return {"out": out, "ranges": ranges}


def _exact_outward(x, sign):
    """The nearest bf16 that is not inside, in 64 bits."""
    y = x.to(torch.bfloat16)
    inside = (y.float() < x) if sign > 0 else (y.float() > x)
    away = torch.full_like(y, sign * math.inf)
    return torch.where(inside, torch.nextafter(y, away), y).double()
