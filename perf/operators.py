"""The operators with which a model answers, as cases that can be timed: the
quantized paged key / value cache as it is written and read back, the attention
of new tokens over that cache, and an expert layer for the few tokens of a
decoding step.

A case is a dict of plain values; ``op`` says which entry point it stands for:

  write   ops.kv_cache_write: the keys and values of new tokens go into their
          cache slots, quantized to fp8 with one scale for each token and head
  read    ops.kv_cache_read: cache slots come back as 16-bit keys and values
  attend  ops.paged_attention: the new tokens of every sequence (one, or a
          chunk of a prompt) attend over the sequence's pages, causally, with
          or without a window and first tokens that stay visible
  moe     ops.moe_decode: SwiGLU experts on weights quantized once

The plain forms are elementary torch operations in 32 bits.
"""

import math
import os
import sys

import torch

#: set by whoever measures: whether run() calls the framework's operators
own = False

DEV = "cuda"
_DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
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
def _attend(name, B, chunk, ctx, Hq, Hkv, D, page, cache="e4m3", dtype="bf16", ragged=True, window=0, sinks=0,
            lse=False):
    return {"name": name, "op": "attend", "B": B, "chunk": chunk, "ctx": ctx, "Hq": Hq, "Hkv": Hkv, "D": D,
            "page": page, "cache": cache, "dtype": dtype, "ragged": ragged, "window": window, "sinks": sinks,
            "lse": lse}


def _cache_op(name, op, tokens, Hkv, D, page, cache="e4m3", dtype="bf16", skip=0):
    return {"name": name, "op": op, "tokens": tokens, "Hkv": Hkv, "D": D, "page": page, "cache": cache,
            "dtype": dtype, "skip": skip}


def _moe(name, T, E, k, I, H, gran, dtype="bf16", fmt="e4m3", away=0):
    return {"name": name, "op": "moe", "T": T, "E": E, "k": k, "I": I, "H": H, "gran": gran, "dtype": dtype,
            "fmt": fmt, "away": away}


def listed():
    return [
        # one decoding step of 64 sequences: the new token of each goes into the cache
        _cache_op("write_64x8x128", "write", 64, 8, 128, 64),
        # the prompt tokens of one step, some of them padding that has no slot
        _cache_op("write_8192x8x128", "write", 8192, 8, 128, 64, skip=100),
        # a prompt's prefix read back, small heads, small pages, a token count that nothing divides
        _cache_op("read_1021x4x64_e5m2_fp16", "read", 1021, 4, 64, 16, cache="e5m2", dtype="fp16"),
        # a long context read back to be moved or checked
        _cache_op("read_131072x8x128", "read", 131072, 8, 128, 64),
        # one sequence answers token by token over a short context: latency counts
        _attend("decode_1x1000_32h8_d128", 1, 1, 1000, 32, 8, 128, 64, ragged=False),
        # a full decoding batch over contexts of all lengths: the cache's bytes count
        _attend("decode_64x16384_64h8_d128", 64, 1, 16384, 64, 8, 128, 64),
        # a chunk of a long prompt over what the cache already has: the products count
        _attend("chunk_2048_of_16384_32h8_d128", 1, 2048, 16384, 32, 8, 128, 128, ragged=False, lse=True),
        # prompts and answers in one step: chunks of all sizes down to one token, a head of its own
        # for each query head, pages of 16 tokens, a 16-bit cache
        _attend("mixed_16x512_of_4096_16h16_d64", 16, 512, 4096, 16, 16, 64, 16, cache="fp16", dtype="fp16"),
        # chunks under a sliding window, the first four tokens always visible
        _attend("window_4x256_of_16384_32h8_d128", 4, 256, 16384, 32, 8, 128, 64, window=1024, sinks=4),
        # one token through a large expert layer
        _moe("moe_1_top8_of_32x2048x7168", 1, 32, 8, 2048, 7168, "BLOCKWISE"),
        # a small expert layer, sizes that are no multiple of a tile, per-row scales, some experts on another rank
        _moe("moe_7_top2_of_8x1360x2064_fp16", 7, 8, 2, 1360, 2064, "ROWWISE", dtype="fp16", away=2),
        # a decoding batch of 64 tokens through the large layer, per-tensor scales
        _moe("moe_64_top8_of_32x2048x7168", 64, 32, 8, 2048, 7168, "TENSORWISE"),
    ]


def _log(rng, lo, hi, mult=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(mult, int(v / mult + 0.5) * mult)


_PAIRS = 1 * 32 * 2048 * 16384  # query-key pairs of the largest listed chunk, padded
_CACHE = 64 * 16384 * 8 * 128  # bytes of keys of the largest listed batch, padded


def _nameless(case):
    return {n: v for n, v in case.items() if n != "name"}


def draw(rng):
    op = rng.choice(("write", "read", "attend", "attend", "attend", "moe"))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    cache = rng.choice(("e4m3", "e4m3", "e4m3", "e5m2", dtype))
    Hkv, D = rng.choice((1, 2, 4, 8, 16)), rng.choice((64, 128, 128, 128, 256))
    page = rng.choice((16, 32, 64, 128, 48))
    if op in ("write", "read"):
        most = 131072 * 8 * 128 if op == "read" else 8192 * 8 * 128
        tokens = _log(rng, 4, most // (Hkv * D))
        return _nameless(_cache_op("", op, tokens, Hkv, D, page, cache, dtype,
                                   rng.choice((0, 0, 3)) if op == "write" else 0))
    if op == "moe":
        while True:
            E, k = rng.choice((4, 8, 16, 32, 64)), rng.choice((1, 2, 4, 8))
            c = _moe("", _log(rng, 1, 64), E, min(k, E // 2), _log(rng, 128, 2048, 16), _log(rng, 256, 7168, 16),
                     rng.choice(("BLOCKWISE", "ROWWISE", "TENSORWISE", "NONE")), dtype, rng.choice(("e4m3", "e4m3", "e5m2")),
                     rng.choice((0, 0, 1)))
            if c["E"] * c["I"] * c["H"] * (2 if c["gran"] == "NONE" else 1) <= 32 * 2048 * 7168:
                return _nameless(c)
    while True:
        kind = rng.choice(("decode", "chunk", "mixed"))
        B = 1 if kind == "chunk" and rng.random() < 0.5 else _log(rng, 1, 64)
        chunk = 1 if kind == "decode" else _log(rng, 2, 2048)
        ctx = _log(rng, max(16, chunk), 32768)
        Hq = Hkv * rng.choice((1, 2, 4, 8))
        window = rng.choice((0, 0, 0, 128, 1000, 4096))
        c = _attend("", B, chunk, ctx, Hq, Hkv, D, page, cache, dtype, kind != "chunk" or rng.random() < 0.5,
                    window, rng.choice((0, 1, 4, 16)) if window else 0, rng.random() < 0.3)
        size = 1 if cache in _FP8 else 2
        if B * ctx * Hkv * D * size <= _CACHE and B * Hq * chunk * ctx * max(D, 128) <= _PAIRS * 128:
            return _nameless(c)


# ---------------------------------------------------------------------------
# lengths of the sequences: the case's own, so that its work is known
# ---------------------------------------------------------------------------
def _lengths(case):
    """(new tokens, length with them) of every sequence."""
    B, chunk, ctx = case["B"], case["chunk"], case["ctx"]
    if not case["ragged"]:
        return [chunk] * B, [ctx] * B
    g = torch.Generator().manual_seed(B * 100003 + ctx)
    u, w = torch.rand(B, generator=g).tolist(), torch.rand(B, generator=g).tolist()
    new = [max(1, int(round(chunk ** x))) for x in u]
    new[0] = chunk
    if B > 1 and chunk > 1:
        new[-1] = 1
    lens = [max(n, int(ctx * (0.1 + 0.9 * x))) for n, x in zip(new, w)]
    lens[0] = ctx
    return new, lens


def _pairs(new, length, window, sinks):
    """(query-key pairs, keys that any of the new tokens sees) of one sequence."""
    if not window:
        return new * (length - new) + new * (new + 1) // 2, length
    pairs = 0
    for i in range(length - new, length):
        lo = max(0, i - window + 1)
        pairs += i + 1 - lo + min(sinks, lo)
    lo = max(0, length - new - window + 1)
    return pairs, length - lo + min(sinks, lo)


def work(case):
    op = case["op"]
    if op in ("write", "read"):
        rows = (case["tokens"] - case["skip"]) * case["Hkv"] * 2
        D, fp8 = case["D"], case["cache"] in _FP8
        return {"bytes": rows * (2 * D + (D + 4 if fp8 else 2 * D)) + 8 * case["tokens"], "flops": 3.0 * rows * D}
    if op == "moe":
        T, E, k, I, H = (case[x] for x in ("T", "E", "k", "I", "H"))
        # experts that T tokens reach, on average
        n = (E - case["away"]) * (1 - (1 - k / E) ** T)
        w = 2 if case["gran"] == "NONE" else 1
        return {"bytes": n * 3 * I * H * w + 4 * T * H, "flops": 2.0 * 3 * I * H * T * k * (1 - case["away"] / E)}
    new, lens = _lengths(case)
    seen = [_pairs(n, L, case["window"], case["sinks"]) for n, L in zip(new, lens)]
    per = 2 * (case["D"] + 4) if case["cache"] in _FP8 else 4 * case["D"]
    q = sum(new) * case["Hq"] * case["D"]
    return {"bytes": sum(s for _, s in seen) * case["Hkv"] * per + 4 * q + (4 * q // case["D"] if case["lse"] else 0),
            "flops": 4.0 * case["Hq"] * case["D"] * sum(p for p, _ in seen)}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _randn(shape, g):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32)


def _rows_to_fp8(x, fmt):
    """One scale for each row of the last axis: (fp8, inverse scales)."""
    s = _FP8_MAX[fmt] / x.abs().amax(dim=-1).clamp(min=1e-12)
    return (x * s.unsqueeze(-1)).clamp(-_FP8_MAX[fmt], _FP8_MAX[fmt]).to(_FP8[fmt]), 1.0 / s


def _pool(pages, case, g):
    """Cache pages with content: channels of different strength, as keys and values have them."""
    Hkv, page, D = case["Hkv"], case["page"], case["D"]
    strength = torch.exp(0.5 * _randn((1, Hkv, 1, D), g))
    x = torch.empty((pages, Hkv, page, D), dtype=_FP8.get(case["cache"]) or _DT[case["cache"]], device=DEV)
    s = torch.empty((pages, Hkv, page), dtype=torch.float32, device=DEV) if case["cache"] in _FP8 else None
    step = max(1, (1 << 27) // (Hkv * page * D))
    for p in range(0, pages, step):
        n = min(step, pages - p)
        v = _randn((n, Hkv, page, D), g) * strength
        if s is None:
            x[p:p + n] = v.to(x.dtype)
        else:
            x[p:p + n], s[p:p + n] = _rows_to_fp8(v, case["cache"])
    return x, s


def _experts(E, N, K, case, g):
    """Expert weights [E, N, K] quantized once: (data, inverse scales)."""
    gran, fmt = case["gran"], case["fmt"]
    dt = _DT[case["dtype"]]
    w = torch.empty((E, N, K), dtype=dt if gran == "NONE" else _FP8[fmt], device=DEV)
    if gran == "NONE":
        for e in range(E):
            w[e] = (0.02 * _randn((N, K), g)).to(dt)
        return w, None
    m = _FP8_MAX[fmt]
    s = {"TENSORWISE": torch.empty((), device=DEV), "ROWWISE": torch.empty((E, N, 1), device=DEV),
         "BLOCKWISE": torch.empty((E, -(-N // 128), -(-K // 128)), device=DEV)}[gran]
    if gran == "TENSORWISE":
        s.fill_(0.12 / m)  # six standard deviations
    for e in range(E):
        x = 0.02 * _randn((N, K), g)
        if gran == "TENSORWISE":
            up = s
        elif gran == "ROWWISE":
            s[e] = x.abs().amax(dim=1, keepdim=True) / m
            up = s[e]
        else:
            p = torch.zeros((s.shape[1] * 128, s.shape[2] * 128), device=DEV)
            p[:N, :K] = x
            s[e] = p.view(s.shape[1], 128, s.shape[2], 128).abs().amax(dim=(1, 3)) / m
            up = _spread(s[e], N, K)
        w[e] = (x / up).clamp(-m, m).to(w.dtype)
    return w, s


def _spread(s, N, K):
    """Block scales [..., N/128, K/128] as one for each element, [..., N, K]."""
    return s.repeat_interleave(128, dim=-2)[..., :N, :].repeat_interleave(128, dim=-1)[..., :K]


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    op, dt = case["op"], _DT[case["dtype"]]
    st = {"case": case, "dt": dt}
    if op in ("write", "read"):
        T, Hkv, D, page = case["tokens"], case["Hkv"], case["D"], case["page"]
        pages = -(-T // page) + 3
        for n in ("k", "v"):
            st[n + "_cache"], st[n + "_scale"] = _pool(pages, case, g)
        # whole pages in any order, the tokens of a page in theirs
        at = torch.randperm(pages, generator=g, device=DEV)
        pos = torch.arange(T, device=DEV)
        st["slots"] = at[pos // page] * page + pos % page
        if op == "write":
            if case["skip"]:
                st["slots"][torch.randperm(T, generator=g, device=DEV)[:case["skip"]]] = -1
            # k and v are the last two parts of a projection's output, as a model has them
            qkv = torch.empty((T, 3, Hkv, D), dtype=dt, device=DEV).copy_(_randn((T, 3, Hkv, D), g))
            st["k"], st["v"] = qkv[:, 1], qkv[:, 2]
        return st
    if op == "attend":
        B, Hq, D, page = case["B"], case["Hq"], case["D"], case["page"]
        new, lens = _lengths(case)
        most = -(-max(lens) // page)
        need = [-(-n // page) for n in lens]
        pages = sum(need) + 1
        for n in ("k", "v"):
            st[n + "_cache"], st[n + "_scale"] = _pool(pages, case, g)
        order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
        table = torch.full((B, most), -1, dtype=torch.int32, device=DEV)
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = order[at:at + n]
            at += n
        st["table"] = table
        st["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        st["cu"] = torch.tensor([sum(new[:b]) for b in range(B + 1)], dtype=torch.int32, device=DEV)
        st["q"] = _randn((sum(new), Hq, D), g).to(dt)
        st["most_new"], st["most_len"] = max(new), most * page
        return st
    T, E, k, I, H = (case[x] for x in ("T", "E", "k", "I", "H"))
    st["w1"], st["s1"] = _experts(E, 2 * I, H, case, g)
    st["w2"], st["s2"] = _experts(E, H, I, case, g)
    st["x"] = _randn((T, H), g).to(dt)
    logits = _randn((T, E), g)
    top, idx = torch.topk(logits, k, dim=1)
    st["probs"] = torch.softmax(top, dim=1)
    # experts at the end of the list live on another rank
    st["idx"] = torch.where(idx < E - case["away"], idx, torch.full_like(idx, -1))
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(st):
    op = st["case"]["op"]
    if own:
        ops = _ops()
        if op == "write":
            ops.kv_cache_write(st["k"], st["v"], st["k_cache"], st["v_cache"], st["slots"], st["k_scale"], st["v_scale"])
            return _written(st)
        if op == "read":
            return ops.kv_cache_read(st["k_cache"], st["v_cache"], st["slots"], st["k_scale"], st["v_scale"],
                                     out_dtype=st["dt"])
        if op == "attend":
            case = st["case"]
            return ops.paged_attention(st["q"], st["k_cache"], st["v_cache"], st["table"], st["cu"], st["lens"],
                                       st["k_scale"], st["v_scale"], window_size=case["window"] or None,
                                       num_sinks=case["sinks"], return_lse=case["lse"])
        return ops.moe_decode(st["x"], st["w1"], st["w2"], st["idx"], st["probs"], st["s1"], st["s2"])
    return {"write": _plain_write, "read": _plain_read, "attend": _plain_attend, "moe": _plain_moe}[op](st)


def _written(st):
    out = {"k": st["k_cache"], "v": st["v_cache"]}
    if st["k_scale"] is not None:
        out |= {"k_scale": st["k_scale"], "v_scale": st["v_scale"]}
    return out


def _plain_write_one(x, cache, scale, slots, fmt):
    page = cache.shape[2]
    if scale is None:
        cache[slots // page, :, slots % page] = x
        return
    q, inv = _rows_to_fp8(x.float(), fmt)
    # torch moves fp8 values through index_put as bytes
    cache.view(torch.uint8)[slots // page, :, slots % page] = q.view(torch.uint8)
    scale[slots // page, :, slots % page] = inv


def _plain_write(st):
    slots, k, v, fmt = st["slots"], st["k"], st["v"], st["case"]["cache"]
    if st["case"]["skip"]:
        has = slots >= 0
        slots, k, v = slots[has], k[has], v[has]
    _plain_write_one(k, st["k_cache"], st["k_scale"], slots, fmt)
    _plain_write_one(v, st["v_cache"], st["v_scale"], slots, fmt)
    return _written(st)


def _plain_read(st):
    slots, page = st["slots"], st["case"]["page"]
    at = slots // page, slice(None), slots % page
    if st["k_scale"] is None:
        return st["k_cache"][at], st["v_cache"][at]
    return tuple((c.view(torch.uint8)[at].view(c.dtype).float() * s[at].unsqueeze(-1)).to(st["dt"])
                 for c, s in ((st["k_cache"], st["k_scale"]), (st["v_cache"], st["v_scale"])))


def _plain_keys(cache, scale, table):
    """The pages of every sequence in a row, in 32 bits: [B, Hkv, length, D]."""
    B, n = table.shape
    _, Hkv, page, D = cache.shape
    at = table.clamp(min=0).long()
    x = cache.view(torch.uint8)[at].view(cache.dtype).float()  # [B, n, Hkv, page, D]
    if scale is not None:
        x = x * scale[at].unsqueeze(-1)
    return x.permute(0, 2, 1, 3, 4).reshape(B, Hkv, n * page, D)


def _plain_attend(st):
    case, q, cu, lens, M = st["case"], st["q"], st["cu"].long(), st["lens"].long(), st["most_new"]
    B, Hq, Hkv, D, L = case["B"], case["Hq"], case["Hkv"], case["D"], st["most_len"]
    k = _plain_keys(st["k_cache"], st["k_scale"], st["table"])
    v = _plain_keys(st["v_cache"], st["v_scale"], st["table"])
    # new tokens of every sequence, padded to the longest chunk
    i = torch.arange(M, device=DEV)
    new = cu[1:] - cu[:-1]
    there = i < new[:, None]
    at = (cu[:-1, None] + i).clamp(max=q.shape[0] - 1)
    qq = q[at].float().view(B, M, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, Hq // Hkv * M, D)
    s = torch.matmul(qq, k.transpose(2, 3).contiguous()).view(B, Hkv, Hq // Hkv, M, L) * D ** -0.5
    pos = (lens - new)[:, None] + i  # [B, M]
    j = torch.arange(L, device=DEV)
    seen = j <= pos[:, :, None]
    if case["window"]:
        seen = seen & ((j > pos[:, :, None] - case["window"]) | (j < case["sinks"]))
    s.masked_fill_(~seen[:, None, None], float("-inf"))
    m = s.amax(dim=-1, keepdim=True)
    p = s.sub_(m).exp_()
    l = p.sum(dim=-1, keepdim=True)
    o = torch.matmul(p.view(B, Hkv, Hq // Hkv * M, L), v).view(B, Hkv, Hq // Hkv, M, D) / l
    # back to packed tokens: the b-th sequence's i-th token is row cu[b] + i
    o = o.permute(0, 3, 1, 2, 4).reshape(B, M, Hq, D)
    rows = torch.repeat_interleave(torch.arange(B, device=DEV), new, output_size=q.shape[0])
    at = rows, torch.arange(q.shape[0], device=DEV) - cu[rows]
    out = o[at].to(q.dtype)
    if not case["lse"]:
        return out
    return out, (m + l.log()).permute(0, 3, 1, 2, 4).reshape(B, M, Hq)[at]


def _plain_weight(w, s, gran, sel):
    x = w.view(torch.uint8)[sel].view(w.dtype).float() if s is not None else w[sel].float()
    if s is None:
        return x
    if gran == "TENSORWISE":
        return x * s
    return x * (s[sel] if gran == "ROWWISE" else _spread(s[sel], w.shape[1], w.shape[2]))


def _plain_moe(st):
    case, x, idx = st["case"], st["x"].float(), st["idx"]
    T, E, k, gran = case["T"], case["E"], case["k"], case["gran"]
    if T * k <= E:
        # few tokens: only the experts that they go to
        sel = idx.reshape(-1).clamp(min=0)
        token = torch.arange(T, device=DEV).repeat_interleave(k)
        weight = torch.zeros((T * k, T), device=DEV)
        weight[torch.arange(T * k, device=DEV), token] = torch.where(idx >= 0, st["probs"], 0.0).reshape(-1)
    else:
        sel = torch.arange(E, device=DEV)
        weight = torch.where(idx[None] == sel[:, None, None], st["probs"][None], 0.0).sum(dim=2)
    h = torch.matmul(x, _plain_weight(st["w1"], st["s1"], gran, sel).transpose(1, 2))  # [S, T, 2I]
    gate, up = h.chunk(2, dim=2)
    a = gate / (1.0 + torch.exp(-gate)) * up * weight.unsqueeze(-1)
    y = torch.matmul(a, _plain_weight(st["w2"], st["s2"], gran, sel).transpose(1, 2))
    return y.sum(dim=0).to(st["dt"])


# ---------------------------------------------------------------------------
# what a correct answer is, in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    st, op = prepare(case, seed), case["op"]
    return {"write": _exact_write, "read": _exact_read, "attend": _exact_attend, "moe": _exact_moe}[op](st)


def _exact_write(st):
    """Values of the cache after the write, fp8 codes as the values they stand for without the scale."""
    fmt, page = st["case"]["cache"], st["case"]["page"]
    out = {}
    has = torch.nonzero(st["slots"] >= 0).flatten()
    p, o = st["slots"][has] // page, st["slots"][has] % page
    for n in ("k", "v"):
        x = st[n][has].double()
        pool = st[n + "_cache"].double()
        if fmt in _FP8:
            scale = _FP8_MAX[fmt] / x.abs().amax(dim=2).clamp(min=1e-12)
            x = (x * scale[:, :, None]).clamp(-_FP8_MAX[fmt], _FP8_MAX[fmt]).to(_FP8[fmt]).double()
            inv = st[n + "_scale"].double()
            inv[p, :, o] = 1.0 / scale
            out[n + "_scale"] = inv
        pool[p, :, o] = x
        out[n] = pool
    return out


def _exact_read(st):
    page, got = st["case"]["page"], []
    rows = torch.div(st["slots"], page, rounding_mode="floor")
    for n in ("k", "v"):
        # chunks keep the 64-bit copies small
        part = []
        for a in range(0, rows.numel(), 16384):
            p, o = rows[a:a + 16384], st["slots"][a:a + 16384] % page
            x = st[n + "_cache"].view(torch.uint8)[p, :, o].view(st[n + "_cache"].dtype).double()
            part.append(x if st[n + "_scale"] is None else x * st[n + "_scale"][p, :, o].double()[..., None])
        got.append(torch.cat(part))
    return tuple(got)


def _exact_attend(st):
    """Sequence by sequence and head by head, the softmax over the keys that a token sees."""
    case = st["case"]
    cu, lens, page = st["cu"].tolist(), st["lens"].tolist(), case["page"]
    group, D = case["Hq"] // case["Hkv"], case["D"]
    out = torch.empty(st["q"].shape, dtype=torch.float64, device=DEV)
    lse = torch.empty(st["q"].shape[:2], dtype=torch.float64, device=DEV)
    for b, L in enumerate(lens):
        n = cu[b + 1] - cu[b]
        ids = st["table"][b, :-(-L // page)].long()
        q_at = torch.arange(L - n, L, device=DEV)[:, None]
        k_at = torch.arange(L, device=DEV)[None]
        hidden = k_at > q_at
        if case["window"]:
            hidden |= (q_at - k_at >= case["window"]) & (k_at >= case["sinks"])
        for h in range(case["Hkv"]):
            kv = []
            for name in ("k", "v"):
                x = st[name + "_cache"][:, h].view(torch.uint8)[ids].view(st[name + "_cache"].dtype).double()
                if st[name + "_scale"] is not None:
                    x = x * st[name + "_scale"][ids, h].double()[..., None]
                kv.append(x.reshape(-1, D)[:L].contiguous())
            kt = kv[0].t().contiguous()
            for r in range(h * group, h * group + group):
                logits = st["q"][cu[b]:cu[b + 1], r].double() @ kt / math.sqrt(D)
                logits[hidden] = -math.inf
                lse[cu[b]:cu[b + 1], r] = torch.logsumexp(logits, dim=1)
                out[cu[b]:cu[b + 1], r] = torch.softmax(logits, dim=1) @ kv[1]
    return (out, lse) if case["lse"] else out


def _exact_moe(st):
    """Expert by expert, the tokens that go to it."""
    case = st["case"]
    x, I = st["x"].double(), case["I"]
    y = torch.zeros(x.shape, dtype=torch.float64, device=DEV)

    def weight(w, s, e):
        d = w[e].double()
        if s is None:
            return d
        s = s.double()
        if case["gran"] == "TENSORWISE":
            return d * s
        if case["gran"] == "ROWWISE":
            return d * s[e]
        n, k = torch.arange(d.shape[0], device=DEV) // 128, torch.arange(d.shape[1], device=DEV) // 128
        return d * s[e][n][:, k]

    for e in range(case["E"]):
        t, j = torch.nonzero(st["idx"] == e, as_tuple=True)
        if not t.numel():
            continue
        h = x[t] @ weight(st["w1"], st["s1"], e).t().contiguous()
        a = torch.nn.functional.silu(h[:, :I]) * h[:, I:]
        y.index_add_(0, t, a @ weight(st["w2"], st["s2"], e).t().contiguous() * st["probs"][t, j].double()[:, None])
    return y
