"""Host side of the paged cache and attention kernels: argument checks, output
and workspace allocation, the calls into libprimus_turbo_amd.so."""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
from torch.autograd.graph import increment_version

from primus_turbo.pytorch import _C
from primus_turbo.pytorch.core.inference import check_tensors
from primus_turbo.pytorch.core.low_precision import float8_e4m3, float8_e5m2

_SIXTEEN = (torch.bfloat16, torch.float16)
_KIND = {float8_e4m3: _C.PTA_E4M3, float8_e5m2: _C.PTA_E5M2, torch.bfloat16: _C.CACHE_16BIT, torch.float16: _C.CACHE_16BIT}
_IN = {torch.bfloat16: _C.PTA_BF16, torch.float16: _C.PTA_F16, torch.float32: _C.PTA_F32}
_increment_version = getattr(torch._C, "_increment_version", None) or increment_version  # 0.3 us less


def _check_cache(k_cache, v_cache, k_scale_inv, v_scale_inv):
    """(kind, shape) of a pool pair after checking its shapes, types and layout."""
    shape, dtype = k_cache.shape, k_cache.dtype
    assert len(shape) == 4 and v_cache.shape == shape, (
        f"caches must be [num_pages, Hkv, page_size, D], both alike: got {tuple(shape)}, {tuple(v_cache.shape)}"
    )
    assert v_cache.dtype == dtype, "k_cache and v_cache must have one type"
    kind = _KIND.get(dtype)
    assert kind is not None, f"unsupported cache type {dtype}"
    assert k_cache.is_contiguous() and v_cache.is_contiguous(), "caches must be contiguous"
    _, Hkv, page, D = shape
    assert D % 16 == 0 and 16 <= D <= 256, f"head_dim must be a multiple of 16 in [16, 256], got {D}"
    assert page > 0 and Hkv > 0, "page_size and the number of heads must not be 0"
    if kind == _C.CACHE_16BIT:
        assert k_scale_inv is None and v_scale_inv is None, "a 16-bit cache has no scales"
    else:
        assert k_scale_inv is not None and v_scale_inv is not None, "an fp8 cache needs k_scale_inv and v_scale_inv"
        want = shape[:3]
        for s in (k_scale_inv, v_scale_inv):
            assert s.shape == want and s.dtype == torch.float32 and s.is_contiguous(), (
                f"scale_inv must be contiguous float32 {tuple(want)}, got {s.dtype} {tuple(s.shape)}"
            )
    return kind, shape


def _check_slots(slots: torch.Tensor) -> int:
    """Number of slots."""
    shape = slots.shape
    assert len(shape) == 1 and slots.dtype in (torch.int64, torch.int32), "slots must be one-dimensional int32 / int64"
    assert slots.is_contiguous(), "slots must be contiguous"
    return shape[0]


def kv_cache_write_impl(k, v, k_cache, v_cache, slots, k_scale_inv, v_scale_inv) -> None:
    kind, (P, Hkv, page, D) = _check_cache(k_cache, v_cache, k_scale_inv, v_scale_inv)
    shape, dtype = k.shape, k.dtype
    assert len(shape) == 3 and shape[1] == Hkv and shape[2] == D and v.shape == shape, (
        f"k and v must be [T, {Hkv}, {D}], got {tuple(shape)}, {tuple(v.shape)}"
    )
    assert v.dtype == dtype, "k and v must have one type"
    assert kind != _C.CACHE_16BIT or dtype == k_cache.dtype, "a 16-bit cache takes keys and values of its type"
    dt = _IN.get(dtype)
    if dt is None:
        raise TypeError(f"unsupported key / value type {dtype}")
    T = shape[0]
    n = _check_slots(slots)
    assert n == T, f"one slot for each of the {T} tokens, got {n}"
    check_tensors("kv_cache_write", (k, v, k_cache, v_cache, k_scale_inv, v_scale_inv), slots)
    if T == 0:
        return
    ks, vs = k.stride(), v.stride()
    if ks[2] != 1:
        k = k.contiguous()
        ks = k.stride()
    if vs[2] != 1:
        v = v.contiguous()
        vs = v.stride()
    fp8 = kind != _C.CACHE_16BIT
    _C.call(
        "pta_kv_cache_write", k.data_ptr(), v.data_ptr(), dt, T, Hkv, D, ks[0], ks[1], vs[0], vs[1], slots.data_ptr(),
        slots.dtype == torch.int64, k_cache.data_ptr(), v_cache.data_ptr(), kind, P, page,
        k_scale_inv.data_ptr() if fp8 else None, v_scale_inv.data_ptr() if fp8 else None, _C.stream(k.device),
    )
    # torch's count of a tensor's changes, which autograd compares with what it has saved
    _increment_version((k_cache, v_cache, k_scale_inv, v_scale_inv) if fp8 else (k_cache, v_cache))


def kv_cache_read_impl(k_cache, v_cache, slots, k_scale_inv, v_scale_inv, out_dtype) -> Tuple[torch.Tensor, torch.Tensor]:
    kind, (P, Hkv, page, D) = _check_cache(k_cache, v_cache, k_scale_inv, v_scale_inv)
    T = _check_slots(slots)
    dt = _IN.get(out_dtype)
    if dt is None:
        raise TypeError(f"unsupported output type {out_dtype}")
    fp8 = kind != _C.CACHE_16BIT
    assert fp8 or out_dtype == k_cache.dtype, f"a {k_cache.dtype} cache is read back as it is"
    check_tensors("kv_cache_read", (k_cache, v_cache, k_scale_inv, v_scale_inv), slots)
    dev = k_cache.device
    k = torch.empty((T, Hkv, D), dtype=out_dtype, device=dev)
    v = torch.empty_like(k)
    if T > 0:
        _C.call(
            "pta_kv_cache_read", k_cache.data_ptr(), v_cache.data_ptr(), kind, P, page, Hkv, D,
            k_scale_inv.data_ptr() if fp8 else None, v_scale_inv.data_ptr() if fp8 else None, slots.data_ptr(),
            slots.dtype == torch.int64, T, k.data_ptr(), v.data_ptr(), dt, _C.stream(dev),
        )
    return k, v


def paged_attention_impl(
    q, k_cache, v_cache, page_table, cu_seqlens_q, seq_lens, k_scale_inv, v_scale_inv, softmax_scale, window_size,
    num_sinks, return_lse,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    kind, (P, Hkv, page, D) = _check_cache(k_cache, v_cache, k_scale_inv, v_scale_inv)
    shape, dtype = q.shape, q.dtype
    assert len(shape) == 3 and shape[2] == D, f"q must be [T, Hq, {D}], got {tuple(shape)}"
    assert dtype in _SIXTEEN, f"q must be bfloat16 or float16, got {dtype}"
    fp8 = kind != _C.CACHE_16BIT
    assert fp8 or dtype == k_cache.dtype, "a 16-bit cache takes queries of its type"
    T, Hq, _ = shape
    assert Hq > 0 and Hq % Hkv == 0, f"query heads ({Hq}) must be a multiple of cache heads ({Hkv})"
    i32 = torch.int32
    lens_shape, table_shape = seq_lens.shape, page_table.shape
    assert len(lens_shape) == 1 and seq_lens.dtype == i32 and seq_lens.is_contiguous(), (
        "seq_lens must be contiguous one-dimensional int32"
    )
    B = lens_shape[0]
    assert cu_seqlens_q.dtype == i32 and cu_seqlens_q.shape == (B + 1,) and cu_seqlens_q.is_contiguous(), (
        f"cu_seqlens_q must be contiguous int32 [{B + 1}]"
    )
    assert len(table_shape) == 2 and page_table.dtype == i32 and table_shape[0] == B, f"page_table must be int32 [{B}, max_pages]"
    M = table_shape[1]
    table_stride = page_table.stride()
    assert M <= 1 or table_stride[1] == 1, "rows of page_table must be contiguous"
    assert T == 0 or B > 0, "tokens without a sequence"
    assert window_size is None or window_size > 0, f"window_size must be positive or None, got {window_size}"
    assert num_sinks >= 0, "num_sinks must not be negative"
    if softmax_scale is None:
        scale = D ** -0.5
    else:
        scale = float(softmax_scale)
        assert math.isfinite(scale), "softmax_scale must be finite"
    check_tensors("paged_attention", (q, k_cache, v_cache, k_scale_inv, v_scale_inv), page_table, cu_seqlens_q, seq_lens)
    qs = q.stride()
    if qs[2] != 1 or qs[0] % 8 or qs[1] % 8 or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
        qs = q.stride()
    dev = q.device
    out = torch.empty(shape, dtype=dtype, device=dev)
    lse = torch.empty((T, Hq), dtype=torch.float32, device=dev) if return_lse else None
    if T > 0:
        reach = M * page
        # windows past the table's reach hide nothing
        win = 0 if window_size is None or window_size >= reach else int(window_size)
        nbytes = _C.query("pta_paged_attention_workspace_size", T, B, Hq, Hkv, D, M, page)
        ws = _C.workspace(nbytes, dev)
        _C.call(
            "pta_paged_attention", q.data_ptr(), _IN[dtype], T, Hq, D, qs[0], qs[1], k_cache.data_ptr(),
            v_cache.data_ptr(), kind, P, page, Hkv, k_scale_inv.data_ptr() if fp8 else None,
            v_scale_inv.data_ptr() if fp8 else None, page_table.data_ptr(), table_stride[0], M, cu_seqlens_q.data_ptr(),
            seq_lens.data_ptr(), B, scale, win, min(int(num_sinks), reach), out.data_ptr(),
            None if lse is None else lse.data_ptr(), None if ws is None else ws.data_ptr(), max(nbytes, 0), _C.stream(dev),
        )
    return out, lse
