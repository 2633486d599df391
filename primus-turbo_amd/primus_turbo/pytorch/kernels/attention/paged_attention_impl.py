"""Host side of the paged cache and attention kernels: argument checks, output
and workspace allocation, the calls into libprimus_turbo_amd.so."""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from primus_turbo.pytorch import _C
from primus_turbo.pytorch.core.low_precision import float8_e4m3, float8_e5m2

_SIXTEEN = (torch.bfloat16, torch.float16)


def _no_grad(what: str, *tensors: torch.Tensor) -> None:
    assert not (torch.is_grad_enabled() and any(t.requires_grad for t in tensors)), (
        f"{what} has no backward pass: call it under torch.no_grad() or on detached tensors"
    )


def _check_cache(k_cache, v_cache, k_scale_inv, v_scale_inv) -> int:
    """Cache kind of a pool pair after checking its shapes, types and layout."""
    assert k_cache.ndim == 4 and k_cache.shape == v_cache.shape, (
        f"caches must be [num_pages, Hkv, page_size, D], both alike: got {tuple(k_cache.shape)}, {tuple(v_cache.shape)}"
    )
    assert k_cache.dtype == v_cache.dtype, "k_cache and v_cache must have one type"
    assert k_cache.is_contiguous() and v_cache.is_contiguous(), "caches must be contiguous"
    D = k_cache.shape[3]
    assert D % 16 == 0 and 16 <= D <= 256, f"head_dim must be a multiple of 16 in [16, 256], got {D}"
    assert k_cache.shape[2] > 0 and k_cache.shape[1] > 0, "page_size and the number of heads must not be 0"
    if k_cache.dtype in _SIXTEEN:
        assert k_scale_inv is None and v_scale_inv is None, "a 16-bit cache has no scales"
        kind = _C.CACHE_16BIT
    else:
        assert k_cache.dtype in (float8_e4m3, float8_e5m2), f"unsupported cache type {k_cache.dtype}"
        assert k_scale_inv is not None and v_scale_inv is not None, "an fp8 cache needs k_scale_inv and v_scale_inv"
        for s in (k_scale_inv, v_scale_inv):
            assert s.dtype == torch.float32 and s.shape == k_cache.shape[:3] and s.is_contiguous(), (
                f"scale_inv must be contiguous float32 {tuple(k_cache.shape[:3])}, got {s.dtype} {tuple(s.shape)}"
            )
        kind = _C.fp8_code(k_cache.dtype)
    return kind


def _check_devices(first: torch.Tensor, *more: Optional[torch.Tensor]) -> None:
    dev = first.device
    assert all(t is None or t.device == dev for t in more), f"all tensors must be on {dev}"


def _check_slots(slots: torch.Tensor) -> None:
    assert slots.ndim == 1 and slots.dtype in (torch.int32, torch.int64), "slots must be one-dimensional int32 / int64"
    assert slots.is_contiguous(), "slots must be contiguous"


def kv_cache_write_impl(k, v, k_cache, v_cache, slots, k_scale_inv, v_scale_inv) -> None:
    kind = _check_cache(k_cache, v_cache, k_scale_inv, v_scale_inv)
    P, Hkv, page, D = k_cache.shape
    assert k.ndim == 3 and k.shape == v.shape and k.shape[1:] == (Hkv, D), (
        f"k and v must be [T, {Hkv}, {D}], got {tuple(k.shape)}, {tuple(v.shape)}"
    )
    assert k.dtype == v.dtype, "k and v must have one type"
    assert kind != _C.CACHE_16BIT or k.dtype == k_cache.dtype, "a 16-bit cache takes keys and values of its type"
    dt = _C.in_dtype_code(k.dtype)
    _check_slots(slots)
    T = k.shape[0]
    assert slots.shape[0] == T, f"one slot for each of the {T} tokens, got {slots.shape[0]}"
    _check_devices(k, v, k_cache, v_cache, slots, k_scale_inv, v_scale_inv)
    _no_grad("kv_cache_write", k, v)
    if T == 0:
        return
    if k.stride(2) != 1:
        k = k.contiguous()
    if v.stride(2) != 1:
        v = v.contiguous()
    _C.call(
        "pta_kv_cache_write", k.data_ptr(), v.data_ptr(), dt, T, Hkv, D, k.stride(0), k.stride(1), v.stride(0),
        v.stride(1), slots.data_ptr(), int(slots.dtype == torch.int64), k_cache.data_ptr(), v_cache.data_ptr(), kind,
        P, page, _C.ptr(k_scale_inv), _C.ptr(v_scale_inv), _C.stream(k.device),
    )


def kv_cache_read_impl(k_cache, v_cache, slots, k_scale_inv, v_scale_inv, out_dtype) -> Tuple[torch.Tensor, torch.Tensor]:
    kind = _check_cache(k_cache, v_cache, k_scale_inv, v_scale_inv)
    P, Hkv, page, D = k_cache.shape
    _check_slots(slots)
    _check_devices(k_cache, v_cache, slots, k_scale_inv, v_scale_inv)
    assert kind != _C.CACHE_16BIT or out_dtype == k_cache.dtype, f"a {k_cache.dtype} cache is read back as it is"
    dt = _C.out_dtype_code(out_dtype)
    T = slots.shape[0]
    k = torch.empty((T, Hkv, D), dtype=out_dtype, device=k_cache.device)
    v = torch.empty_like(k)
    if T > 0:
        _C.call(
            "pta_kv_cache_read", k_cache.data_ptr(), v_cache.data_ptr(), kind, P, page, Hkv, D, _C.ptr(k_scale_inv),
            _C.ptr(v_scale_inv), slots.data_ptr(), int(slots.dtype == torch.int64), T, k.data_ptr(), v.data_ptr(), dt,
            _C.stream(k_cache.device),
        )
    return k, v


def paged_attention_impl(
    q, k_cache, v_cache, page_table, cu_seqlens_q, seq_lens, k_scale_inv, v_scale_inv, softmax_scale, window_size,
    num_sinks, return_lse,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    kind = _check_cache(k_cache, v_cache, k_scale_inv, v_scale_inv)
    P, Hkv, page, D = k_cache.shape
    assert q.ndim == 3 and q.shape[2] == D, f"q must be [T, Hq, {D}], got {tuple(q.shape)}"
    assert q.dtype in _SIXTEEN, f"q must be bfloat16 or float16, got {q.dtype}"
    assert kind != _C.CACHE_16BIT or q.dtype == k_cache.dtype, "a 16-bit cache takes queries of its type"
    T, Hq = q.shape[0], q.shape[1]
    assert Hq > 0 and Hq % Hkv == 0, f"query heads ({Hq}) must be a multiple of cache heads ({Hkv})"
    assert seq_lens.ndim == 1 and seq_lens.dtype == torch.int32 and seq_lens.is_contiguous(), (
        "seq_lens must be contiguous one-dimensional int32"
    )
    B = seq_lens.shape[0]
    assert cu_seqlens_q.dtype == torch.int32 and cu_seqlens_q.shape == (B + 1,) and cu_seqlens_q.is_contiguous(), (
        f"cu_seqlens_q must be contiguous int32 [{B + 1}]"
    )
    assert page_table.ndim == 2 and page_table.dtype == torch.int32 and page_table.shape[0] == B, (
        f"page_table must be int32 [{B}, max_pages]"
    )
    assert page_table.shape[1] <= 1 or page_table.stride(1) == 1, "rows of page_table must be contiguous"
    assert T == 0 or B > 0, "tokens without a sequence"
    assert window_size is None or window_size > 0, f"window_size must be positive or None, got {window_size}"
    assert num_sinks >= 0, "num_sinks must not be negative"
    scale = D ** -0.5 if softmax_scale is None else float(softmax_scale)
    assert math.isfinite(scale), "softmax_scale must be finite"
    _check_devices(q, k_cache, v_cache, page_table, cu_seqlens_q, seq_lens, k_scale_inv, v_scale_inv)
    _no_grad("paged_attention", q)
    if q.stride(2) != 1 or q.stride(0) % 8 or q.stride(1) % 8 or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
    out = torch.empty((T, Hq, D), dtype=q.dtype, device=q.device)
    lse = torch.empty((T, Hq), dtype=torch.float32, device=q.device) if return_lse else None
    if T > 0:
        M = page_table.shape[1]
        # windows past the table's reach hide nothing
        win = 0 if window_size is None or window_size >= M * page else int(window_size)
        ws = _C.workspace(_C.query("pta_paged_attention_workspace_size", T, B, Hq, Hkv, D, M, page), q.device)
        _C.call(
            "pta_paged_attention", q.data_ptr(), _C.in_dtype_code(q.dtype), T, Hq, D, q.stride(0), q.stride(1),
            k_cache.data_ptr(), v_cache.data_ptr(), kind, P, page, Hkv, _C.ptr(k_scale_inv), _C.ptr(v_scale_inv),
            page_table.data_ptr(), page_table.stride(0), M, cu_seqlens_q.data_ptr(), seq_lens.data_ptr(), B, scale, win,
            min(int(num_sinks), M * page), out.data_ptr(), _C.ptr(lse), _C.ptr(ws), 0 if ws is None else ws.numel(),
            _C.stream(q.device),
        )
    return out, lse
