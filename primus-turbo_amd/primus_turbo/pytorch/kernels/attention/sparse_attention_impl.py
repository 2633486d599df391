"""Host side of the attention through selected pages: argument checks, output and
workspace allocation, the calls into libprimus_turbo_amd.so."""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from primus_turbo.pytorch import _C
from primus_turbo.pytorch.core.inference import check_tensors
from primus_turbo.pytorch.kernels.attention.kv_pages_impl import check_ranges
from primus_turbo.pytorch.kernels.attention.paged_attention_impl import _IN, _SIXTEEN, _check_cache, _increment_version


def _check_batch(page_table, cu_seqlens_q, seq_lens) -> Tuple[int, int, int]:
    """(sequences, pages of a row, stride of a row)"""
    i32 = torch.int32
    assert seq_lens.dim() == 1 and seq_lens.dtype == i32 and seq_lens.is_contiguous(), "seq_lens must be contiguous one-dimensional int32"
    B = seq_lens.shape[0]
    assert cu_seqlens_q.dtype == i32 and cu_seqlens_q.shape == (B + 1,) and cu_seqlens_q.is_contiguous(), (
        f"cu_seqlens_q must be contiguous int32 [{B + 1}]"
    )
    shape, stride = page_table.shape, page_table.stride()
    assert len(shape) == 2 and page_table.dtype == i32 and shape[0] == B, f"page_table must be int32 [{B}, max_pages]"
    assert shape[1] <= 1 or stride[1] == 1, "rows of page_table must be contiguous"
    return B, shape[1], stride[0]


def _check_choice(num_selected, num_first, num_last) -> Tuple[int, int, int]:
    take, first, last = int(num_selected), int(num_first), int(num_last)
    assert first >= 0 and last >= 1, f"num_first must not be negative and num_last at least 1, got {first}, {last}"
    assert take >= first + last, f"num_selected ({take}) must hold the first ({first}) and the last pages ({last})"
    return take, first, last


def _queries(q: torch.Tensor) -> torch.Tensor:
    qs = q.stride()
    return q.clone(memory_format=torch.contiguous_format) if qs[2] != 1 or qs[0] % 8 or qs[1] % 8 or q.data_ptr() % 16 else q


def kv_page_ranges_impl(k_cache, page_table, cu_seqlens_q, seq_lens, key_ranges, k_scale_inv) -> None:
    kind, (P, Hkv, page, D) = _check_cache(k_cache, k_cache, k_scale_inv, k_scale_inv)
    check_ranges(key_ranges, k_cache.shape)
    B, M, st = _check_batch(page_table, cu_seqlens_q, seq_lens)
    check_tensors("kv_page_ranges", (k_cache, key_ranges, k_scale_inv), page_table, cu_seqlens_q, seq_lens)
    if B == 0:
        return
    dev = k_cache.device
    _C.call_on(
        dev, "pta_kv_page_ranges", k_cache.data_ptr(), kind, k_cache.dtype == torch.float16, P, page, Hkv, D, _C.ptr(k_scale_inv),
        page_table.data_ptr(), st, M, cu_seqlens_q.data_ptr(), seq_lens.data_ptr(), B, key_ranges.data_ptr(), _C.stream(dev),
    )
    _increment_version((key_ranges,))


def select_pages_impl(
    q, key_ranges, page_table, cu_seqlens_q, seq_lens, page_size, num_selected, num_first, num_last
) -> Tuple[torch.Tensor, torch.Tensor]:
    shape = key_ranges.shape
    assert len(shape) == 4 and shape[2] == 2 and key_ranges.dtype == torch.bfloat16 and key_ranges.is_contiguous(), (
        f"key_ranges must be contiguous bfloat16 [num_pages, Hkv, 2, D], got {key_ranges.dtype} {tuple(shape)}"
    )
    P, Hkv, _, D = shape
    assert Hkv > 0 and D % 16 == 0 and 16 <= D <= 256, f"head_dim must be a multiple of 16 in [16, 256], got {D}"
    assert q.dim() == 3 and q.shape[2] == D, f"q must be [T, Hq, {D}], got {tuple(q.shape)}"
    assert q.dtype in _SIXTEEN, f"q must be bfloat16 or float16, got {q.dtype}"
    T, Hq, _ = q.shape
    assert Hq > 0 and Hq % Hkv == 0, f"query heads ({Hq}) must be a multiple of cache heads ({Hkv})"
    B, M, st = _check_batch(page_table, cu_seqlens_q, seq_lens)
    assert T == 0 or B > 0, "tokens without a sequence"
    page = int(page_size)
    assert page > 0, "page_size must not be 0"
    take, first, last = _check_choice(num_selected, num_first, num_last)
    check_tensors("select_pages", (q, key_ranges), page_table, cu_seqlens_q, seq_lens)
    q = _queries(q)
    dev = q.device
    sel = torch.empty((T, Hkv, min(take, M)), dtype=torch.int32, device=dev)
    lens = torch.empty((T,), dtype=torch.int32, device=dev)
    if T > 0:
        nbytes = _C.query_on(dev, "pta_select_pages_workspace_size", T, Hkv, M)
        ws = _C.workspace(nbytes, dev)
        _C.call_on(
            dev, "pta_select_pages", q.data_ptr(), _IN[q.dtype], T, Hq, D, q.stride(0), q.stride(1), key_ranges.data_ptr(), P, page,
            Hkv, page_table.data_ptr(), st, M, cu_seqlens_q.data_ptr(), seq_lens.data_ptr(), B, take, first, last, sel.data_ptr(),
            lens.data_ptr(), _C.ptr(ws), nbytes, _C.stream(dev),
        )
    return sel, lens


def sparse_paged_attention_impl(
    q, k_cache, v_cache, key_ranges, page_table, cu_seqlens_q, seq_lens, k_scale_inv, v_scale_inv, num_selected, num_first, num_last,
    softmax_scale, return_lse,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    kind, (P, Hkv, page, D) = _check_cache(k_cache, v_cache, k_scale_inv, v_scale_inv)
    check_ranges(key_ranges, k_cache.shape)
    shape, dtype = q.shape, q.dtype
    assert len(shape) == 3 and shape[2] == D, f"q must be [T, Hq, {D}], got {tuple(shape)}"
    assert dtype in _SIXTEEN, f"q must be bfloat16 or float16, got {dtype}"
    fp8 = kind != _C.CACHE_16BIT
    assert fp8 or dtype == k_cache.dtype, "a 16-bit cache takes queries of its type"
    T, Hq, _ = shape
    assert Hq > 0 and Hq % Hkv == 0, f"query heads ({Hq}) must be a multiple of cache heads ({Hkv})"
    B, M, st = _check_batch(page_table, cu_seqlens_q, seq_lens)
    assert T == 0 or B > 0, "tokens without a sequence"
    take, first, last = _check_choice(num_selected, num_first, num_last)
    if softmax_scale is None:
        scale = D ** -0.5
    else:
        scale = float(softmax_scale)
        assert scale > 0.0 and math.isfinite(scale), "softmax_scale must be positive and finite"
    check_tensors("sparse_paged_attention", (q, k_cache, v_cache, k_scale_inv, v_scale_inv, key_ranges), page_table, cu_seqlens_q, seq_lens)
    q = _queries(q)
    dev = q.device
    out = torch.empty(shape, dtype=dtype, device=dev)
    lse = torch.empty((T, Hq), dtype=torch.float32, device=dev) if return_lse else None
    if T > 0:
        nbytes = _C.query_on(dev, "pta_sparse_paged_attention_workspace_size", T, B, Hq, Hkv, D, M, page, take)
        ws = _C.workspace(nbytes, dev)
        qs = q.stride()
        _C.call_on(
            dev, "pta_sparse_paged_attention", q.data_ptr(), _IN[dtype], T, Hq, D, qs[0], qs[1], k_cache.data_ptr(), v_cache.data_ptr(),
            kind, P, page, Hkv, k_scale_inv.data_ptr() if fp8 else None, v_scale_inv.data_ptr() if fp8 else None,
            key_ranges.data_ptr(), page_table.data_ptr(), st, M, cu_seqlens_q.data_ptr(), seq_lens.data_ptr(), B, take, first, last,
            scale, out.data_ptr(), None if lse is None else lse.data_ptr(), _C.ptr(ws), nbytes, _C.stream(dev),
        )
    return out, lse
