"""Host side of the operators on whole pages of a paged cache: argument checks,
output and workspace allocation, the calls into libprimus_turbo_amd.so."""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from primus_turbo.pytorch import _C
from primus_turbo.pytorch.core.inference import check_tensors
from primus_turbo.pytorch.kernels.attention.paged_attention_impl import _KIND, _check_cache, _increment_version

_INT = (torch.int32, torch.int64)


def check_ranges(key_ranges: torch.Tensor, shape: torch.Size) -> None:
    """Ranges of the keys of a pool of the given shape."""
    want = (*shape[:-2], 2, shape[-1])
    assert key_ranges.shape == want and key_ranges.dtype == torch.bfloat16 and key_ranges.is_contiguous(), (
        f"key_ranges must be contiguous bfloat16 {want}, got {key_ranges.dtype} {tuple(key_ranges.shape)}"
    )


def _check_pools(k_cache, v_cache, k_scale_inv, v_scale_inv, key_ranges):
    """(kind, layers, pages, heads, page size, D, the tensors) of pools with or without a dimension of layers."""
    shape = k_cache.shape
    if len(shape) == 4:
        kind, (P, Hkv, page, D) = _check_cache(k_cache, v_cache, k_scale_inv, v_scale_inv)
        L = 1
    else:
        dtype = k_cache.dtype
        assert len(shape) == 5 and v_cache.shape == shape, (
            f"caches must be [(layers,) num_pages, Hkv, page_size, D], both alike: got {tuple(shape)}, {tuple(v_cache.shape)}"
        )
        assert v_cache.dtype == dtype, "k_cache and v_cache must have one type"
        kind = _KIND.get(dtype)
        assert kind is not None, f"unsupported cache type {dtype}"
        assert k_cache.is_contiguous() and v_cache.is_contiguous(), "caches must be contiguous"
        L, P, Hkv, page, D = shape
        assert D % 16 == 0 and 16 <= D <= 256, f"head_dim must be a multiple of 16 in [16, 256], got {D}"
        assert page > 0 and Hkv > 0, "page_size and the number of heads must not be 0"
        if kind == _C.CACHE_16BIT:
            assert k_scale_inv is None and v_scale_inv is None, "a 16-bit cache has no scales"
        else:
            assert k_scale_inv is not None and v_scale_inv is not None, "an fp8 cache needs k_scale_inv and v_scale_inv"
            want = shape[:4]
            for s in (k_scale_inv, v_scale_inv):
                assert s.shape == want and s.dtype == torch.float32 and s.is_contiguous(), (
                    f"scale_inv must be contiguous float32 {tuple(want)}, got {s.dtype} {tuple(s.shape)}"
                )
    tensors = (k_cache, v_cache) if k_scale_inv is None else (k_cache, v_cache, k_scale_inv, v_scale_inv)
    if key_ranges is not None:
        check_ranges(key_ranges, shape)
        tensors += (key_ranges,)
    return kind, L, P, Hkv, page, D, tensors


def kv_cache_copy_impl(k_cache, v_cache, src_pages, dst_pages, k_scale_inv, v_scale_inv, key_ranges) -> None:
    kind, L, P, Hkv, page, D, tensors = _check_pools(k_cache, v_cache, k_scale_inv, v_scale_inv, key_ranges)
    shape, dtype = src_pages.shape, src_pages.dtype
    assert len(shape) == 1 and dtype in _INT and dst_pages.shape == shape and dst_pages.dtype == dtype, (
        "src_pages and dst_pages must be one-dimensional int32 / int64 of one type and length"
    )
    assert src_pages.is_contiguous() and dst_pages.is_contiguous(), "src_pages and dst_pages must be contiguous"
    check_tensors("kv_cache_copy", tensors, src_pages, dst_pages)
    if shape[0] == 0 or L == 0:
        return
    dev = k_cache.device
    _C.call_on(
        dev, "pta_kv_cache_copy", k_cache.data_ptr(), v_cache.data_ptr(), kind, L, P, Hkv, page, D, _C.ptr(k_scale_inv),
        _C.ptr(v_scale_inv), _C.ptr(key_ranges), src_pages.data_ptr(), dst_pages.data_ptr(), dtype == torch.int64, shape[0],
        _C.stream(dev),
    )
    _increment_version(tensors)


def kv_cache_fork_impl(
    k_cache, v_cache, page_table, seq_lens, parents: Optional[torch.Tensor], k_scale_inv, v_scale_inv, key_ranges, reserve, compact
) -> Tuple[torch.Tensor, torch.Tensor]:
    kind, L, P, Hkv, page, D, tensors = _check_pools(k_cache, v_cache, k_scale_inv, v_scale_inv, key_ranges)
    i32 = torch.int32
    assert seq_lens.dim() == 1 and seq_lens.dtype == i32 and seq_lens.is_contiguous(), "seq_lens must be contiguous one-dimensional int32"
    B = seq_lens.shape[0]
    assert page_table.dim() == 2 and page_table.dtype == i32 and page_table.shape[0] == B, f"page_table must be int32 [{B}, max_pages]"
    M = page_table.shape[1]
    assert M <= 1 or page_table.stride(1) == 1, "rows of page_table must be contiguous"
    others = [page_table, seq_lens]
    N = B
    if parents is not None:
        assert parents.dim() == 1 and parents.dtype in _INT and parents.is_contiguous(), "parents must be contiguous one-dimensional int32 / int64"
        N = parents.shape[0]
        others.append(parents)
    reserve = min(int(reserve), 2**31 - 1)  # more than any length
    assert reserve >= 0, "reserve must not be negative"
    check_tensors("kv_cache_fork", tensors, *others)
    dev = k_cache.device
    table = torch.empty((N, M), dtype=i32, device=dev)
    lens = torch.empty((N,), dtype=i32, device=dev)
    if N == 0:
        return table, lens
    nbytes = _C.query_on(dev, "pta_kv_cache_fork_workspace_size", N, M, P, bool(compact))
    ws = _C.workspace(nbytes, dev)
    _C.call_on(
        dev, "pta_kv_cache_fork", k_cache.data_ptr(), v_cache.data_ptr(), kind, L, P, Hkv, page, D, _C.ptr(k_scale_inv),
        _C.ptr(v_scale_inv), _C.ptr(key_ranges), page_table.data_ptr(), page_table.stride(0), M, seq_lens.data_ptr(), B,
        _C.ptr(parents), parents is not None and parents.dtype == torch.int64, N, reserve, bool(compact), table.data_ptr(),
        lens.data_ptr(), _C.ptr(ws), nbytes, _C.stream(dev),
    )
    _increment_version(tensors)
    return table, lens
