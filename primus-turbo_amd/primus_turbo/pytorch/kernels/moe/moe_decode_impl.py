"""Host side of the few-token expert kernels: argument checks, output and
workspace allocation, the call into libprimus_turbo_amd.so."""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from primus_turbo.pytorch import _C
from primus_turbo.pytorch.core.low_precision import ScalingGranularity, float8_e4m3, float8_e5m2
from primus_turbo.pytorch.core.quantized_tensor import QuantizedTensor


def _weight(w, scale, name: str) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(data, scale_inv) of a weight given as a QuantizedTensor or as its parts."""
    if not isinstance(w, QuantizedTensor):
        return w, scale
    assert scale is None, f"{name} is a QuantizedTensor: it brings its scale_inv"
    g = w.granularity
    assert g != ScalingGranularity.MX_BLOCKWISE, "moe_decode: MX_BLOCKWISE weights are not supported"
    if g == ScalingGranularity.ROWWISE:
        assert w.quantized_axis == 2, f"{name} must be quantized along its last axis"
    if g == ScalingGranularity.BLOCKWISE:
        assert w.block_size == 128 and w.scaling_recipe is not None and w.scaling_recipe.use_2d_block, (
            f"{name} must have 128 x 128 blocks"
        )
    return w.qdata, w.scale_inv


def _granularity(w, scale, name: str) -> int:
    """0 for a 16-bit weight, else the granularity that the scale's shape says."""
    if scale is None:
        return 0
    E, N, K = w.shape
    assert scale.dtype == torch.float32 and scale.is_contiguous(), f"{name}'s scale_inv must be contiguous float32"
    if scale.numel() == 1 and scale.ndim <= 1:
        return _C.PTA_TENSORWISE
    if tuple(scale.shape) == (E, N, 1):
        return _C.PTA_ROWWISE
    assert tuple(scale.shape) == (E, -(-N // 128), -(-K // 128)), (
        f"{name}'s scale_inv must be one value, {(E, N, 1)} or {(E, -(-N // 128), -(-K // 128))}, got {tuple(scale.shape)}"
    )
    return _C.PTA_BLOCKWISE


def moe_decode_impl(x, w_gate_up, w_down, topk_idx, topk_probs, gate_up_scale_inv, down_scale_inv) -> torch.Tensor:
    w1, s1 = _weight(w_gate_up, gate_up_scale_inv, "w_gate_up")
    w2, s2 = _weight(w_down, down_scale_inv, "w_down")
    assert x.ndim == 2 and x.dtype in (torch.bfloat16, torch.float16), "x must be [T, H] bfloat16 or float16"
    assert w1.ndim == 3 and w2.ndim == 3, "expert weights must be 3-dimensional"
    T, H = x.shape
    E, I = w2.shape[0], w2.shape[2]
    assert w1.shape == (E, 2 * I, H) and w2.shape[1] == H, (
        f"weights must be [E, 2 I, {H}] and [E, {H}, I], got {tuple(w1.shape)} and {tuple(w2.shape)}"
    )
    assert w1.dtype == w2.dtype and (s1 is None) == (s2 is None), "both weights must be of one kind"
    assert w1.is_contiguous() and w2.is_contiguous(), "expert weights must be contiguous"
    assert 0 < E <= 1024, f"1 to 1024 experts, got {E}"
    assert H > 0 and I > 0 and H % 16 == 0 and I % 16 == 0, f"H and I must be multiples of 16, got {H}, {I}"
    if s1 is None:
        assert w1.dtype == x.dtype, f"weights must be of x's type or fp8 with scale_inv, got {w1.dtype}"
        kind = _C.CACHE_16BIT
    else:
        assert w1.dtype in (float8_e4m3, float8_e5m2), f"scaled weights must be fp8, got {w1.dtype}"
        kind = _C.fp8_code(w1.dtype)
    gran = _granularity(w1, s1, "w_gate_up")
    assert gran == _granularity(w2, s2, "w_down"), "both weights must have one granularity"
    assert topk_idx.ndim == 2 and topk_idx.shape[0] == T and topk_idx.dtype in (torch.int32, torch.int64), (
        f"topk_idx must be [{T}, k] int32 or int64"
    )
    k = topk_idx.shape[1]
    assert 0 < k <= 32, f"1 to 32 experts a token, got {k}"
    assert topk_probs.shape == topk_idx.shape and topk_probs.dtype == torch.float32, "topk_probs must be float32 like topk_idx"
    dev = x.device
    assert all(t is None or t.device == dev for t in (w1, w2, s1, s2, topk_idx, topk_probs)), f"all tensors must be on {dev}"
    assert not (torch.is_grad_enabled() and (x.requires_grad or topk_probs.requires_grad)), (
        "moe_decode has no backward pass: call it under torch.no_grad() or on detached tensors"
    )
    y = torch.empty((T, H), dtype=x.dtype, device=dev)
    if T == 0:
        return y
    if x.stride(1) != 1 or x.stride(0) % 8 or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
    topk_idx, topk_probs = topk_idx.contiguous(), topk_probs.contiguous()
    ws = _C.workspace(_C.query("pta_moe_decode_workspace_size", T, E, k, I), dev)
    _C.call(
        "pta_moe_decode", x.data_ptr(), _C.in_dtype_code(x.dtype), T, H, x.stride(0), w1.data_ptr(), w2.data_ptr(), kind,
        _C.ptr(s1), _C.ptr(s2), gran, E, I, topk_idx.data_ptr(), int(topk_idx.dtype == torch.int64),
        topk_probs.data_ptr(), k, y.data_ptr(), ws.data_ptr(), ws.numel(), _C.stream(dev),
    )
    return y
