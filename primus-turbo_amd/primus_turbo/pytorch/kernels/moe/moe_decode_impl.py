"""Host side of the few-token expert kernels: argument checks, output and
workspace allocation, the call into libprimus_turbo_amd.so."""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from primus_turbo.pytorch import _C
from primus_turbo.pytorch.core.inference import check_tensors, refuse_gradients
from primus_turbo.pytorch.core.low_precision import ScalingGranularity, float8_e4m3, float8_e5m2
from primus_turbo.pytorch.core.quantized_tensor import QuantizedTensor


_X = {torch.bfloat16: _C.PTA_BF16, torch.float16: _C.PTA_F16}


def _weight(w, scale, name: str) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(data, scale_inv) of a weight given as a QuantizedTensor or as its parts."""
    if not isinstance(w, QuantizedTensor):
        return w, scale
    assert scale is None, f"{name} is a QuantizedTensor: it brings its scale_inv"
    if w.requires_grad:
        refuse_gradients("moe_decode", w)
    g = w.granularity
    assert g != ScalingGranularity.MX_BLOCKWISE, "moe_decode: MX_BLOCKWISE weights are not supported"
    if g == ScalingGranularity.ROWWISE:
        assert w.quantized_axis == 2, f"{name} must be quantized along its last axis"
    if g == ScalingGranularity.BLOCKWISE:
        assert w.block_size == 128 and w.scaling_recipe is not None and w.scaling_recipe.use_2d_block, (
            f"{name} must have 128 x 128 blocks"
        )
    return w.qdata, w.scale_inv


def _granularity(scale, E: int, N: int, K: int, name: str) -> int:
    """The granularity that the shape of the scale of an [E, N, K] weight says."""
    shape = scale.shape
    assert scale.dtype == torch.float32 and scale.is_contiguous(), f"{name}'s scale_inv must be contiguous float32"
    if len(shape) <= 1 and scale.numel() == 1:
        return _C.PTA_TENSORWISE
    if shape == (E, N, 1):
        return _C.PTA_ROWWISE
    assert shape == (E, -(-N // 128), -(-K // 128)), (
        f"{name}'s scale_inv must be one value, {(E, N, 1)} or {(E, -(-N // 128), -(-K // 128))}, got {tuple(shape)}"
    )
    return _C.PTA_BLOCKWISE


def moe_decode_impl(x, w_gate_up, w_down, topk_idx, topk_probs, gate_up_scale_inv, down_scale_inv) -> torch.Tensor:
    w1, s1 = _weight(w_gate_up, gate_up_scale_inv, "w_gate_up")
    w2, s2 = _weight(w_down, down_scale_inv, "w_down")
    xshape, dtype = x.shape, x.dtype
    assert len(xshape) == 2 and dtype in _X, "x must be [T, H] bfloat16 or float16"
    shape1, shape2 = w1.shape, w2.shape
    assert len(shape1) == 3 and len(shape2) == 3, "expert weights must be 3-dimensional"
    T, H = xshape
    E, _, I = shape2
    assert shape1 == (E, 2 * I, H) and shape2[1] == H, (
        f"weights must be [E, 2 I, {H}] and [E, {H}, I], got {tuple(shape1)} and {tuple(shape2)}"
    )
    wtype = w1.dtype
    assert w2.dtype == wtype and (s1 is None) == (s2 is None), "both weights must be of one kind"
    assert w1.is_contiguous() and w2.is_contiguous(), "expert weights must be contiguous"
    assert 0 < E <= 1024, f"1 to 1024 experts, got {E}"
    assert H > 0 and I > 0 and H % 16 == 0 and I % 16 == 0, f"H and I must be multiples of 16, got {H}, {I}"
    if s1 is None:
        assert wtype == dtype, f"weights must be of x's type or fp8 with scale_inv, got {wtype}"
        kind, gran = _C.CACHE_16BIT, 0
    else:
        assert wtype in (float8_e4m3, float8_e5m2), f"scaled weights must be fp8, got {wtype}"
        kind = _C.fp8_code(wtype)
        gran = _granularity(s1, E, 2 * I, H, "w_gate_up")
        assert gran == _granularity(s2, E, H, I, "w_down"), "both weights must have one granularity"
    idx_shape, idx_type = topk_idx.shape, topk_idx.dtype
    assert len(idx_shape) == 2 and idx_shape[0] == T and idx_type in (torch.int64, torch.int32), (
        f"topk_idx must be [{T}, k] int32 or int64"
    )
    k = idx_shape[1]
    assert 0 < k <= 32, f"1 to 32 experts a token, got {k}"
    assert topk_probs.shape == idx_shape and topk_probs.dtype == torch.float32, "topk_probs must be float32 like topk_idx"
    check_tensors("moe_decode", (x, topk_probs, w1, w2, s1, s2), topk_idx)
    dev = x.device
    y = torch.empty(xshape, dtype=dtype, device=dev)
    if T == 0:
        return y
    xs = x.stride()
    if xs[1] != 1 or xs[0] % 8 or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
        xs = x.stride()
    if not topk_idx.is_contiguous():
        topk_idx = topk_idx.contiguous()
    if not topk_probs.is_contiguous():
        topk_probs = topk_probs.contiguous()
    nbytes = _C.query("pta_moe_decode_workspace_size", T, E, k, I)
    ws = _C.workspace(nbytes, dev)
    _C.call(
        "pta_moe_decode", x.data_ptr(), _X[dtype], T, H, xs[0], w1.data_ptr(), w2.data_ptr(), kind,
        None if s1 is None else s1.data_ptr(), None if s2 is None else s2.data_ptr(), gran, E, I, topk_idx.data_ptr(),
        idx_type == torch.int64, topk_probs.data_ptr(), k, y.data_ptr(), ws.data_ptr(), nbytes, _C.stream(dev),
    )
    return y
