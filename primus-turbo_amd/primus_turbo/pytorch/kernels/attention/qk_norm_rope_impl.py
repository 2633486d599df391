"""Host side of the norms and rotation of queries and keys: argument checks,
output and workspace allocation, the calls into libprimus_turbo_amd.so."""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
from torch._subclasses.fake_tensor import FakeTensor

from primus_turbo.pytorch import _C
from primus_turbo.pytorch.core.inference import check_tensors
from primus_turbo.pytorch.kernels.attention.paged_attention_impl import _IN, _check_cache, _check_slots, _increment_version

_INT, _F32, _DENSE = (torch.int32, torch.int64), torch.float32, torch.contiguous_format


def _check_rotation(cos, sin, positions, lead, D) -> int:
    """Rotated elements of a head."""
    shape = cos.shape
    assert len(shape) == 2 and sin.shape == shape, f"cos and sin must be [positions, rot_dim / 2], both alike: got {tuple(shape)}, {tuple(sin.shape)}"
    assert cos.dtype == _F32 and sin.dtype == _F32 and cos.is_contiguous() and sin.is_contiguous(), "cos and sin must be contiguous float32"
    rot = 2 * shape[1]
    assert 2 <= rot <= D, f"cos and sin turn {rot} elements of a head of {D}"
    assert positions.dtype in _INT and positions.shape == lead, f"positions must be int32 / int64 {tuple(lead)}, got {positions.dtype} {tuple(positions.shape)}"
    return rot


def _check_weight(w: Optional[torch.Tensor], D: int) -> int:
    """Type code."""
    if w is None:
        return 0
    assert w.shape == (D,) and w.is_contiguous(), f"a weight must be contiguous [{D}], got {tuple(w.shape)}"
    dt = _IN.get(w.dtype)
    if dt is None:
        raise TypeError(f"unsupported weight type {w.dtype}")
    return dt


def _check_eps(eps) -> float:
    eps = float(eps)
    assert eps >= 0.0 and math.isfinite(eps), f"eps must be finite and not negative, got {eps}"
    return eps


def _rows(x: torch.Tensor) -> torch.Tensor:
    """[..., H, D] as [T, H, D], in place where the strides allow; D contiguous."""
    if x.dim() != 3:
        x = x.reshape(x.shape[:-2].numel(), *x.shape[-2:])
    return x if x.stride(2) == 1 else x.contiguous()


def check_qk(q, k, cos, sin, positions, q_weight, k_weight, eps) -> float:
    """eps, after checking all that both directions take."""
    shape, kshape, dtype = q.shape, k.shape, q.dtype
    if dtype not in _IN:
        raise TypeError(f"unsupported type of queries and keys {dtype}")
    assert k.dtype == dtype, "q and k must have one type"
    lead = shape[:-2]
    assert len(shape) >= 2 and len(kshape) == len(shape) and lead == kshape[:-2] and shape[-1] == kshape[-1], (
        f"q and k must be [..., heads, D] with the same tokens and D, got {tuple(shape)}, {tuple(kshape)}"
    )
    D = shape[-1]
    assert D % 2 == 0 and 2 <= D <= 256, f"head_dim must be even and at most 256, got {D}"
    _check_rotation(cos, sin, positions, lead, D)
    _check_weight(q_weight, D)
    _check_weight(k_weight, D)
    eps = _check_eps(eps)
    assert not cos.requires_grad and not sin.requires_grad, "cos and sin get no gradients"
    # one is enough: they do not go together with tensors that have memory
    assert not isinstance(q, FakeTensor), "qk_norm_rope runs on memory: fake tensors have none"
    dev = q.get_device()
    for t in (k, cos, sin, positions, q_weight, k_weight):
        assert t is None or (t.get_device() == dev and t.device == q.device), f"all tensors must be on {q.device}"
    assert dev >= 0 or not torch.cuda.is_available(), f"all tensors must be GPU tensors, got {q.device}"
    return eps


def qk_norm_rope_impl(q, k, cos, sin, positions, q_weight, k_weight, eps, interleaved) -> Tuple[torch.Tensor, torch.Tensor]:
    """Arguments as check_qk has passed them."""
    dtype, dev = q.dtype, q.device
    q_out, k_out = torch.empty_like(q, memory_format=_DENSE), torch.empty_like(k, memory_format=_DENSE)
    q, k = _rows(q), _rows(k)
    if not positions.is_contiguous():
        positions = positions.contiguous()
    (T, Hq, D), Hkv, (P, half) = q.shape, k.shape[1], cos.shape
    qs, ks = q.stride(), k.stride()
    _C.call_on(
        dev, "pta_qk_norm_rope", q.data_ptr(), k.data_ptr(), _IN[dtype], T, Hq, Hkv, D, qs[0], qs[1], ks[0], ks[1], cos.data_ptr(),
        sin.data_ptr(), P, 2 * half, positions.data_ptr(), positions.dtype == torch.int64,
        None if q_weight is None else q_weight.data_ptr(), 0 if q_weight is None else _IN[q_weight.dtype],
        None if k_weight is None else k_weight.data_ptr(), 0 if k_weight is None else _IN[k_weight.dtype], eps, interleaved,
        q_out.data_ptr(), k_out.data_ptr(), _C.stream(dev),
    )
    return q_out, k_out


_NONE = None, 0, (0, 0), None, (0, 0), None, None, None, 0


def _side(g, x, w, want):
    """What the backward pass takes of the queries or of the keys."""
    if g is None:
        return _NONE
    dx = torch.empty_like(g, memory_format=_DENSE)
    g = _rows(g)
    if w is None:
        return g, g.shape[1], g.stride(), None, (0, 0), dx, None, None, 0
    x = _rows(x)
    return g, g.shape[1], g.stride(), x, x.stride(), dx, torch.empty_like(w) if want else None, w.data_ptr(), _IN[w.dtype]


def qk_norm_rope_backward_impl(
    gq: Optional[torch.Tensor], gk: Optional[torch.Tensor], q, k, cos, sin, positions, q_weight, k_weight, eps, interleaved, want_qw, want_kw
):
    """Gradients of (q, k, q_weight, k_weight); None for gq or gk leaves that side out.
    q and k may be None where they have no weight."""
    like = gk if gq is None else gq
    dev, dtype, D = like.device, like.dtype, like.shape[-1]
    if not positions.is_contiguous():
        positions = positions.contiguous()
    gq, Hq, gqs, q, qs, dq, dqw, qw, qwd = _side(gq, q, q_weight, want_qw)
    gk, Hkv, gks, k, ks, dk, dkw, kw, kwd = _side(gk, k, k_weight, want_kw)
    T, (P, half) = positions.numel(), cos.shape
    nbytes = _C.query_on(dev, "pta_qk_norm_rope_backward_workspace_size", T, Hq, Hkv, D) if want_qw or want_kw else 0
    ws, ptr = _C.workspace(nbytes, dev), _C.ptr
    _C.call_on(
        dev, "pta_qk_norm_rope_backward", ptr(gq), ptr(gk), gqs[0], gqs[1], gks[0], gks[1], ptr(q), ptr(k),
        _IN[dtype], T, Hq, Hkv, D, qs[0], qs[1], ks[0], ks[1], cos.data_ptr(), sin.data_ptr(), P, 2 * half,
        positions.data_ptr(), positions.dtype == torch.int64, qw, qwd, kw, kwd, eps, interleaved, ptr(dq), ptr(dk),
        ptr(dqw), ptr(dkw), ptr(ws), nbytes, _C.stream(dev),
    )
    return dq, dk, dqw, dkw


def qk_norm_rope_cache_write_impl(
    q, k, v, cos, sin, positions, k_cache, v_cache, slots, k_scale_inv, v_scale_inv, q_weight, k_weight, eps, interleaved
) -> torch.Tensor:
    kind, (P, Hkv, page, D) = _check_cache(k_cache, v_cache, k_scale_inv, v_scale_inv)
    shape, kshape, dtype = q.shape, k.shape, q.dtype
    assert len(shape) == 3 and shape[2] == D, f"q must be [T, Hq, {D}], got {tuple(shape)}"
    T, Hq, _ = shape
    assert kshape == (T, Hkv, D) and v.shape == kshape, f"k and v must be [{T}, {Hkv}, {D}], got {tuple(kshape)}, {tuple(v.shape)}"
    assert dtype in (torch.bfloat16, torch.float16), f"q, k and v must be bfloat16 or float16, got {dtype}"
    assert k.dtype == dtype and v.dtype == dtype, "q, k and v must have one type"
    fp8 = kind != _C.CACHE_16BIT
    assert fp8 or dtype == k_cache.dtype, "a 16-bit cache takes keys and values of its type"
    n = _check_slots(slots)
    assert n == T, f"one slot for each of the {T} tokens, got {n}"
    rot = _check_rotation(cos, sin, positions, shape[:1], D)
    assert positions.is_contiguous(), "positions must be contiguous"
    qwd, kwd = _check_weight(q_weight, D), _check_weight(k_weight, D)
    eps = _check_eps(eps)
    check_tensors("qk_norm_rope_cache_write", (q, k, v, cos, sin, k_cache, v_cache, k_scale_inv, v_scale_inv, q_weight, k_weight),
                  slots, positions)
    dev = q.device
    out = torch.empty_like(q, memory_format=_DENSE)
    if T == 0:
        return out
    qs, ks, vs = q.stride(), k.stride(), v.stride()
    if qs[2] != 1 or ks[2] != 1 or vs[2] != 1:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
        qs, ks, vs = q.stride(), k.stride(), v.stride()
    _C.call_on(
        dev, "pta_qk_norm_rope_cache_write", q.data_ptr(), k.data_ptr(), v.data_ptr(), _IN[dtype], T, Hq, Hkv, D, qs[0], qs[1],
        ks[0], ks[1], vs[0], vs[1], cos.data_ptr(), sin.data_ptr(), cos.shape[0], rot, positions.data_ptr(),
        positions.dtype == torch.int64, None if q_weight is None else q_weight.data_ptr(), qwd,
        None if k_weight is None else k_weight.data_ptr(), kwd, eps, bool(interleaved), slots.data_ptr(), slots.dtype == torch.int64,
        k_cache.data_ptr(), v_cache.data_ptr(), kind, P, page, k_scale_inv.data_ptr() if fp8 else None,
        v_scale_inv.data_ptr() if fp8 else None, out.data_ptr(), _C.stream(dev),
    )
    _increment_version((k_cache, v_cache, k_scale_inv, v_scale_inv) if fp8 else (k_cache, v_cache))
    return out
