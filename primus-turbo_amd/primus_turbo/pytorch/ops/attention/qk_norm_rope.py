"""Norms of queries and keys for each head and the rotation by their positions,
in one pass, with a backward pass; and the same for new tokens whose keys and
values go straight into a paged cache (no reference counterpart: there the norms
and the rotation are separate operators).

For a row x, the D elements of one token and head:

  n = x * (mean(x^2) + eps)^(-1/2) * weight     without a weight: n = x
  y = n, the pairs (a, b) of its first R elements turned by the token's angles:
      (a cos - b sin, a sin + b cos)

``cos`` and ``sin`` are [positions, R / 2] float32 tables, whose row p has the
angles of position p (scaled in whatever way the model asks for); R, even, is D or
less.  Pairs are (i, i + R / 2), with ``interleaved`` (2 i, 2 i + 1).  A token whose
position lies outside the tables, -1 for padding, gets zeros and gives no gradient.
Everything is fp32 up to the one rounding of the result, the sums of squares too: a row
whose squares leave its range becomes zeros (elements beyond about 1e18) or, where eps is
0, inaccurate and at last infinite (all below about 1e-19).  Elements beyond the first R
depend on the others through the norm alone.  Under torch.compile the calls run between
its graphs; fake tensors are refused.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from primus_turbo.pytorch.kernels.attention.qk_norm_rope_impl import (
    check_qk,
    qk_norm_rope_backward_impl,
    qk_norm_rope_cache_write_impl,
    qk_norm_rope_impl,
)

__all__ = ["qk_norm_rope", "qk_norm_rope_cache_write"]


def _backward(ctx, gq, gk):
    q, k, cos, sin, positions, q_weight, k_weight = ctx.saved_tensors
    need_q, need_k, _, _, _, need_qw, need_kw, _, _ = ctx.needs_input_grad
    eps, interleaved = ctx.how
    dq, dk, dqw, dkw = qk_norm_rope_backward_impl(gq if need_q or need_qw else None, gk if need_k or need_kw else None, q, k, cos, sin,
                                                  positions, q_weight, k_weight, eps, interleaved, need_qw, need_kw)
    return dq if need_q else None, dk if need_k else None, None, None, None, dqw, dkw, None, None


_backward_once = once_differentiable(_backward)


class _QKNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, cos, sin, positions, q_weight, k_weight, eps, interleaved):
        # the rotation alone needs nothing of its inputs
        ctx.save_for_backward(None if q_weight is None else q, None if k_weight is None else k, cos, sin, positions, q_weight, k_weight)
        ctx.how = eps, interleaved
        return qk_norm_rope_impl(q, k, cos, sin, positions, q_weight, k_weight, eps, interleaved)

    @staticmethod
    def backward(ctx, gq, gk):
        # with gradients enabled (create_graph) a second derivative has to fail, not to be missing
        return (_backward_once if torch.is_grad_enabled() else _backward)(ctx, gq, gk)


@torch._dynamo.disable
def qk_norm_rope(
    q: torch.Tensor,
    k: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    positions: torch.Tensor,
    q_weight: Optional[torch.Tensor] = None,
    k_weight: Optional[torch.Tensor] = None,
    *,
    eps: float = 1e-6,
    interleaved: bool = False,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Normed and rotated (q, k), of the inputs' shapes and type, contiguous.

    ``q``: [..., Hq, D], ``k``: [..., Hkv, D], bfloat16, float16 or float32; they may be
    parts of a projection's output.  D is even and at most 256.  ``positions``: [...]
    int32 / int64.  ``q_weight``, ``k_weight``: [D] of any of these types, or None for
    no norm.  Gradients go to q, k and the weights; the weights' are summed over all
    tokens and heads in fp32, in a fixed order.  There is no second derivative.
    """
    eps = check_qk(q, k, cos, sin, positions, q_weight, k_weight, eps)
    return _QKNormRope.apply(q, k, cos, sin, positions, q_weight, k_weight, eps, bool(interleaved))


@torch._dynamo.disable
def qk_norm_rope_cache_write(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    positions: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    slots: torch.Tensor,
    k_scale_inv: Optional[torch.Tensor] = None,
    v_scale_inv: Optional[torch.Tensor] = None,
    *,
    q_weight: Optional[torch.Tensor] = None,
    k_weight: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    interleaved: bool = False,
) -> torch.Tensor:
    """``qk_norm_rope`` of new tokens, whose keys and values go into their cache slots as
    ``kv_cache_write`` puts them there, in one launch; returns the queries.

    ``q``: [T, Hq, D], ``k``, ``v``: [T, Hkv, D], bfloat16 or float16.  Caches, scales and
    ``slots`` are ``kv_cache_write``'s (a token without a slot gets its query all the
    same); an fp8 row is quantized from the fp32 key, so it may differ by a rounding from
    the one that the two calls would write.  Inference only.
    """
    return qk_norm_rope_cache_write_impl(q, k, v, cos, sin, positions, k_cache, v_cache, slots, k_scale_inv, v_scale_inv, q_weight,
                                         k_weight, eps, interleaved)
