"""Paged key / value cache and the attention of new tokens over it, for
inference (no reference counterpart: the reference's attention is for training).

A cache is four tensors that the caller allocates and keeps:

  k_cache, v_cache          [num_pages, Hkv, page_size, D], float8_e4m3fn or
                            float8_e5m2, or the model's 16-bit type
  k_scale_inv, v_scale_inv  [num_pages, Hkv, page_size] float32 for fp8, else None

D is a multiple of 16 up to 256; page_size is free.  A slot, page * page_size +
offset, names the place of one token.  Lengths, slots and page tables stay on
the device; nothing here synchronizes, so the calls can be captured in a HIP
graph and replayed with new lengths, slots and pages written in place.  Under
torch.compile they run between its graphs (fullgraph=True, export and fake
tensors are refused).  A tensor that needs gradients is refused outside
torch.no_grad(), caches and scales too.
"""

from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from primus_turbo.pytorch.kernels.attention.paged_attention_impl import (
    kv_cache_read_impl,
    kv_cache_write_impl,
    paged_attention_impl,
)

__all__ = ["kv_cache_write", "kv_cache_read", "paged_attention"]


@torch._dynamo.disable
def kv_cache_write(
    k: torch.Tensor,
    v: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    slots: torch.Tensor,
    k_scale_inv: Optional[torch.Tensor] = None,
    v_scale_inv: Optional[torch.Tensor] = None,
) -> None:
    """Write the keys and values of new tokens, [T, Hkv, D], into their cache slots, in place.

    ``slots``: [T] int32 / int64; a token whose slot is below 0 or past the pool
    is skipped (padding), and no slot may be named twice.  An fp8 cache gets each
    (token, head) row quantized as ``quantize_fp8(..., ScalingGranularity.ROWWISE,
    axis=-1)`` does, byte for byte, with its ``scale_inv``; a 16-bit cache gets
    copies.  ``k`` and ``v`` may be slices of a larger tensor (their last dimension
    is contiguous).
    """
    kv_cache_write_impl(k, v, k_cache, v_cache, slots, k_scale_inv, v_scale_inv)


@torch._dynamo.disable
def kv_cache_read(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    slots: torch.Tensor,
    k_scale_inv: Optional[torch.Tensor] = None,
    v_scale_inv: Optional[torch.Tensor] = None,
    *,
    out_dtype: torch.dtype = torch.bfloat16,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Read cache slots back: (keys, values), each [T, Hkv, D] of ``out_dtype``.

    fp8 entries come back as ``out_dtype(fp8 * scale_inv)``; a 16-bit cache is
    copied, and ``out_dtype`` has to be its type.  A slot below 0 or past the
    pool reads as zeros.
    """
    return kv_cache_read_impl(k_cache, v_cache, slots, k_scale_inv, v_scale_inv, out_dtype)


@torch._dynamo.disable
def paged_attention(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    page_table: torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    seq_lens: torch.Tensor,
    k_scale_inv: Optional[torch.Tensor] = None,
    v_scale_inv: Optional[torch.Tensor] = None,
    *,
    softmax_scale: Optional[float] = None,
    window_size: Optional[int] = None,
    num_sinks: int = 0,
    return_lse: bool = False,
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Causal attention of every sequence's new tokens over its cached pages.

    ``q``: [T, Hq, D] bfloat16 / float16, the new tokens of all sequences one
    after the other; sequence b owns rows ``cu_seqlens_q[b]`` up to
    ``cu_seqlens_q[b + 1]`` (int32, [B + 1]): one token while decoding, a chunk
    of a prompt, or none.  ``seq_lens``: [B] int32, cached tokens of each
    sequence with the new ones (which ``kv_cache_write`` has put there).
    ``page_table``: [B, max_pages] int32; key j is in page ``page_table[b, j //
    page_size]``.  Query head h reads cache head ``h // (Hq // Hkv)``.

    ``softmax_scale``: D ** -0.5 unless given.  ``window_size``: a token at
    position t sees the keys j with t - j < window_size and the first
    ``num_sinks`` tokens; None: all j <= t.

    Returns [T, Hq, D] of q's type and, with ``return_lse``, the fp32 [T, Hq]
    logarithms of the softmax's sums.  A token that sees no key (a length of
    zero, or shorter than its new tokens) gets zeros and -inf, and so do rows that
    no sequence owns, ahead of ``cu_seqlens_q[0]`` and from ``cu_seqlens_q[B]`` on
    (a batch padded to a fixed size); one that sees only keys with logits of -inf
    gets NaN and -inf.  A value scale that is NaN or infinite makes NaN of the
    rows that see its token, of their sums too.

    The probabilities are rounded to q's type before they multiply the values, and
    the result once more; everything else is fp32.  Inference only: there is no
    backward pass.
    """
    out, lse = paged_attention_impl(q, k_cache, v_cache, page_table, cu_seqlens_q, seq_lens, k_scale_inv, v_scale_inv,
                                    softmax_scale, window_size, num_sinks, return_lse)
    return (out, lse) if return_lse else out
