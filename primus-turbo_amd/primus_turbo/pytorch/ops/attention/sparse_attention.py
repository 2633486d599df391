"""Attention of new tokens over a paged cache through few of its pages, chosen for
each token and cache head by a cheap score, for inference (no reference counterpart).

Beside the cache of ``kv_cache_write`` the caller keeps

  key_ranges   [num_pages, Hkv, 2, D] bfloat16

each channel's smallest and largest key of every page, which ``kv_page_ranges`` brings
up to date after the new keys are written.  For the query heads q_1 .. q_G of a cache
head the score of a page is

  sum_d (sum_i max(q_id, 0)) hi_d + (sum_i min(q_id, 0)) lo_d

the largest that sum_i q_i . k can be for a key k of the page, in 64 bits.  A token
attends through the first ``num_first`` and the last ``num_last`` of the pages that it
sees, the last being its own, and the best of the others up to ``num_selected`` in all
(ties to the earlier page; a NaN counts as the largest).  With no more pages than that
the result is ``paged_attention``'s.  Lengths and tables stay on the device; the calls
may be captured.
"""

from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from primus_turbo.pytorch.kernels.attention.sparse_attention_impl import (
    kv_page_ranges_impl,
    select_pages_impl,
    sparse_paged_attention_impl,
)

__all__ = ["kv_page_ranges", "select_pages", "sparse_paged_attention"]


@torch._dynamo.disable
def kv_page_ranges(
    k_cache: torch.Tensor,
    page_table: torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    seq_lens: torch.Tensor,
    key_ranges: torch.Tensor,
    k_scale_inv: Optional[torch.Tensor] = None,
) -> None:
    """Bring the ranges of the pages in which new tokens lie up to date, in place.

    The other arguments are ``paged_attention``'s.  A page's range is that of its tokens
    below the sequence's length, rounded outward to bfloat16 (a channel in which a key is
    NaN has NaN); other pages' ranges stay as they are.  A page with new tokens is one
    sequence's alone, as ``kv_cache_fork`` leaves it.
    """
    kv_page_ranges_impl(k_cache, page_table, cu_seqlens_q, seq_lens, key_ranges, k_scale_inv)


@torch._dynamo.disable
def select_pages(
    q: torch.Tensor,
    key_ranges: torch.Tensor,
    page_table: torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    seq_lens: torch.Tensor,
    page_size: int,
    *,
    num_selected: int,
    num_first: int = 1,
    num_last: int = 2,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """The pages through which ``sparse_paged_attention`` attends: (pages [T, Hkv,
    min(num_selected, max_pages)] int32, in the sequence's order, -1 behind the last, and
    [T] int32 how many keys of them a token sees, 0 for one that sees none)."""
    return select_pages_impl(q, key_ranges, page_table, cu_seqlens_q, seq_lens, page_size, num_selected, num_first, num_last)


@torch._dynamo.disable
def sparse_paged_attention(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    key_ranges: torch.Tensor,
    page_table: torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    seq_lens: torch.Tensor,
    k_scale_inv: Optional[torch.Tensor] = None,
    v_scale_inv: Optional[torch.Tensor] = None,
    *,
    num_selected: int,
    num_first: int = 1,
    num_last: int = 2,
    softmax_scale: Optional[float] = None,
    return_lse: bool = False,
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """``paged_attention`` of every token over the pages selected for it (without a window).

    A token of a chunk has pages of its own, whose ranges have to be up to date for the
    whole chunk.  A chunk's tokens go over their pages together: where they take more
    than about a quarter of the table, ``paged_attention`` of all of it is faster.
    ``softmax_scale`` is positive.  What a token that sees no key gets, what is rounded
    and what the cache may hold is as in ``paged_attention``.
    """
    out, lse = sparse_paged_attention_impl(q, k_cache, v_cache, key_ranges, page_table, cu_seqlens_q, seq_lens, k_scale_inv, v_scale_inv,
                                           num_selected, num_first, num_last, softmax_scale, return_lse)
    return (out, lse) if return_lse else out
