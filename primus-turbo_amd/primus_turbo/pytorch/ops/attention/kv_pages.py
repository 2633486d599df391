"""Pages of a paged cache as wholes: copied, and their books kept on the device, for
inference (no reference counterpart).

A cache is what ``kv_cache_write`` has, or all layers' at once: pools [layers,
num_pages, Hkv, page_size, D], whose layers' page ids mean the same tokens (a layer's
own operators take ``k_cache[l]``), with scales [layers, num_pages, Hkv, page_size].
``key_ranges`` ([layers,] num_pages, Hkv, 2, D]), where they are kept, go along.
Lengths and tables stay on the device and nothing here synchronizes: both calls may be
captured in a HIP graph.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from primus_turbo.pytorch.kernels.attention.kv_pages_impl import kv_cache_copy_impl, kv_cache_fork_impl

__all__ = ["kv_cache_copy", "kv_cache_fork"]


@torch._dynamo.disable
def kv_cache_copy(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    src_pages: torch.Tensor,
    dst_pages: torch.Tensor,
    k_scale_inv: Optional[torch.Tensor] = None,
    v_scale_inv: Optional[torch.Tensor] = None,
    *,
    key_ranges: Optional[torch.Tensor] = None,
) -> None:
    """Page ``dst_pages[i]`` becomes a copy of page ``src_pages[i]``, in place, in every layer.

    ``src_pages``, ``dst_pages``: int32 / int64 of one length.  A pair with a page below 0
    or past the pool is skipped.  One source may have many destinations; a destination is
    named once and is no other pair's source: what such a page holds is not defined.
    """
    kv_cache_copy_impl(k_cache, v_cache, src_pages, dst_pages, k_scale_inv, v_scale_inv, key_ranges)


@torch._dynamo.disable
def kv_cache_fork(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    page_table: torch.Tensor,
    seq_lens: torch.Tensor,
    parents: Optional[torch.Tensor] = None,
    k_scale_inv: Optional[torch.Tensor] = None,
    v_scale_inv: Optional[torch.Tensor] = None,
    *,
    key_ranges: Optional[torch.Tensor] = None,
    reserve: int = 0,
    compact: bool = False,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Sequences that go on from others: (page table, lengths) of the new ones, whose
    pages are theirs in the cache afterwards.

    New sequence i has the tokens of sequence ``parents[i]`` (int32 / int64, [N]; None:
    every sequence goes on as it is): several answers to a prompt, the beams of a step, a
    batch without the sequences that have ended.  ``page_table`` [B, max_pages] int32 and
    ``seq_lens`` [B] int32 are ``paged_attention``'s and stay as they are.

    Pages that a sequence fills are shared.  Its last page, if it is partly filled, stays
    with the first new sequence that ends in it (with none if it is another one's full
    page); the others get copies.  ``reserve``: every new sequence gets the pages of that
    many further tokens, as far as ``max_pages`` reach.  Copies and fresh pages go to the
    lowest pages that no new sequence has, in the order of the sequences.  Pages of
    sequences that nobody goes on from, and pages past a length, are free.  ``compact``:
    the n pages that the new sequences have become pages 0 to n - 1, unless pages run out.

    New rows end in -1.  A sequence for which the pages run out gets length -1 and no
    pages, and so does one that goes on from it (a parent's length below 0 is handed on);
    one whose parent does not exist gets length 0.  Table entries outside the pool (pages
    that read as zeros) stay as they are.
    """
    return kv_cache_fork_impl(k_cache, v_cache, page_table, seq_lens, parents, k_scale_inv, v_scale_inv, key_ranges, reserve, compact)
