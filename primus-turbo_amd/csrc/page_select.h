// Which pages of a long context a token attends through, as the attention's C entry calls it.
#pragma once

#include "common.h"

namespace pta {

// Tiles of tokens: the pages that any token of a tile takes, as one list for each cache head
constexpr int64_t PS_TILE_PAGES = 2048; // of a sequence at most
struct PSTiles {
    int       tokens; // of a tile, 16 at most
    int       cap;    // pages of a list at most
    int2     *list;   // [tiles, Hkv, cap]: page of the pool, position of its first key
    uint16_t *masks;  // [tiles, Hkv, cap]: bit i: the tile's i-th token takes it
    int32_t  *counts; // [tiles, Hkv]
    int32_t  *pos;    // [T]: the token's position, -1 where it sees nothing
};

// Bytes for the choice among `max_pages` pages; tile: tokens of a tile, or 1
size_t ps_workspace(int64_t num_tokens, int64_t Hkv, int64_t max_pages, int64_t tile);
int    ps_check(int64_t num_tokens, int64_t num_seqs, int64_t Hq, int64_t Hkv, int64_t D, int64_t num_pages, int64_t page_size,
                int64_t max_pages, int64_t num_selected, int64_t num_first, int64_t num_last);
// selected [T, Hkv, min(num_selected, max_pages)], or tiles instead (max_pages up to PS_TILE_PAGES);
// selected_cu [T + 1] gets 0, 1, 2, ... (may be null without tiles)
int    ps_select(const void *q, int q_dtype, int64_t num_tokens, int64_t Hq, int64_t D, int64_t q_stride_t, int64_t q_stride_h,
                 const void *key_ranges, int64_t num_pages, int64_t page_size, int64_t Hkv, const int32_t *page_table, int64_t table_stride,
                 int64_t max_pages, const int32_t *cu_seqlens_q, const int32_t *seq_lens, int64_t num_seqs, int64_t num_selected,
                 int64_t num_first, int64_t num_last, int32_t *selected, const PSTiles *tiles, int32_t *selected_lens, int32_t *selected_cu,
                 void *workspace, hipStream_t stream);

} // namespace pta
