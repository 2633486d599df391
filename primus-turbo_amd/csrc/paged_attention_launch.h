// Kernel choice by cache kind and head dimension (instantiated per query type).
#pragma once

#include <algorithm>

#include "paged_attention.h"

namespace pta {

template <int QT, int KIND, int DP> void attn_launch_d(const AttnCall &c, hipStream_t st) {
    const AttnArgs &n = c.narrow, &w = c.wide;
    const unsigned  n_blocks = static_cast<unsigned>(n.B) * n.split * n.Hkv, w_blocks = static_cast<unsigned>(w.slots) * w.Hkv;
    const unsigned  pads = static_cast<unsigned>(c.pads);
    if (c.has_narrow && c.has_wide) attn_both_kernel<QT, KIND, DP><<<w_blocks + n_blocks + pads, 256, 0, st>>>(w, n, w_blocks, c.pads);
    else if (c.has_wide) attn_wide_kernel<QT, KIND, DP><<<w_blocks + pads, 256, 0, st>>>(w, c.pads);
    else attn_narrow_kernel<QT, KIND, DP><<<n_blocks + pads, 256, 0, st>>>(n, c.pads);
}

template <int QT, int KIND> void attn_launch_k(const AttnCall &c, int D, hipStream_t st) {
    if (D <= 64) attn_launch_d<QT, KIND, 64>(c, st);
    else if (D <= 128) attn_launch_d<QT, KIND, 128>(c, st);
    else attn_launch_d<QT, KIND, 256>(c, st);
}

template <int QT> void attn_launch(const AttnCall &c, int kind, hipStream_t st) {
    const int D = c.has_narrow ? c.narrow.D : c.wide.D;
    if (kind == PTA_E4M3) attn_launch_k<QT, PTA_E4M3>(c, D, st);
    else if (kind == PTA_E5M2) attn_launch_k<QT, PTA_E5M2>(c, D, st);
    else attn_launch_k<QT, PTA_CACHE_16BIT>(c, D, st);
    const int n = c.has_narrow && c.narrow.split > 1 ? c.narrow.B * c.narrow.Hkv * c.narrow_join_parts : 0;
    const int w = c.has_wide && c.wide.split_goal > 0 ? c.wide.slots * c.wide.Hkv * ATT_JOIN_PARTS : 0;
    if (n + w == 0) return;
    auto join = c.narrow.split > 4 ? attn_join_kernel<QT, 4> : attn_join_kernel<QT, 1>;
    join<<<static_cast<unsigned>(n + w), 256, 0, st>>>(c.narrow, c.wide, n, c.narrow_join_parts);
}

// Pages of whole runs of 32 keys: ranges and attention of 1024 tokens over 16384, 16 of 256 pages of 64,
// 32 / 8 heads of 64, 128 and 256, e4m3, take 105, 157 and 453 us, by a key at a time 118, 179 and 574
// (bf16 caches 111, 178 and 468; 155, 251 and 668).
template <int QT, int KIND, int DP> void attn_launch_tiles_d(const AttnArgs &a, hipStream_t st) {
    const unsigned grid = static_cast<unsigned>(a.B) * a.split * a.Hkv;
    if (a.page % 32 == 0 && a.num_pages > 0) attn_tile_kernel<QT, KIND, DP, true><<<grid, 256, 0, st>>>(a);
    else attn_tile_kernel<QT, KIND, DP, false><<<grid, 256, 0, st>>>(a);
}

template <int QT, int KIND> void attn_launch_tiles_k(const AttnArgs &a, hipStream_t st) {
    if (a.D <= 64) attn_launch_tiles_d<QT, KIND, 64>(a, st);
    else if (a.D <= 128) attn_launch_tiles_d<QT, KIND, 128>(a, st);
    else attn_launch_tiles_d<QT, KIND, 256>(a, st);
}

template <int QT> void attn_launch_tiles(const AttnArgs &a, int kind, hipStream_t st) {
    if (kind == PTA_E4M3) attn_launch_tiles_k<QT, PTA_E4M3>(a, st);
    else if (kind == PTA_E5M2) attn_launch_tiles_k<QT, PTA_E5M2>(a, st);
    else attn_launch_tiles_k<QT, PTA_CACHE_16BIT>(a, st);
    if (a.split == 1) return;
    // the parts are the tokens': each is a sequence of its own here, whose length says
    // whether it sees a key
    AttnArgs  x = a;
    const int parts = static_cast<int>(std::min<int64_t>(ATT_JOIN_PARTS, cdiv(static_cast<int64_t>(a.G) * (a.D / 4), 64)));
    x.B         = a.Tq;
    const int n = a.Tq * a.Hkv * parts;
    auto join   = a.split > 4 ? attn_join_kernel<QT, 4> : attn_join_kernel<QT, 1>;
    join<<<static_cast<unsigned>(n), 256, 0, st>>>(x, x, n, parts);
}

} // namespace pta
