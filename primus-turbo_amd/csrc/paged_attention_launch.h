// Kernel choice by cache kind and head dimension (instantiated per query type).
#pragma once

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

} // namespace pta
