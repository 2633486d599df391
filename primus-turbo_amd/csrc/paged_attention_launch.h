// Kernel choice by cache kind and head dimension (instantiated per query type).
#pragma once

#include "paged_attention.h"

namespace pta {

template <int QT, int KIND, int DP> void attn_launch_d(const AttnArgs &a, int rows, hipStream_t st) {
    if (rows == ATT_NARROW_ROWS) {
        const unsigned grid = static_cast<unsigned>(a.B) * a.tiles * a.split * a.Hkv;
        attn_narrow_kernel<QT, KIND, DP><<<grid, 256, 0, st>>>(a);
        if (a.split > 1) attn_join_rows_kernel<QT><<<static_cast<unsigned>(cdiv(static_cast<int64_t>(a.Tq) * a.Hq * (a.D / 4), 64)), 256, 0, st>>>(a);
    } else {
        const unsigned grid = static_cast<unsigned>(a.slots) * static_cast<unsigned>(a.Hkv);
        attn_wide_kernel<QT, KIND, DP><<<grid, 256, 0, st>>>(a);
        if (a.split_goal > 0) attn_join_kernel<QT, ATT_WIDE_ROWS><<<dim3(grid, ATT_JOIN_PARTS), 256, 0, st>>>(a);
    }
}

template <int QT, int KIND> void attn_launch_k(const AttnArgs &a, int rows, hipStream_t st) {
    if (a.D <= 64) attn_launch_d<QT, KIND, 64>(a, rows, st);
    else if (a.D <= 128) attn_launch_d<QT, KIND, 128>(a, rows, st);
    else attn_launch_d<QT, KIND, 256>(a, rows, st);
}

template <int QT> void attn_launch(const AttnArgs &a, int kind, int rows, hipStream_t st) {
    if (kind == PTA_E4M3) attn_launch_k<QT, PTA_E4M3>(a, rows, st);
    else if (kind == PTA_E5M2) attn_launch_k<QT, PTA_E5M2>(a, rows, st);
    else attn_launch_k<QT, PTA_CACHE_16BIT>(a, rows, st);
}

} // namespace pta
