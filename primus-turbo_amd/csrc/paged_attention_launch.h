// Kernel choice by cache kind and head dimension (instantiated per query type).
#pragma once

#include "paged_attention.h"

namespace pta {

template <int QT, int KIND, int DP> void attn_launch_d(const AttnArgs &a, bool wide, hipStream_t st) {
    const unsigned grid = static_cast<unsigned>(a.slots) * static_cast<unsigned>(a.Hkv);
    if (wide) {
        attn_wide_kernel<QT, KIND, DP, ATT_WIDE_ROWS / 32><<<grid, ATT_WIDE_ROWS * 2, 0, st>>>(a);
        if (a.split_goal > 0) attn_join_kernel<QT, ATT_WIDE_ROWS><<<grid, 256, 0, st>>>(a);
    } else {
        attn_narrow_kernel<QT, KIND, DP><<<grid, 256, 0, st>>>(a);
        if (a.split_goal > 0) attn_join_kernel<QT, ATT_NARROW_ROWS><<<grid, 256, 0, st>>>(a);
    }
}

template <int QT, int KIND> void attn_launch_k(const AttnArgs &a, bool wide, hipStream_t st) {
    if (a.D <= 64) attn_launch_d<QT, KIND, 64>(a, wide, st);
    else if (a.D <= 128) attn_launch_d<QT, KIND, 128>(a, wide, st);
    else attn_launch_d<QT, KIND, 256>(a, wide, st);
}

template <int QT> void attn_launch(const AttnArgs &a, int kind, bool wide, hipStream_t st) {
    if (kind == PTA_E4M3) attn_launch_k<QT, PTA_E4M3>(a, wide, st);
    else if (kind == PTA_E5M2) attn_launch_k<QT, PTA_E5M2>(a, wide, st);
    else attn_launch_k<QT, PTA_CACHE_16BIT>(a, wide, st);
}

} // namespace pta
