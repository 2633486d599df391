// Attention through few pages of a long context: the range of each page's keys, the
// scores that a token's pages are chosen by, and the choice.
//
// Range of a page and head: each channel's smallest and largest key (fp32: fp8 value
// times scale), rounded outward to bf16, so that it holds every key; a channel with a
// NaN has NaN.
//
// Score of page g for token t and cache head h, whose query heads are q_1 .. q_G:
//
//   score = sum_d hi_d P_d - lo_d N_d,   P_d = sum_i max(q_id, 0),  N_d = sum_i max(-q_id, 0)
//
// the largest that sum_i q_i . k can be for a key k within the ranges.  The heads'
// sum turns G products of 2 D into one.  It is computed in 64 bits.  The forms below sum in
// orders of their own, so that scores closer than a few roundings (2^-53 of the sum of the
// terms' magnitudes each) may rank otherwise in another form; within a form a score depends
// on its query and range alone, and equal ranges tie.  A NaN counts as +inf: pages with NaN
// are attended, and show.  The first `first` and the last `last` pages of those that a
// token sees are taken always, the rest by score, ties to the lower page.
#include <algorithm>
#include <climits>

#include "page_select.h"

namespace pta {
namespace {

constexpr int PS_NT = 256;

struct PSArgs {
    const uint16_t *q;
    int64_t         q_st, q_sh;
    const uint16_t *ranges;  // [P, Hkv, 2, D] bf16
    const int32_t  *table;
    int64_t         table_st;
    const int32_t  *cu, *lens;
    uint64_t       *keys;    // workspace: [tokens of a slice, Hkv, M] scores as ordered whole numbers
    int32_t        *sel;      // [T, Hkv, K] pages of the pool, rising in the sequence; -1 behind the last
    PSTiles         tiles;    // tokens > 0: lists for tiles instead
    int32_t        *sel_lens; // [T] keys of them that the token sees
    int32_t        *sel_cu;  // [T + 1] 0, 1, 2, ... (may be null)
    int             T, B, Hq, Hkv, G, D, M, P, page;
    int             take, first, last, K;
    int             t0, n;   // the slice
};


// A token's sequence and its place in it; b < 0: it has none.
struct PSToken {
    int b, pos, len, n, i;
};
__device__ __forceinline__ PSToken ps_place(const PSArgs &a, int t, int lo) {
    PSToken   s = {-1, -1, 0, 0, 0};
    const int tok0 = min(max(a.cu[lo], 0), a.T), end = min(max(a.cu[lo + 1], tok0), a.T);
    if (t < tok0 || t >= end) return s;
    s.b   = lo;
    s.n   = end - tok0;
    s.i   = t - tok0;
    s.len = static_cast<int>(min(static_cast<int64_t>(max(a.lens[lo], 0)), static_cast<int64_t>(a.M) * a.page));
    s.pos = s.len - s.n + s.i;
    return s;
}
// The last sequence that begins at or before t, 64 of them looked at together: all lanes
// of a wave ask for the same token, and get it into scalar registers
__device__ __forceinline__ PSToken ps_token(const PSArgs &a, int t) {
    int lo = 0, hi = a.B;
    while (hi - lo > 1) {
        const int step = (hi - lo + 63) / 64, at = lo + lane_id() * step;
        const int n    = __popcll(__ballot(at < hi && a.cu[min(at, hi - 1)] <= t));
        lo += max(n - 1, 0) * step;
        hi = min(lo + step, hi);
    }
    PSToken s = ps_place(a, t, __builtin_amdgcn_readfirstlane(lo));
    for (int *f : {&s.b, &s.pos, &s.len, &s.n, &s.i}) *f = __builtin_amdgcn_readfirstlane(*f);
    return s;
}
// The same by bisection, for lanes with tokens of their own
__device__ __forceinline__ PSToken ps_token_of_lane(const PSArgs &a, int t) {
    int lo = 0, hi = a.B;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (a.cu[mid] <= t) lo = mid;
        else hi = mid;
    }
    return ps_place(a, t, lo);
}

// ---- ranges ------------------------------------------------------------------------
struct PRArgs {
    const uint8_t *kc;
    const float   *ks;
    const int32_t *table;
    int64_t        table_st;
    const int32_t *cu, *lens;
    uint16_t      *ranges;
    int            B, Hkv, D, M, P, page, parts;
};

// The smaller and the larger of two, NaN if one is
__device__ __forceinline__ float pr_less(float x, float y) { return x < y || x != x ? x : y; }
__device__ __forceinline__ float pr_more(float x, float y) { return x > y || x != x ? x : y; }

__device__ __forceinline__ uint16_t pr_outward(float x, bool up) {
    const uint32_t u = __float_as_uint(x);
    if (x != x) return 0x7fc0;
    const bool away = (u & 0xffffu) != 0 && ((u >> 31) != 0) != up;
    return static_cast<uint16_t>((u >> 16) + away);
}

// Workgroup = (head, part, sequence), for every parts-th page that holds new tokens.  A
// thread has 4 channels of every GROUPS-th key, NL threads a key.  A few pages are a chain of
// reads: 64 pages of 32 tokens, 4 heads of 64, 5 us (with 16 channels a thread, and so four
// times the rows to join in LDS, 7.2).
template <int KIND, int NL> __global__ __launch_bounds__(PS_NT) void pr_ranges_kernel(PRArgs a) {
    constexpr int     GROUPS = PS_NT / NL;
    constexpr bool    FP8    = KIND == PTA_E4M3 || KIND == PTA_E5M2;
    __shared__ float4 red[2][GROUPS][NL];
    const int         h = blockIdx.x % a.Hkv, w = blockIdx.x / a.Hkv, part = w % a.parts, b = w / a.parts;
    const int64_t     fresh = static_cast<int64_t>(a.cu[b + 1]) - a.cu[b];
    const int         len = static_cast<int>(min(static_cast<int64_t>(max(a.lens[b], 0)), static_cast<int64_t>(a.M) * a.page));
    if (fresh <= 0 || len == 0) return;
    const int  first = static_cast<int>(max(static_cast<int64_t>(0), len - fresh)) / a.page, l = threadIdx.x % NL, g = threadIdx.x / NL;
    const bool in = l * 4 < a.D;
    for (int pg = first + part; pg * static_cast<int64_t>(a.page) < len; pg += a.parts) {
        const int u = a.table[b * a.table_st + pg];
        if (u < 0 || u >= a.P) continue;
        const int     n = min(a.page, len - pg * a.page);
        const int64_t row0 = (static_cast<int64_t>(u) * a.Hkv + h) * a.page;
        float         lo[4], hi[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            lo[e] = INFINITY;
            hi[e] = -INFINITY;
        }
        if (in)
#pragma unroll 8
            for (int j = g; j < n; j += GROUPS) {
                float         v[4];
                const int64_t at = (row0 + j) * a.D + l * 4;
                if constexpr (FP8) {
                    const int   x = *reinterpret_cast<const int *>(a.kc + at);
                    const float sc = a.ks[row0 + j];
                    if constexpr (KIND == PTA_E4M3) {
                        v[0] = __builtin_amdgcn_cvt_f32_fp8(x, 0) * sc; v[1] = __builtin_amdgcn_cvt_f32_fp8(x, 1) * sc;
                        v[2] = __builtin_amdgcn_cvt_f32_fp8(x, 2) * sc; v[3] = __builtin_amdgcn_cvt_f32_fp8(x, 3) * sc;
                    } else {
                        v[0] = __builtin_amdgcn_cvt_f32_bf8(x, 0) * sc; v[1] = __builtin_amdgcn_cvt_f32_bf8(x, 1) * sc;
                        v[2] = __builtin_amdgcn_cvt_f32_bf8(x, 2) * sc; v[3] = __builtin_amdgcn_cvt_f32_bf8(x, 3) * sc;
                    }
                } else {
                    const uint2 x = *reinterpret_cast<const uint2 *>(a.kc + 2 * at);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t y = (e < 2 ? x.x : x.y) >> (16 * (e & 1)) & 0xffffu;
                        v[e] = KIND == PTA_CACHE_16BIT ? bf16_bits_to_f32(y) : f16_bits_to_f32(y);
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    lo[e] = pr_less(v[e], lo[e]);
                    hi[e] = pr_more(v[e], hi[e]);
                }
            }
        red[0][g][l] = make_float4(lo[0], lo[1], lo[2], lo[3]);
        red[1][g][l] = make_float4(hi[0], hi[1], hi[2], hi[3]);
        __syncthreads();
        for (int d = threadIdx.x; d < 2 * a.D; d += PS_NT) {
            const bool   up = d >= a.D;
            const int    c = up ? d - a.D : d;
            const float *p = reinterpret_cast<const float *>(&red[up][0][0]) + c;
            float        x = p[0];
#pragma unroll 8
            for (int i = 1; i < GROUPS; ++i) x = up ? pr_more(p[i * NL * 4], x) : pr_less(p[i * NL * 4], x);
            a.ranges[((static_cast<int64_t>(u) * a.Hkv + h) * 2 + up) * a.D + c] = pr_outward(x, up);
        }
        __syncthreads(); // the next page's values come to the same place
    }
}

// ---- scores ------------------------------------------------------------------------
// sum over groups of LPR lanes
template <int CTRL> __device__ __forceinline__ double ps_dpp(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const int      a = __builtin_amdgcn_mov_dpp(static_cast<int>(u), CTRL, 0xf, 0xf, false);
    const int      b = __builtin_amdgcn_mov_dpp(static_cast<int>(u >> 32), CTRL, 0xf, 0xf, false);
    return __builtin_bit_cast(double, static_cast<uint64_t>(static_cast<uint32_t>(a)) | (static_cast<uint64_t>(static_cast<uint32_t>(b)) << 32));
}
template <int LPR> __device__ __forceinline__ double ps_sum(double v) {
    v += ps_dpp<PTA_DPP_QUAD_XOR1>(v);
    v += ps_dpp<PTA_DPP_QUAD_XOR2>(v);
    v += ps_dpp<PTA_DPP_ROW_HALF_MIRROR>(v);
    if constexpr (LPR >= 16) v += ps_dpp<PTA_DPP_ROW_MIRROR>(v);
    if constexpr (LPR >= 32) v += __shfl_xor(v, 16);
    return v;
}

// Scores in their order as whole numbers; 0 is below all of them
__device__ __forceinline__ uint64_t ps_key(double s) {
    if (s != s) s = INFINITY;
    const uint64_t u = __builtin_bit_cast(uint64_t, s + 0.0); // -0 counts as 0
    return (u >> 63) ? ~u : u | (1ull << 63);
}

// A query's channel to the sums of the positive and of the negative parts; to both if it is
// NaN, which has to reach the score
__device__ __forceinline__ void ps_add(float v, double &up, double &down) {
    up += v < 0.0f ? 0.0f : v;
    down += v > 0.0f ? 0.0f : v;
}
template <int QT> __device__ __forceinline__ void ps_channel(const PSArgs &a, int t, int h, int d, double &up, double &down) {
    const uint16_t *q = a.q + t * a.q_st + static_cast<int64_t>(h) * a.G * a.q_sh + d;
    up = down = 0.0;
#pragma unroll 8
    for (int i = 0; i < a.G; ++i) {
        const uint32_t x = q[i * a.q_sh];
        ps_add(QT == PTA_BF16 ? bf16_bits_to_f32(x) : f16_bits_to_f32(x), up, down);
    }
}

// Keys of pages [j0, j1) of the token's sequence to out: a page's range to LPR of the NT
// threads, 8 channels each, four pages of a thread's loads together.
template <int LPR, int NT>
__device__ __forceinline__ void ps_scores(const PSArgs &a, const double (&sums)[2][8 * LPR], const int32_t *row, int h, int j0, int j1, uint64_t *out) {
    constexpr int GROUPS = NT / LPR, PAGES = 4;
    const int     l = threadIdx.x % LPR, g = threadIdx.x / LPR, d = l * 8;
    const bool    in = d < a.D;
    double        up[8], down[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        up[e]   = in ? sums[0][d + e] : 0.0;
        down[e] = in ? sums[1][d + e] : 0.0;
    }
    for (int p0 = j0 + g; p0 < j1; p0 += GROUPS * PAGES) {
        uint4 lo[PAGES], hi[PAGES];
        bool  there[PAGES];
#pragma unroll
        for (int i = 0; i < PAGES; ++i) {
            const int j = p0 + i * GROUPS, u = j < j1 ? row[j] : -1;
            there[i]    = in && u >= 0 && u < a.P; // a page outside the pool holds zeros
            const uint16_t *r = a.ranges + (static_cast<int64_t>(there[i] ? u : 0) * a.Hkv + h) * 2 * a.D + (in ? d : 0);
            lo[i] = hi[i] = make_uint4(0, 0, 0, 0);
            if (there[i]) {
                lo[i] = *reinterpret_cast<const uint4 *>(r);
                hi[i] = *reinterpret_cast<const uint4 *>(r + a.D);
            }
        }
#pragma unroll
        for (int i = 0; i < PAGES; ++i) {
            const int      j = p0 + i * GROUPS;
            const uint32_t wl[4] = {lo[i].x, lo[i].y, lo[i].z, lo[i].w}, wh[4] = {hi[i].x, hi[i].y, hi[i].z, hi[i].w};
            double         x = 0.0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t bl = e % 2 ? wl[e / 2] & 0xffff0000u : wl[e / 2] << 16, bh = e % 2 ? wh[e / 2] & 0xffff0000u : wh[e / 2] << 16;
                x = fma(up[e], static_cast<double>(__uint_as_float(bh)), fma(down[e], static_cast<double>(__uint_as_float(bl)), x));
            }
            if (!there[i]) x = 0.0; // also where a query is not finite
            x = ps_sum<LPR>(x);
            if (l == 0 && j < j1) out[j] = ps_key(x);
        }
    }
}

// Few tokens with many pages (1 token, 2048 pages, 8 heads of 128: 5.4 us): pages [c per, (c + 1) per)
// of token t for head h.  Bound by the chain of reads: the token's place, queries and page numbers, ranges.
template <int QT, int LPR> __global__ __launch_bounds__(PS_NT) void ps_score_kernel(PSArgs a, int per, int parts) {
    __shared__ double sums[2][8 * LPR];
    const uint32_t w = blockIdx.x, h = w % a.Hkv, w1 = w / a.Hkv, c = w1 % parts, ti = w1 / parts;
    const int      t = a.t0 + static_cast<int>(ti);
    const PSToken  s = ps_token(a, t);
    if (s.b < 0 || s.pos < 0) return;
    const int n = s.pos / a.page + 1, j0 = c * per, j1 = min(j0 + per, n);
    if (j0 >= j1 || n <= a.take) return;
    if (static_cast<int>(threadIdx.x) < a.D) ps_channel<QT>(a, t, h, threadIdx.x, sums[0][threadIdx.x], sums[1][threadIdx.x]);
    __syncthreads();
    ps_scores<LPR, PS_NT>(a, sums, a.table + s.b * a.table_st, h, j0, j1, a.keys + (static_cast<int64_t>(ti) * a.Hkv + h) * a.M);
}

// Chunks: 16 tokens by 16 pages on the 64-bit matrix instruction, D = R B with a page's
// range as a row of R (2 D channels, the smallest keys, then the largest) and a token's
// sums as a column of B, which all pages read from LDS.  Which channel is which step of
// the contraction is free: quarter k of the lanes has channels [k D / 2, (k + 1) D / 2),
// one run of its page's range.  Tokens of several sequences are gone through sequence by
// sequence, with the other tokens' columns unused.
//
// 1024 tokens by 256 pages, 8 heads of 128: 31 us, of which the matrix pipe is busy 14 (64
// cycles an instruction); by vector instructions, token by token, 113.
typedef double ps_d4 __attribute__((ext_vector_type(4)));
constexpr int  PS_TILE = 16;

template <int QT, int DP> __global__ __launch_bounds__(PS_NT) void ps_score_tile_kernel(PSArgs a, int per, int parts) {
    __shared__ double sums[2 * DP * PS_TILE]; // [channel][token]
    __shared__ int    sb[PS_TILE], spos[PS_TILE];
    const uint32_t    w = blockIdx.x, h = w % a.Hkv, w1 = w / a.Hkv, c = w1 % parts, tile = w1 / parts;
    const int         ti0 = static_cast<int>(tile) * PS_TILE, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (tid < PS_TILE) {
        PSToken s = {-1, -1, 0, 0, 0};
        if (ti0 + tid < a.n) s = ps_token_of_lane(a, a.t0 + ti0 + tid);
        sb[tid]   = s.pos < 0 ? -1 : s.b;
        spos[tid] = s.pos;
    }
    for (int x = tid; x < PS_TILE * (a.D / 8); x += PS_NT) {
        const int i = x % PS_TILE, d = x / PS_TILE * 8;
        double    up[8], down[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) up[e] = down[e] = 0.0;
        if (ti0 + i < a.n) {
            const uint16_t *q = a.q + (a.t0 + ti0 + i) * a.q_st + static_cast<int64_t>(h) * a.G * a.q_sh + d;
#pragma unroll 4
            for (int g = 0; g < a.G; ++g) {
                float v[8];
                load8<QT>(q, g * a.q_sh, v);
#pragma unroll
                for (int e = 0; e < 8; ++e) ps_add(v[e], up[e], down[e]);
            }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            sums[(d + e) * PS_TILE + i]       = down[e];
            sums[(a.D + d + e) * PS_TILE + i] = up[e];
        }
    }
    __syncthreads();
    const int r = lane & 15, quarter = lane >> 4, half = a.D / 2;
    const int b_me = sb[r], own_me = spos[r] / a.page; // of the lane's token
    uint64_t *out  = a.keys + (static_cast<int64_t>(ti0 + r) * a.Hkv + h) * a.M;
    for (int i0 = 0; i0 < PS_TILE;) {
        const int b = sb[i0];
        int       i1 = i0 + 1;
        while (i1 < PS_TILE && sb[i1] == b) ++i1;
        const int n = b < 0 ? 0 : spos[i1 - 1] / a.page + 1, j0 = static_cast<int>(c) * per, j1 = min(j0 + per, n);
        i0 = i1;
        if (n <= a.take) continue;
        const int32_t *row = a.table + b * a.table_st;
        for (int p0 = j0 + wave * 16; p0 < j1; p0 += PS_NT / 64 * 16) {
            const int       u = p0 + r < j1 ? row[p0 + r] : -1;
            const bool      there = u >= 0 && u < a.P; // a page outside the pool holds zeros
            const uint16_t *x = a.ranges + (static_cast<int64_t>(there ? u : 0) * a.Hkv + h) * 2 * a.D + quarter * half;
            const double   *y = sums + quarter * half * PS_TILE + r;
            uint4           v[DP / 16];
#pragma unroll
            for (int s = 0; s < DP / 16; ++s) v[s] = there && s * 8 < half ? *reinterpret_cast<const uint4 *>(x + s * 8) : make_uint4(0, 0, 0, 0);
            ps_d4 acc = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
            for (int s = 0; s < DP / 16; ++s) {
                if (s * 8 >= half) break;
                const uint32_t z[4] = {v[s].x, v[s].y, v[s].z, v[s].w};
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    acc = __builtin_amdgcn_mfma_f64_16x16x4f64(
                        static_cast<double>(__uint_as_float(e % 2 ? z[e / 2] & 0xffff0000u : z[e / 2] << 16)), y[(s * 8 + e) * PS_TILE], acc, 0, 0, 0);
            }
            const uint64_t is = __ballot(there); // pages in its low 16 bits
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int g = quarter + 4 * i, j = p0 + g; // the lane's i-th score is of this page
                if (b_me != b || j >= j1 || j > own_me) continue;
                out[j] = ps_key(is >> g & 1 ? acc[i] : 0.0);
            }
        }
    }
}

// ---- choice ------------------------------------------------------------------------
// and, or of a wave's lanes
__device__ __forceinline__ uint32_t ps_dpp_u32(uint32_t v, int step) {
    switch (step) {
    case 0: return __builtin_amdgcn_mov_dpp(v, PTA_DPP_QUAD_XOR1, 0xf, 0xf, false);
    case 1: return __builtin_amdgcn_mov_dpp(v, PTA_DPP_QUAD_XOR2, 0xf, 0xf, false);
    case 2: return __builtin_amdgcn_mov_dpp(v, PTA_DPP_ROW_HALF_MIRROR, 0xf, 0xf, false);
    default: return __builtin_amdgcn_mov_dpp(v, PTA_DPP_ROW_MIRROR, 0xf, 0xf, false);
    }
}
__device__ __forceinline__ void ps_common(uint32_t &all, uint32_t &any) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        all &= ps_dpp_u32(all, i);
        any |= ps_dpp_u32(any, i);
    }
    auto x = __builtin_amdgcn_permlane16_swap(all, all, false, false);
    auto y = __builtin_amdgcn_permlane16_swap(any, any, false, false);
    all = x[0] & x[1];
    any = y[0] | y[1];
    x   = __builtin_amdgcn_permlane32_swap(all, all, false, false);
    y   = __builtin_amdgcn_permlane32_swap(any, any, false, false);
    all = __builtin_amdgcn_readfirstlane(x[0] & x[1]);
    any = __builtin_amdgcn_readfirstlane(y[0] | y[1]);
}

// Bits of the high halves that all scores of a wave have, or any; not of pages taken always
template <int E> __device__ __forceinline__ void ps_bits(const uint64_t (&key)[E], uint32_t &common, uint32_t &any) {
    common = ~0u;
    any    = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const uint32_t x = static_cast<uint32_t>(key[e] >> 32);
        common &= key[e] + 1 > 1 ? x : ~0u;
        any |= key[e] + 1 > 1 ? x : 0u;
    }
    ps_common(common, any);
}

// The least of the `take` largest of a wave's keys (0: none): its bits from the highest that
// differs on; a bit is set if enough keys have it.  The search ends when exactly as many are
// left.  The high halves come first, whose comparisons are cheaper: all but ties differ there.
template <int E> __device__ __forceinline__ uint64_t ps_least(const uint64_t (&key)[E], int take) {
    uint32_t common, any;
    ps_bits<E>(key, common, any);
    const int top   = 31 - __clz(common ^ any); // -1: they differ in none
    uint64_t  least = static_cast<uint64_t>(top < 0 ? any : any & ~((2u << top) - 1)) << 32;
    for (int bit = top; bit >= 0; --bit) {
        const uint32_t cand = static_cast<uint32_t>(least >> 32) | (1u << bit);
        int            c = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) c += __popcll(__ballot(static_cast<uint32_t>(key[e] >> 32) >= cand));
        if (c >= take) least = static_cast<uint64_t>(cand) << 32;
        if (c == take) return least; // all of these and no others
    }
    for (int bit = 31; bit >= 0; --bit) {
        const uint64_t cand = least | (1ull << bit);
        int            c = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) c += __popcll(__ballot(key[e] >= cand));
        if (c >= take) least = cand;
        if (c == take) return least;
    }
    return least;
}

// A page's key in the choice: that of its score, above all of them for the first and last pages
__device__ __forceinline__ uint64_t ps_at(const PSArgs &a, const uint64_t *keys, int own, int j) {
    return j < a.first || own - j < a.last ? ~0ull : keys[j];
}

// What a token gets without a choice; true if it needs one.  All threads call it.
__device__ __forceinline__ bool ps_begin(const PSArgs &a, const PSToken &s, int t, int h, int own, int take, int32_t *sel) {
    if (h == 0 && threadIdx.x == 0) {
        a.sel_lens[t] = own >= 0 ? (take - 1) * a.page + (s.pos - own * a.page) + 1 : 0;
        if (a.sel_cu != nullptr) {
            a.sel_cu[t] = t;
            if (t == a.T - 1) a.sel_cu[a.T] = a.T;
        }
    }
    for (int j = take + static_cast<int>(threadIdx.x); j < a.K; j += blockDim.x) sel[j] = -1;
    if (own < 0) return false;
    if (own + 1 > a.take) return true;
    const int32_t *row = a.table + s.b * a.table_st;
    for (int j = threadIdx.x; j <= own; j += blockDim.x) sel[j] = row[j];
    return false;
}

// One wave's choice among up to 64 E pages: the keys above the least, and of those equal to it
// the first ones, in the pages' order.
template <int E> __device__ __forceinline__ void ps_take(const PSArgs &a, const uint64_t *keys, int own, int take, const int32_t *row, int32_t *sel) {
    const int lane = lane_id(), n = own + 1;
    uint64_t  key[E];
#pragma unroll
    for (int e = 0; e < E; ++e) key[e] = e * 64 + lane < n ? ps_at(a, keys, own, e * 64 + lane) : 0; // below every score
    const uint64_t least = ps_least<E>(key, take), below = (1ull << lane) - 1;
    int            above = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) above += __popcll(__ballot(key[e] > least));
    int at = 0, room = take - above; // of the equal ones
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const uint64_t eq = __ballot(key[e] == least);
        const uint64_t m  = __ballot(key[e] > least || (key[e] == least && __popcll(eq & below) < room));
        if (m >> lane & 1) sel[at + __popcll(m & below)] = row[e * 64 + lane];
        at += __popcll(m);
        room -= min(room, static_cast<int>(__popcll(eq)));
    }
}

// Up to 256 or 512 pages, a wave for (token, head); bound by the search's steps, about 3 E
// instructions each
template <int E> __global__ __launch_bounds__(64) void ps_choose_kernel(PSArgs a) {
    const int      ti = blockIdx.x / a.Hkv, h = blockIdx.x - ti * a.Hkv, t = a.t0 + ti;
    const PSToken  s = ps_token(a, t);
    const int      own = s.b >= 0 && s.pos >= 0 ? s.pos / a.page : -1, take = min(own + 1, a.take);
    int32_t       *sel = a.sel + (static_cast<int64_t>(t) * a.Hkv + h) * a.K;
    if (!ps_begin(a, s, t, h, own, take, sel)) return;
    ps_take<E>(a, a.keys + (static_cast<int64_t>(ti) * a.Hkv + h) * a.M, own, take, a.table + s.b * a.table_st, sel);
}

// Few tokens with up to 512 pages: scores and choice in one workgroup for (token, head) (64
// tokens of 285 pages on average, 4 heads of 64: 12.9 us, as two kernels 16.5)
constexpr int PS_ONE = 512;
template <int QT, int LPR> __global__ __launch_bounds__(1024) void ps_select_kernel(PSArgs a) {
    __shared__ double   sums[2][8 * LPR];
    __shared__ uint64_t keys[PS_ONE];
    const int      ti = blockIdx.x / a.Hkv, h = blockIdx.x - ti * a.Hkv, t = a.t0 + ti;
    const PSToken  s = ps_token(a, t);
    const int      own = s.b >= 0 && s.pos >= 0 ? s.pos / a.page : -1, take = min(own + 1, a.take);
    int32_t       *sel = a.sel + (static_cast<int64_t>(t) * a.Hkv + h) * a.K;
    if (!ps_begin(a, s, t, h, own, take, sel)) return;
    const int32_t *row = a.table + s.b * a.table_st;
    if (static_cast<int>(threadIdx.x) < a.D) ps_channel<QT>(a, t, h, threadIdx.x, sums[0][threadIdx.x], sums[1][threadIdx.x]);
    __syncthreads();
    ps_scores<LPR, 1024>(a, sums, row, h, 0, own + 1, keys);
    __syncthreads();
    if (threadIdx.x < 64) ps_take<PS_ONE / 64>(a, keys, own, take, row, sel);
}

// More pages: NW waves for (token, head), wave w with keys [64 w E, 64 (w + 1) E), E a lane;
// what does not fit is read again for every step of the search.  The search is ps_least's, with
// a barrier a step (2048 pages, 8 heads: 10.7 us; 12 with 4 or 16 waves, 17 with one of 32 keys a lane).
template <int NW, int E> __global__ __launch_bounds__(64 * NW) void ps_choose_many_kernel(PSArgs a) {
    constexpr int  CAP = 64 * NW * E;
    __shared__ int cnt[2][2][NW];
    const int      ti = blockIdx.x / a.Hkv, h = blockIdx.x - ti * a.Hkv, t = a.t0 + ti;
    const int      lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const PSToken  s = ps_token(a, t);
    const int      own = s.b >= 0 && s.pos >= 0 ? s.pos / a.page : -1, n = own + 1, take = min(n, a.take);
    int32_t       *sel = a.sel + (static_cast<int64_t>(t) * a.Hkv + h) * a.K;
    if (!ps_begin(a, s, t, h, own, take, sel)) return;
    const int32_t  *row = a.table + s.b * a.table_st;
    const uint64_t *in = a.keys + (static_cast<int64_t>(ti) * a.Hkv + h) * a.M;
    uint64_t        key[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int j = (wave * E + e) * 64 + lane;
        key[e]      = j < n ? ps_at(a, in, own, j) : 0; // below every score
    }
    // sums of x and of y over the workgroup, and over the waves before
    int  buf = 0;
    auto all = [&](int x, int y, int &sx, int &sy, int &bx, int &by) {
        if (lane == 0) {
            cnt[buf][0][wave] = x;
            cnt[buf][1][wave] = y;
        }
        __syncthreads();
        sx = sy = bx = by = 0;
        for (int w = 0; w < NW; ++w) {
            if (w < wave) {
                bx += cnt[buf][0][w];
                by += cnt[buf][1][w];
            }
            sx += cnt[buf][0][w];
            sy += cnt[buf][1][w];
        }
        buf ^= 1;
    };
    uint64_t least = 0;
    bool done = false;
    int  top  = 63;
    if (n <= CAP) {
        uint32_t common, any;
        ps_bits<E>(key, common, any);
        if (lane == 0) {
            cnt[1][0][wave] = static_cast<int>(common);
            cnt[1][1][wave] = static_cast<int>(any);
        }
        __syncthreads(); // the next to write there comes behind the next barrier but one
        for (int w = 0; w < NW; ++w) {
            common &= static_cast<uint32_t>(cnt[1][0][w]);
            any |= static_cast<uint32_t>(cnt[1][1][w]);
        }
        top   = 63 - __clz(common ^ any); // 31: they differ in none
        least = static_cast<uint64_t>(top < 32 ? any : any & ~((2u << (top - 32)) - 1)) << 32;
    }
    for (int bit = top; bit >= 0 && !done; --bit) {
        const uint64_t cand = least | (1ull << bit);
        int            c = 0;
#pragma unroll
        for (int e = 0; e < E; ++e)
            c += __popcll(__ballot(bit >= 32 ? static_cast<uint32_t>(key[e] >> 32) >= static_cast<uint32_t>(cand >> 32) : key[e] >= cand));
        for (int j0 = CAP; j0 < n; j0 += 64 * NW) {
            const int j = j0 + static_cast<int>(threadIdx.x);
            c += __popcll(__ballot(j < n && ps_at(a, in, own, min(j, n - 1)) >= cand));
        }
        int total, none, b0, b1;
        all(c, 0, total, none, b0, b1);
        if (total >= take) least = cand;
        done = total == take;
    }
    // all above the least, and of those equal to it the first ones
    int above = 0, equal = 0, sa, se, ba, be;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        above += __popcll(__ballot(key[e] > least));
        equal += __popcll(__ballot(key[e] == least));
    }
    all(above, equal, sa, se, ba, be);
    int more = 0; // above, beyond what fits
    for (int j0 = CAP; j0 < n; j0 += 64 * NW) {
        const int j = j0 + static_cast<int>(threadIdx.x);
        more += __popcll(__ballot(j < n && ps_at(a, in, own, min(j, n - 1)) > least));
    }
    int sm, s0, b0, b1;
    all(more, 0, sm, s0, b0, b1);
    const int      room = take - sa - sm; // of the equal ones
    const uint64_t below = (1ull << lane) - 1;
    auto put = [&](bool gt, bool eq, int j, int &g, int &q) {
        const uint64_t mg = __ballot(gt), mq = __ballot(eq);
        const int      rq = q + __popcll(mq & below);
        if (gt || (eq && rq < room)) sel[g + __popcll(mg & below) + min(rq, room)] = row[j];
        g += __popcll(mg);
        q += __popcll(mq);
    };
    int g = ba, q = be;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        put(key[e] > least, key[e] == least, (wave * E + e) * 64 + lane, g, q);
    }
    int g0 = sa, q0 = se;
    for (int j0 = CAP; j0 < n; j0 += 64 * NW) {
        const int      j = j0 + static_cast<int>(threadIdx.x);
        const uint64_t x = ps_at(a, in, own, min(j, n - 1));
        const bool     gt = j < n && x > least, eq = j < n && x == least;
        int            tg, tq, wg, wq;
        all(__popcll(__ballot(gt)), __popcll(__ballot(eq)), tg, tq, wg, wq);
        int gg = g0 + wg, qq = q0 + wq;
        put(gt, eq, j, gg, qq);
        g0 += tg;
        q0 += tq;
    }
}

// Chunks: a workgroup for (tile of tokens, head), a wave a token.  The pages that any of the
// tile's tokens takes become one list in the order of the sequence, with a bit for each token
// that takes the page; sequence after sequence where the tile has tokens of several.
template <int E> __global__ __launch_bounds__(1024) void ps_choose_tile_kernel(PSArgs a) {
    __shared__ uint64_t bits[16][E]; // by token: pages 64 e + lane
    __shared__ int      seq[16], pages[16], sum[16];
    const int           tile = a.t0 / a.tiles.tokens + blockIdx.x / a.Hkv, h = blockIdx.x % a.Hkv, tt = a.tiles.tokens;
    const int           lane = threadIdx.x & 63, wave = threadIdx.x >> 6, t = tile * tt + wave;
    PSToken             s = {-1, -1, 0, 0, 0};
    if (t < a.T) s = ps_token(a, t);
    const bool some = s.b >= 0 && s.pos >= 0;
    const int  own = some ? s.pos / a.page : -1, n = own + 1, take = min(n, a.take);
    if (h == 0 && lane == 0 && t < a.T) {
        a.sel_lens[t]  = some ? (take - 1) * a.page + (s.pos - own * a.page) + 1 : 0;
        a.tiles.pos[t] = some ? s.pos : -1;
        a.sel_cu[t]    = t;
        if (t == a.T - 1) a.sel_cu[a.T] = a.T;
    }
    if (lane == 0) {
        seq[wave]   = some ? s.b : -1;
        pages[wave] = n;
    }
    uint64_t key[E];
    if (n > a.take) {
        const uint64_t *in = a.keys + (static_cast<int64_t>(t - a.t0) * a.Hkv + h) * a.M;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int j = e * 64 + lane;
            key[e]      = j < n ? ps_at(a, in, own, j) : 0;
        }
        const uint64_t least = ps_least<E>(key, take);
        int            above = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) above += __popcll(__ballot(key[e] > least));
        int room = take - above; // of the equal ones
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const uint64_t eq = __ballot(key[e] == least);
            const uint64_t m  = __ballot(key[e] > least || (key[e] == least && __popcll(eq & ((1ull << lane) - 1)) < room));
            room -= min(room, static_cast<int>(__popcll(eq)));
            if (lane == 0) bits[wave][e] = m;
        }
    } else {
        for (int e = lane; e < E; e += 64) bits[wave][e] = n >= 64 * (e + 1) ? ~0ull : n > 64 * e ? (1ull << (n - 64 * e)) - 1 : 0;
    }
    __syncthreads();
    const int64_t at = (static_cast<int64_t>(tile) * a.Hkv + h) * a.tiles.cap;
    int           count = 0;
    for (int i0 = 0; i0 < tt;) {
        const int b = seq[i0];
        int       i1 = i0 + 1;
        while (i1 < tt && seq[i1] == b) ++i1;
        if (b >= 0) {
            const int32_t *row = a.table + b * a.table_st;
            for (int j0 = 0; j0 < pages[i1 - 1]; j0 += 64 * tt) {
                const int j = j0 + static_cast<int>(threadIdx.x);
                uint32_t  mask = 0;
                if (j < 64 * E)
                    for (int i = i0; i < i1; ++i) mask |= static_cast<uint32_t>(bits[i][j >> 6] >> (j & 63) & 1) << i;
                const uint64_t m = __ballot(mask != 0);
                if (lane == 0) sum[wave] = __popcll(m);
                __syncthreads();
                int before = count + __popcll(m & ((1ull << lane) - 1));
                for (int w = 0; w < tt; ++w) {
                    if (w < wave) before += sum[w];
                    count += sum[w];
                }
                if (mask != 0) {
                    a.tiles.list[at + before]  = make_int2(row[j], j * a.page);
                    a.tiles.masks[at + before] = static_cast<uint16_t>(mask);
                }
                __syncthreads(); // the sums are read
            }
        }
        i0 = i1;
    }
    if (threadIdx.x == 0) a.tiles.counts[tile * a.Hkv + h] = count;
}

// Keys of a slice of tokens at most: 256 MB, or one token's
constexpr int64_t PS_SLICE = 256 << 20;
// a multiple of `tile` tokens
int64_t ps_slice(int64_t T, int64_t Hkv, int64_t M, int64_t tile) {
    return std::min<int64_t>(T, std::max<int64_t>(1, PS_SLICE / std::max<int64_t>(1, Hkv * M * 8) / tile) * tile);
}

} // namespace

size_t ps_workspace(int64_t T, int64_t Hkv, int64_t M, int64_t tile) { return static_cast<size_t>(ps_slice(T, Hkv, M, tile) * Hkv * M * 8); }

int ps_check(int64_t T, int64_t num_seqs, int64_t Hq, int64_t Hkv, int64_t D, int64_t num_pages, int64_t page_size, int64_t max_pages,
             int64_t take, int64_t first, int64_t last) {
    PTA_CHECK_ARG(T >= 0 && num_seqs >= 0 && num_pages >= 0 && page_size > 0 && max_pages >= 0, "bad sizes");
    PTA_CHECK_ARG(Hkv > 0 && Hq > 0 && Hq % Hkv == 0, "query heads (%lld) must be a multiple of cache heads (%lld)",
                  static_cast<long long>(Hq), static_cast<long long>(Hkv));
    PTA_CHECK_ARG(D >= 16 && D <= 256 && D % 16 == 0, "head_dim must be a multiple of 16 in [16, 256] (got %lld)", static_cast<long long>(D));
    PTA_CHECK_ARG(page_size <= INT_MAX && num_pages <= INT_MAX / page_size && num_pages * page_size <= INT_MAX / Hkv,
                  "the cache has 2^31 rows (pages * page_size * heads) or more");
    PTA_CHECK_ARG(max_pages <= (INT_MAX - 1024) / page_size, "page_table spans 2^31 tokens or more");
    PTA_CHECK_ARG(T <= (INT_MAX - 1024) / Hq && T < (1 << 24) && num_seqs < (1 << 24), "too many tokens or sequences");
    PTA_CHECK_ARG(first >= 0 && last >= 1 && first <= INT_MAX / 2 && last <= INT_MAX / 2 && take >= first + last && take <= INT_MAX / 2,
                  "num_selected must hold the first and the last pages, one of those at least");
    return PTA_OK;
}

// Scores go by tiles of tokens from two tokens a sequence on
static bool ps_tiles(const PSArgs &a) { return a.T >= 2 * a.B; }

template <int QT> static void ps_select_one(const PSArgs &a, hipStream_t st) {
    const unsigned grid = static_cast<unsigned>(a.n) * a.Hkv;
    if (a.D <= 64) ps_select_kernel<QT, 8><<<grid, 1024, 0, st>>>(a);
    else if (a.D <= 128) ps_select_kernel<QT, 16><<<grid, 1024, 0, st>>>(a);
    else ps_select_kernel<QT, 32><<<grid, 1024, 0, st>>>(a);
}

template <int QT> static void ps_score(const PSArgs &a, hipStream_t st) {
    const bool    tiles = ps_tiles(a);
    const int64_t items = (tiles ? cdiv(a.n, PS_TILE) : a.n) * a.Hkv;
    // pages in as many parts as give every CU four workgroups, one round of a workgroup at least
    const int64_t least = tiles ? 64 : 32, want = cdiv(4 * device_cu_count(), items);
    const int     per = static_cast<int>(std::max<int64_t>(least, cdiv(cdiv(a.M, want), least) * least)), parts = static_cast<int>(cdiv(a.M, per));
    const unsigned grid = static_cast<unsigned>(items * parts);
    if (tiles) {
        if (a.D <= 64) ps_score_tile_kernel<QT, 64><<<grid, PS_NT, 0, st>>>(a, per, parts);
        else if (a.D <= 128) ps_score_tile_kernel<QT, 128><<<grid, PS_NT, 0, st>>>(a, per, parts);
        else ps_score_tile_kernel<QT, 256><<<grid, PS_NT, 0, st>>>(a, per, parts);
    } else {
        if (a.D <= 64) ps_score_kernel<QT, 8><<<grid, PS_NT, 0, st>>>(a, per, parts);
        else if (a.D <= 128) ps_score_kernel<QT, 16><<<grid, PS_NT, 0, st>>>(a, per, parts);
        else ps_score_kernel<QT, 32><<<grid, PS_NT, 0, st>>>(a, per, parts);
    }
}

static int ps_launch(PSArgs a, int q_dtype, void *workspace, hipStream_t st) {
    a.keys = static_cast<uint64_t *>(workspace);
    const int tile = a.tiles.tokens, step = static_cast<int>(ps_slice(a.T, a.Hkv, a.M, std::max(1, tile)));
    for (a.t0 = 0; a.t0 < a.T; a.t0 += step) {
        a.n = std::min(step, a.T - a.t0);
        if (!ps_tiles(a) && a.M <= PS_ONE) {
            if (q_dtype == PTA_BF16) ps_select_one<PTA_BF16>(a, st);
            else ps_select_one<PTA_F16>(a, st);
            PTA_CHECK_LAUNCH();
            continue;
        }
        if (a.M > a.take) {
            if (q_dtype == PTA_BF16) ps_score<PTA_BF16>(a, st);
            else ps_score<PTA_F16>(a, st);
            PTA_CHECK_LAUNCH();
        }
        const unsigned grid = static_cast<unsigned>(tile > 0 ? cdiv(a.n, tile) : a.n) * a.Hkv, threads = 64 * tile;
        if (tile > 0) {
            if (a.M <= 256) ps_choose_tile_kernel<4><<<grid, threads, 0, st>>>(a);
            else if (a.M <= 512) ps_choose_tile_kernel<8><<<grid, threads, 0, st>>>(a);
            else if (a.M <= 1024) ps_choose_tile_kernel<16><<<grid, threads, 0, st>>>(a);
            else ps_choose_tile_kernel<32><<<grid, threads, 0, st>>>(a);
        } else if (a.M <= 256) ps_choose_kernel<4><<<grid, 64, 0, st>>>(a);
        else if (a.M <= 512) ps_choose_kernel<8><<<grid, 64, 0, st>>>(a);
        else if (a.M <= 2048) ps_choose_many_kernel<8, 4><<<grid, 512, 0, st>>>(a);
        else ps_choose_many_kernel<16, 8><<<grid, 1024, 0, st>>>(a);
        PTA_CHECK_LAUNCH();
    }
    return PTA_OK;
}

} // namespace pta

using namespace pta;

extern "C" int pta_kv_page_ranges(const void *k_cache, int cache_kind, int is_f16, int64_t num_pages, int64_t page_size, int64_t Hkv, int64_t D,
                                  const float *k_scale_inv, const int32_t *page_table, int64_t table_stride, int64_t max_pages,
                                  const int32_t *cu_seqlens_q, const int32_t *seq_lens, int64_t num_seqs, void *key_ranges,
                                  pta_stream_t stream) {
    clear_error();
    PTA_CHECK_ARG(cache_kind == PTA_E4M3 || cache_kind == PTA_E5M2 || cache_kind == PTA_CACHE_16BIT, "unknown cache kind %d", cache_kind);
    if (int rc = ps_check(0, num_seqs, Hkv, Hkv, D, num_pages, page_size, max_pages, 1, 0, 1)) return rc;
    if (num_seqs == 0 || num_pages == 0 || max_pages == 0) return PTA_OK;
    PTA_CHECK_ARG(k_cache && page_table && cu_seqlens_q && seq_lens && key_ranges, "null pointer");
    PTA_CHECK_ARG(aligned16(k_cache) && aligned16(key_ranges), "cache pools must be 16-byte aligned");
    PTA_CHECK_ARG(cache_kind == PTA_CACHE_16BIT || k_scale_inv, "an fp8 cache needs its scales");
    PTA_CHECK_ARG(num_seqs <= INT_MAX / 4 / Hkv, "too many sequences");
    PRArgs a = {};
    a.kc = static_cast<const uint8_t *>(k_cache); a.ks = k_scale_inv;
    a.table = page_table; a.table_st = table_stride; a.cu = cu_seqlens_q; a.lens = seq_lens;
    a.ranges = static_cast<uint16_t *>(key_ranges);
    a.B = static_cast<int>(num_seqs); a.Hkv = static_cast<int>(Hkv); a.D = static_cast<int>(D);
    a.M = static_cast<int>(max_pages); a.P = static_cast<int>(num_pages); a.page = static_cast<int>(page_size);
    // the host does not know how many pages hold new tokens: four workgroups a CU share them
    a.parts = static_cast<int>(std::min<int64_t>(max_pages, cdiv(4 * device_cu_count(), num_seqs * Hkv)));
    const unsigned    grid = static_cast<unsigned>(num_seqs * Hkv * a.parts);
    const hipStream_t st = as_stream(stream);
#define PTA_PR(KIND)                                                                               \
    do {                                                                                           \
        if (D <= 64) pr_ranges_kernel<KIND, 16><<<grid, PS_NT, 0, st>>>(a);                        \
        else if (D <= 128) pr_ranges_kernel<KIND, 32><<<grid, PS_NT, 0, st>>>(a);                  \
        else pr_ranges_kernel<KIND, 64><<<grid, PS_NT, 0, st>>>(a);                                \
    } while (0)
    if (cache_kind == PTA_E4M3) PTA_PR(PTA_E4M3);
    else if (cache_kind == PTA_E5M2) PTA_PR(PTA_E5M2);
    else if (!is_f16) PTA_PR(PTA_CACHE_16BIT);
    else PTA_PR(PTA_CACHE_16BIT + 1);
#undef PTA_PR
    PTA_CHECK_LAUNCH();
    return PTA_OK;
}

extern "C" size_t pta_select_pages_workspace_size(int64_t num_tokens, int64_t Hkv, int64_t max_pages) {
    if (num_tokens <= 0 || Hkv <= 0 || max_pages <= 0) return 0;
    return ps_workspace(num_tokens, Hkv, max_pages, 1);
}

namespace pta {
int ps_select(const void *q, int q_dtype, int64_t num_tokens, int64_t Hq, int64_t D, int64_t q_stride_t, int64_t q_stride_h,
              const void *key_ranges, int64_t num_pages, int64_t page_size, int64_t Hkv, const int32_t *page_table, int64_t table_stride,
              int64_t max_pages, const int32_t *cu_seqlens_q, const int32_t *seq_lens, int64_t num_seqs, int64_t num_selected,
              int64_t num_first, int64_t num_last, int32_t *selected, const PSTiles *tiles, int32_t *selected_lens, int32_t *selected_cu,
              void *workspace, hipStream_t st) {
    PTA_CHECK_ARG(q_dtype == PTA_BF16 || q_dtype == PTA_F16, "queries must be bfloat16 or float16 (type %d)", q_dtype);
    if (int rc = ps_check(num_tokens, num_seqs, Hq, Hkv, D, num_pages, page_size, max_pages, num_selected, num_first, num_last)) return rc;
    if (num_tokens == 0) return PTA_OK;
    PTA_CHECK_ARG(num_seqs > 0, "tokens without a sequence");
    PTA_CHECK_ARG(q && cu_seqlens_q && seq_lens && selected_lens && (max_pages == 0 || (page_table && (selected || tiles))) && (num_pages == 0 || key_ranges),
                  "null pointer");
    PTA_CHECK_ARG(aligned16(q) && aligned16(key_ranges) && q_stride_t % 8 == 0 && q_stride_h % 8 == 0,
                  "queries and ranges must be 16-byte aligned, with strides of multiples of 8 elements");
    PSArgs a = {};
    a.q = static_cast<const uint16_t *>(q); a.q_st = q_stride_t; a.q_sh = q_stride_h;
    a.ranges = static_cast<const uint16_t *>(key_ranges);
    a.table = page_table; a.table_st = table_stride; a.cu = cu_seqlens_q; a.lens = seq_lens;
    if (tiles != nullptr) a.tiles = *tiles;
    a.sel = selected; a.sel_lens = selected_lens; a.sel_cu = selected_cu;
    a.T = static_cast<int>(num_tokens); a.B = static_cast<int>(num_seqs); a.Hq = static_cast<int>(Hq); a.Hkv = static_cast<int>(Hkv);
    a.G = static_cast<int>(Hq / Hkv); a.D = static_cast<int>(D); a.M = static_cast<int>(max_pages); a.P = static_cast<int>(num_pages);
    a.page = static_cast<int>(page_size);
    a.take = static_cast<int>(num_selected); a.first = static_cast<int>(num_first); a.last = static_cast<int>(num_last);
    a.K = static_cast<int>(std::min(num_selected, max_pages));
    return ps_launch(a, q_dtype, workspace, st);
}
} // namespace pta

extern "C" int pta_select_pages(const void *q, int q_dtype, int64_t num_tokens, int64_t Hq, int64_t D, int64_t q_stride_t, int64_t q_stride_h,
                                const void *key_ranges, int64_t num_pages, int64_t page_size, int64_t Hkv, const int32_t *page_table,
                                int64_t table_stride, int64_t max_pages, const int32_t *cu_seqlens_q, const int32_t *seq_lens,
                                int64_t num_seqs, int64_t num_selected, int64_t num_first, int64_t num_last, int32_t *selected,
                                int32_t *selected_lens, void *workspace, size_t workspace_bytes, pta_stream_t stream) {
    clear_error();
    const size_t need = pta_select_pages_workspace_size(num_tokens, Hkv, max_pages);
    PTA_CHECK_ARG(need == 0 || (workspace && aligned16(workspace) && workspace_bytes >= need), "workspace too small: %zu bytes needed, %zu given",
                  need, workspace_bytes);
    return ps_select(q, q_dtype, num_tokens, Hq, D, q_stride_t, q_stride_h, key_ranges, num_pages, page_size, Hkv, page_table, table_stride,
                     max_pages, cu_seqlens_q, seq_lens, num_seqs, num_selected, num_first, num_last, selected, nullptr, selected_lens, nullptr,
                     workspace, as_stream(stream));
}
