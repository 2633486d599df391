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
// sum turns G products of 2 D into one.  It is computed in 64 bits, where the order of
// the sum does not show: the choice is the same whatever the launch's shape, and ties
// are what the formula says they are.  A NaN counts as +inf: pages with NaN are
// attended, and show.  The first `first` and the last `last` pages of those that a
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
    int32_t        *sel;     // [T, Hkv, K] pages of the pool, rising in the sequence; -1 behind the last
    int32_t        *sel_lens; // [T] keys of them that the token sees
    int32_t        *sel_cu;  // [T + 1] 0, 1, 2, ... (may be null)
    int             T, B, Hq, Hkv, G, D, M, P, page;
    int             take, first, last, K;
    int             t0, n;   // the slice
};


// The token's sequence by bisection, and its place in it; b < 0: it has none.
struct PSToken {
    int b, pos, len, n, i;
};
__device__ __forceinline__ PSToken ps_token(const int32_t *cu, const int32_t *lens, int B, int T, int t, int64_t most) {
    PSToken s = {-1, -1, 0, 0, 0};
    int     lo = 0, hi = B; // the last b with cu[b] <= t
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (cu[mid] <= t) lo = mid;
        else hi = mid;
    }
    const int tok0 = min(max(cu[lo], 0), T), end = min(max(cu[lo + 1], tok0), T);
    if (B <= 0 || t < tok0 || t >= end) return s;
    s.b   = lo;
    s.n   = end - tok0;
    s.i   = t - tok0;
    s.len = static_cast<int>(min(static_cast<int64_t>(max(lens[lo], 0)), most));
    s.pos = s.len - s.n + s.i;
    return s;
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
// thread has 4 channels of every GROUPS-th key, NL threads a key.
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

// Pages [c per, (c + 1) per) of token t for head h; 8 channels a lane
template <int QT, int LPR> __global__ __launch_bounds__(PS_NT) void ps_score_kernel(PSArgs a, int per, int parts) {
    constexpr int  GROUPS = PS_NT / LPR, PAGES = 4;
    const uint32_t w = blockIdx.x, h = w % a.Hkv, w1 = w / a.Hkv, c = w1 % parts, ti = w1 / parts;
    const int      t = a.t0 + static_cast<int>(ti);
    const PSToken  s = ps_token(a.cu, a.lens, a.B, a.T, t, static_cast<int64_t>(a.M) * a.page);
    if (s.b < 0 || s.pos < 0) return;
    const int own = s.pos / a.page, n = own + 1, j0 = c * per, j1 = min(j0 + per, n);
    if (j0 >= j1 || n <= a.take) return;
    const int  l = threadIdx.x % LPR, g = threadIdx.x / LPR, d = l * 8;
    const bool in = d < a.D;
    double     up[8], down[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) up[e] = down[e] = 0.0;
    if (in)
        for (int i = 0; i < a.G; ++i) {
            float v[8];
            load8<QT>(a.q, t * a.q_st + (h * a.G + i) * a.q_sh + d, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                // both for a NaN: it has to reach the score
                up[e] += v[e] > 0.0f || v[e] != v[e] ? v[e] : 0.0f;
                down[e] += v[e] < 0.0f || v[e] != v[e] ? v[e] : 0.0f;
            }
        }
    uint64_t      *out = a.keys + (static_cast<int64_t>(ti) * a.Hkv + h) * a.M;
    const int32_t *row = a.table + s.b * a.table_st;
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
            if (l == 0 && j < j1) out[j] = j < a.first || own - j < a.last ? ~0ull : ps_key(x);
        }
    }
}

// ---- choice ------------------------------------------------------------------------
// NW waves for (token, head), wave w with keys [64 w E, 64 (w + 1) E), E a lane; what
// does not fit is read again for every step.  The bits of the least key that is taken
// are found from the highest on: a bit is set if at least `take` keys have it.
template <int NW, int E> __global__ __launch_bounds__(64 * NW) void ps_choose_kernel(PSArgs a) {
    constexpr int  CAP = 64 * NW * E;
    __shared__ int cnt[2][2][NW];
    const int      ti = blockIdx.x / a.Hkv, h = blockIdx.x - ti * a.Hkv, t = a.t0 + ti;
    const int      lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const PSToken  s = ps_token(a.cu, a.lens, a.B, a.T, t, static_cast<int64_t>(a.M) * a.page);
    const bool     some = s.b >= 0 && s.pos >= 0;
    const int      n = some ? s.pos / a.page + 1 : 0, take = min(n, a.take);
    int32_t       *sel = a.sel + (static_cast<int64_t>(t) * a.Hkv + h) * a.K;
    if (h == 0 && threadIdx.x == 0) {
        a.sel_lens[t] = some ? (take - 1) * a.page + s.pos % a.page + 1 : 0;
        if (a.sel_cu != nullptr) {
            a.sel_cu[t] = t;
            if (t == a.T - 1) a.sel_cu[a.T] = a.T;
        }
    }
    for (int j = take + static_cast<int>(threadIdx.x); j < a.K; j += 64 * NW) sel[j] = -1;
    if (!some) return;
    const int32_t *row = a.table + s.b * a.table_st;
    if (n <= a.take) {
        for (int j = threadIdx.x; j < n; j += 64 * NW) sel[j] = row[j];
        return;
    }
    const uint64_t *in = a.keys + (static_cast<int64_t>(ti) * a.Hkv + h) * a.M;
    uint64_t        key[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int j = (wave * E + e) * 64 + lane;
        key[e]      = j < n ? in[j] : 0; // below every score: `least` is at least 1
    }
    // keys of the workgroup for which f holds, and g
    int  buf = 0;
    auto all = [&](int x, int y, int &sx, int &sy, int &bx, int &by) {
        sx = x;
        sy = y;
        bx = by = 0;
        if constexpr (NW > 1) {
            if (lane == 0) {
                cnt[buf][0][wave] = x;
                cnt[buf][1][wave] = y;
            }
            __syncthreads();
            sx = sy = 0;
            for (int w = 0; w < NW; ++w) {
                if (w < wave) {
                    bx += cnt[buf][0][w];
                    by += cnt[buf][1][w];
                }
                sx += cnt[buf][0][w];
                sy += cnt[buf][1][w];
            }
            buf ^= 1;
        }
    };
    uint64_t least = 0;
    for (int bit = 63; bit >= 0; --bit) {
        const uint64_t cand = least | (1ull << bit);
        int            c = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) c += __popcll(__ballot(key[e] >= cand));
        for (int j0 = CAP; j0 < n; j0 += 64 * NW) {
            const int j = j0 + static_cast<int>(threadIdx.x);
            c += __popcll(__ballot(j < n && in[min(j, n - 1)] >= cand));
        }
        int total, none, b0, b1;
        all(c, 0, total, none, b0, b1);
        if (total >= take) least = cand;
        if (total == take) break; // all of these and no others
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
        more += __popcll(__ballot(j < n && in[min(j, n - 1)] > least));
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
        const int j = (wave * E + e) * 64 + lane;
        put(j < n && key[e] > least, j < n && key[e] == least, j, g, q);
    }
    int g0 = sa, q0 = se;
    for (int j0 = CAP; j0 < n; j0 += 64 * NW) {
        const int      j = j0 + static_cast<int>(threadIdx.x);
        const uint64_t x = in[min(j, n - 1)];
        const bool     gt = j < n && x > least, eq = j < n && x == least;
        int            tg, tq, wg, wq;
        all(__popcll(__ballot(gt)), __popcll(__ballot(eq)), tg, tq, wg, wq);
        int gg = g0 + wg, qq = q0 + wq;
        put(gt, eq, j, gg, qq);
        g0 += tg;
        q0 += tq;
    }
}

// Keys of a slice of tokens at most: 256 MB, or one token's
constexpr int64_t PS_SLICE = 256 << 20;
int64_t ps_slice(int64_t T, int64_t Hkv, int64_t M) { return std::max<int64_t>(1, std::min<int64_t>(T, PS_SLICE / std::max<int64_t>(1, Hkv * M * 8))); }

} // namespace

size_t ps_workspace(int64_t T, int64_t Hkv, int64_t M) { return static_cast<size_t>(ps_slice(T, Hkv, M) * Hkv * M * 8); }

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

template <int QT> static void ps_score(const PSArgs &a, hipStream_t st) {
    // pages in as many parts as give every CU four workgroups, 32 of them at least
    const int64_t want = cdiv(4 * device_cu_count(), static_cast<int64_t>(a.n) * a.Hkv);
    const int     per = static_cast<int>(std::max<int64_t>(32, cdiv(cdiv(a.M, want), 32) * 32)), parts = static_cast<int>(cdiv(a.M, per));
    const unsigned grid = static_cast<unsigned>(static_cast<int64_t>(a.n) * a.Hkv * parts);
    if (a.D <= 64) ps_score_kernel<QT, 8><<<grid, PS_NT, 0, st>>>(a, per, parts);
    else if (a.D <= 128) ps_score_kernel<QT, 16><<<grid, PS_NT, 0, st>>>(a, per, parts);
    else ps_score_kernel<QT, 32><<<grid, PS_NT, 0, st>>>(a, per, parts);
}

static int ps_launch(PSArgs a, int q_dtype, void *workspace, hipStream_t st) {
    a.keys = static_cast<uint64_t *>(workspace);
    const int step = static_cast<int>(ps_slice(a.T, a.Hkv, a.M));
    for (a.t0 = 0; a.t0 < a.T; a.t0 += step) {
        a.n = std::min(step, a.T - a.t0);
        if (a.M > a.take) {
            if (q_dtype == PTA_BF16) ps_score<PTA_BF16>(a, st);
            else ps_score<PTA_F16>(a, st);
            PTA_CHECK_LAUNCH();
        }
        const unsigned grid = static_cast<unsigned>(a.n) * a.Hkv;
        if (a.M <= 512) ps_choose_kernel<1, 8><<<grid, 64, 0, st>>>(a);
        else if (a.M <= 2048) ps_choose_kernel<4, 8><<<grid, 256, 0, st>>>(a);
        else ps_choose_kernel<16, 8><<<grid, 1024, 0, st>>>(a);
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
    return ps_workspace(num_tokens, Hkv, max_pages);
}

namespace pta {
int ps_select(const void *q, int q_dtype, int64_t num_tokens, int64_t Hq, int64_t D, int64_t q_stride_t, int64_t q_stride_h,
              const void *key_ranges, int64_t num_pages, int64_t page_size, int64_t Hkv, const int32_t *page_table, int64_t table_stride,
              int64_t max_pages, const int32_t *cu_seqlens_q, const int32_t *seq_lens, int64_t num_seqs, int64_t num_selected,
              int64_t num_first, int64_t num_last, int32_t *selected, int32_t *selected_lens, int32_t *selected_cu, void *workspace,
              hipStream_t st) {
    PTA_CHECK_ARG(q_dtype == PTA_BF16 || q_dtype == PTA_F16, "queries must be bfloat16 or float16 (type %d)", q_dtype);
    if (int rc = ps_check(num_tokens, num_seqs, Hq, Hkv, D, num_pages, page_size, max_pages, num_selected, num_first, num_last)) return rc;
    if (num_tokens == 0) return PTA_OK;
    PTA_CHECK_ARG(num_seqs > 0, "tokens without a sequence");
    PTA_CHECK_ARG(q && cu_seqlens_q && seq_lens && selected_lens && (max_pages == 0 || (page_table && selected)) && (num_pages == 0 || key_ranges),
                  "null pointer");
    PTA_CHECK_ARG(aligned16(q) && aligned16(key_ranges) && q_stride_t % 8 == 0 && q_stride_h % 8 == 0,
                  "queries and ranges must be 16-byte aligned, with strides of multiples of 8 elements");
    PSArgs a = {};
    a.q = static_cast<const uint16_t *>(q); a.q_st = q_stride_t; a.q_sh = q_stride_h;
    a.ranges = static_cast<const uint16_t *>(key_ranges);
    a.table = page_table; a.table_st = table_stride; a.cu = cu_seqlens_q; a.lens = seq_lens;
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
                     max_pages, cu_seqlens_q, seq_lens, num_seqs, num_selected, num_first, num_last, selected, selected_lens, nullptr,
                     workspace, as_stream(stream));
}
