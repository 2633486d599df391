// Attention of new tokens over a paged cache: the kernels.
//
// Token i of the n new ones of a sequence of length L (with them) sits at
// position t = L - n + i and sees the keys j <= t, under a window only those
// with t - j < window or j < sinks:
//
//   o = sum_j softmax_j(scale * q.k_j) v_j,   lse = ln sum_j exp(scale * q.k_j)
//
// with k_j = ks_j k8_j and v_j = vs_j v8_j for an fp8 cache.  The scales never
// touch the elements: fp8 converts exactly to the queries' 16-bit type, and
// with the base-2 logits of the scaled values
//
//   u_j = (q.k8_j) * (scale * log2(e) * ks_j) + log2(vs_j),   m = max_j u_j,
//   p_j = 2^(u_j - m):   l = sum_j p_j / vs_j,   O = sum_j p_j v8_j,   o = O / l
//
// P stays in [0, 1] however large or small the scales are, which fp16 needs,
// and is rounded once, to the 16 bits that the matrix instructions take;
// logits, m, l and O are fp32.
//
// The query heads of one key / value head are rows of one matrix, r = i * G + g
// (G = Hq / Hkv), so a key is read once for all of them.  Both products are
// computed transposed: S^T = K Q^T has keys as rows and queries as columns, so
// the softmax statistics of a query are values of one lane (its column), and
// the registers of S^T are the operand of O^T = V^T P^T as they are: the
// contraction runs over the keys in the order in which S^T holds them, and V
// comes from LDS through the transposing read in that order.
//
// Two kernels share this: the wide one (32 rows a wave, keys and values staged
// in LDS for all waves) where there are many rows, the narrow one (16 rows,
// keys straight into registers, every wave on keys of its own) where there are
// few and the cache's bytes bound the call.  The keys of a row tile may be split
// over several workgroups; a last kernel joins their parts.
#pragma once

#include <climits>

#include "common.h"

namespace pta {

constexpr int ATT_NONE = INT_MIN; // desc of a slot without work

struct AttnArgs {
    const uint16_t *q;
    int64_t         q_st, q_sh;
    const uint8_t  *kc, *vc;
    const float    *ks, *vs;
    const int32_t  *table;
    int64_t         table_st;
    const int32_t  *cu, *lens;
    uint16_t       *out; // [Tq, Hq, D]
    float          *lse; // [Tq, Hq] or null
    float          *part_o;  // [slots, Hkv, BQ, D]
    float2         *part_ml; // [slots, Hkv, BQ]
    int4           *desc;    // [slots]: sequence, row tile, chunk, chunks
    int             B, Tq, Hq, Hkv, G, D;
    int             num_pages, page, max_pages;
    int             window, sinks; // window 0: none
    float           scale_log2;
    int             slots;      // work items per key / value head that the grid holds
    int             split_goal; // 0: row tiles are never split
    int             min_chunk;  // in key tiles
};

typedef float    att_f4 __attribute__((ext_vector_type(4)));
typedef float    att_f16 __attribute__((ext_vector_type(16)));
typedef short    att_s4 __attribute__((ext_vector_type(4)));
typedef __bf16   att_b8 __attribute__((ext_vector_type(8)));
typedef __bf16   att_b2 __attribute__((ext_vector_type(2)));
typedef _Float16 att_h8 __attribute__((ext_vector_type(8)));
typedef _Float16 att_h2 __attribute__((ext_vector_type(2)));

// ---- the queries' type: matrix instructions, packing, exact fp8 conversion ----
template <int QT> struct AttT;
template <> struct AttT<PTA_BF16> {
    static __device__ __forceinline__ att_f16 mfma32(uint4 a, uint4 b, att_f16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(att_b8, a), __builtin_bit_cast(att_b8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ att_f4 mfma16(uint4 a, uint4 b, att_f4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(att_b8, a), __builtin_bit_cast(att_b8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float x, float y) {
        att_b2 r;
        r[0] = static_cast<__bf16>(x);
        r[1] = static_cast<__bf16>(y);
        return __builtin_bit_cast(uint32_t, r);
    }
    template <int KIND> static __device__ __forceinline__ uint2 from_fp8(uint32_t w) {
        if constexpr (KIND == PTA_E4M3)
            return make_uint2(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false)),
                              __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true)));
        else
            return make_uint2(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w, 1.0f, false)),
                              __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w, 1.0f, true)));
    }
};
template <> struct AttT<PTA_F16> {
    static __device__ __forceinline__ att_f16 mfma32(uint4 a, uint4 b, att_f16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(att_h8, a), __builtin_bit_cast(att_h8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ att_f4 mfma16(uint4 a, uint4 b, att_f4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(att_h8, a), __builtin_bit_cast(att_h8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float x, float y) {
        att_h2 r;
        r[0] = static_cast<_Float16>(x);
        r[1] = static_cast<_Float16>(y);
        return __builtin_bit_cast(uint32_t, r);
    }
    template <int KIND> static __device__ __forceinline__ uint2 from_fp8(uint32_t w) {
        if constexpr (KIND == PTA_E4M3)
            return make_uint2(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false)),
                              __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true)));
        else
            return make_uint2(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_bf8(w, 1.0f, false)),
                              __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_bf8(w, 1.0f, true)));
    }
};

// 8 cache elements as 8 values of the queries' type
template <int QT, int KIND> __device__ __forceinline__ uint4 att_cvt8(uint32_t lo, uint32_t hi) {
    const uint2 a = AttT<QT>::template from_fp8<KIND>(lo), b = AttT<QT>::template from_fp8<KIND>(hi);
    return make_uint4(a.x, a.y, b.x, b.y);
}

// 4 x 16-bit transposed LDS read: within 16 lanes, lane i addresses elements
// 4 (i % 4) .. + 3 of row i / 4 and receives column i of the four rows.
__device__ __forceinline__ uint2 att_tr16(const uint16_t *p) {
    typedef __attribute__((address_space(3))) att_s4 lds_s4;
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_s4 *)reinterpret_cast<att_s4 *>(const_cast<uint16_t *>(p))));
}

__device__ __forceinline__ float att_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float att_log2(float x) { return __builtin_amdgcn_logf(x); }

// sum(v, v of lane ^ 16), sum(v, v of lane ^ 32): see max_xor16 / max_xor32
__device__ __forceinline__ float add_xor16(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float add_xor32(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// ---------------------------------------------------------------------------
// work items
// ---------------------------------------------------------------------------
// One item: the rows of row tile `tile` of sequence b against keys number
// [t0, t1) of the tile's list of key tiles (t0 == t1: none).  The list of a row
// tile: key tiles [0, n_sink), then those from lo_tile on.
struct AttnItem {
    int b, tile, chunk, chunks; // b < 0: no work
    int row0, rows;             // rows [row0, row0 + rows) of the sequence
    int tok0;                   // first new token of the sequence in q
    int pos0;                   // position of the sequence's token 0
    int kend;                   // keys [0, kend): seen by some row, or hidden by the window only
    int lo;                     // first key inside the window of some row
    int n_sink, lo_tile;
    int t0, t1;
};

struct AttnSeq {
    int n, len, tok0; // new tokens, length, first token; n = 0: none
};

// Lengths of a sequence, held inside what the tensors have room for.
__device__ __forceinline__ AttnSeq attn_seq(const AttnArgs &a, int b) {
    AttnSeq s;
    s.tok0        = min(max(a.cu[b], 0), a.Tq);
    const int end = min(max(a.cu[b + 1], s.tok0), a.Tq);
    s.n           = end - s.tok0;
    s.len         = static_cast<int>(min(static_cast<int64_t>(max(a.lens[b], 0)),
                                         static_cast<int64_t>(a.max_pages) * a.page));
    return s;
}

// Key tiles that a row tile of this sequence goes through at most.
template <int KT> __device__ __forceinline__ int attn_tiles(const AttnArgs &a, const AttnSeq &s, int bq) {
    const int full = (s.len + KT - 1) / KT;
    if (a.window <= 0) return full;
    const int64_t span = static_cast<int64_t>(a.window) + bq / a.G + 1;
    const int64_t win  = span / KT + 2 + (min(a.sinks, s.len) + KT - 1) / KT;
    return static_cast<int>(min(static_cast<int64_t>(full), win));
}

// Finds the item of slot `slot`; all threads of the workgroup call it (`red`:
// 2 * 8 words of LDS).  Items are numbered sequence by sequence, row tile by row
// tile, chunk by chunk; a chunk is `C` key tiles, C such that all items of a
// head fit the grid: sum over the row tiles of ceil(k / C) <= sum(k) / C + tiles.
template <int BQ, int KT, int NTHR> __device__ AttnItem attn_find(const AttnArgs &a, int slot, uint32_t *red) {
    constexpr int NW = NTHR / 64;
    const int     tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    auto scan = [&](uint32_t v, uint32_t &total) -> uint32_t { // inclusive prefix sum over the workgroup
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t o = __shfl_up(v, d);
            if (lane >= d) v += o;
        }
        __syncthreads();
        if (lane == 63) red[wave] = v;
        __syncthreads();
        uint32_t before = 0;
        total           = 0;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            if (w < wave) before += red[w];
            total += red[w];
        }
        return v + before;
    };
    AttnItem it;
    it.b    = -1;
    int   C = INT_MAX;
    if (a.split_goal > 0) {
        // sums past 32 bits only make C larger than needed: in floating point
        float w = 0.0f;
        for (int b0 = 0; b0 < a.B; b0 += NTHR) {
            const int b = b0 + tid;
            if (b < a.B) {
                const AttnSeq s = attn_seq(a, b);
                const float   r = static_cast<float>((static_cast<int64_t>(s.n) * a.G + BQ - 1) / BQ);
                w += r * static_cast<float>(attn_tiles<KT>(a, s, BQ));
            }
        }
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) w += __shfl_xor(w, d);
        if (lane == 0) red[8 + wave] = __float_as_uint(w);
        __syncthreads();
        w = 0.0f;
#pragma unroll
        for (int i = 0; i < NW; ++i) w += __uint_as_float(red[8 + i]);
        // above the quotient by more than the sum's rounding: the grid holds all items
        C = max(a.min_chunk, static_cast<int>(fminf(w * 1.001f / static_cast<float>(a.split_goal), 1e9f)) + 1);
    }
    uint32_t seen = 0;
    for (int b0 = 0; b0 < a.B; b0 += NTHR) {
        const int b = b0 + tid;
        AttnSeq   s = {0, 0, 0};
        uint32_t  tiles = 0, chunks = 1;
        if (b < a.B) {
            s      = attn_seq(a, b);
            tiles  = static_cast<uint32_t>((static_cast<int64_t>(s.n) * a.G + BQ - 1) / BQ);
            const int k = attn_tiles<KT>(a, s, BQ);
            chunks      = k > C ? (k - 1) / C + 1 : 1;
        }
        uint32_t       total;
        const uint32_t mine = tiles * chunks;
        const uint32_t incl = scan(mine, total);
        if (static_cast<uint32_t>(slot) < seen + total) {
            const uint32_t at = static_cast<uint32_t>(slot) - seen;
            __syncthreads();
            if (at < incl && at >= incl - mine) {
                red[0] = b;
                red[1] = at - (incl - mine);
                red[2] = chunks;
            }
            __syncthreads();
            it.b      = static_cast<int>(red[0]);
            it.chunks = static_cast<int>(red[2]);
            it.tile   = static_cast<int>(red[1]) / it.chunks;
            it.chunk  = static_cast<int>(red[1]) - it.tile * it.chunks;
            break;
        }
        seen += total;
    }
    if (it.b < 0) return it;
    const AttnSeq s = attn_seq(a, it.b);
    it.tok0 = s.tok0;
    it.pos0 = s.len - s.n; // below 0 where more tokens came than the length says: those see nothing
    it.row0 = it.tile * BQ;
    it.rows = min(BQ, s.n * a.G - it.row0);
    const int pmin = it.pos0 + it.row0 / a.G, pmax = it.pos0 + (it.row0 + it.rows - 1) / a.G;
    it.kend = max(0, min(pmax + 1, s.len));
    it.lo   = a.window > 0 ? max(0, pmin - a.window + 1) : 0;
    it.lo   = min(it.lo, it.kend);
    // sink tiles that the window's tiles do not cover
    const int first = it.lo / KT, last = (it.kend + KT - 1) / KT;
    it.n_sink  = min(a.window > 0 ? (min(a.sinks, it.kend) + KT - 1) / KT : 0, first);
    it.lo_tile = first;
    const int n = it.n_sink + max(0, last - first);
    const int64_t c0 = static_cast<int64_t>(it.chunk) * C;
    it.t0 = static_cast<int>(min(c0, static_cast<int64_t>(n)));
    it.t1 = it.chunk == it.chunks - 1 ? n : static_cast<int>(min(c0 + C, static_cast<int64_t>(n)));
    return it;
}

__device__ __forceinline__ int attn_key0(const AttnItem &it, int t, int KT) {
    return (t < it.n_sink ? t : it.lo_tile + t - it.n_sink) * KT;
}

// Pool row of key j for head h (row = (page * Hkv + h) * page_size + offset), or
// -1 where there is none: past the keys, hidden from every row by the window, or
// on a page outside the pool.
__device__ __forceinline__ int attn_key_row(const AttnArgs &a, const AttnItem &it, int h, int j) {
    if (j >= it.kend || (j < it.lo && j >= a.sinks)) return -1;
    const uint32_t p  = static_cast<uint32_t>(j) / static_cast<uint32_t>(a.page);
    const int      pg = a.table[it.b * a.table_st + p];
    if (pg < 0 || pg >= a.num_pages) return -1;
    return (pg * a.Hkv + h) * a.page + (j - static_cast<int>(p) * a.page);
}

// ---------------------------------------------------------------------------
// wide kernel: NW waves of 32 rows, key tiles of 64 in LDS
// ---------------------------------------------------------------------------
template <int QT, int KIND, int DP, int NW>
__global__ __launch_bounds__(NW * 64, DP > 128 ? 1 : 2) void attn_wide_kernel(AttnArgs a) {
    constexpr int  KT = 64, BQ = 32 * NW, NT = NW * 64;
    constexpr bool FP8 = KIND != PTA_CACHE_16BIT;
    constexpr int  ES  = FP8 ? 1 : 2;       // bytes of a cache element
    constexpr int  EC  = 16 / ES;           // elements of a 16-byte piece
    constexpr int  CPR = DP / EC;           // pieces of a row
    constexpr int  NP  = KT * CPR / NT;     // pieces of a thread and pool
    constexpr int  KC  = DP / 8;            // 16-byte pieces of a staged row
    constexpr int  VS  = DP + 32;           // elements of a staged value row: the transposed read's 8 rows
                                            // of 64 bytes then fall into different banks
    static_assert(KT * CPR % NT == 0, "pieces");
    __shared__ __align__(16) uint16_t sk[2][KT * DP];
    __shared__ __align__(16) uint16_t sv[2][KT * VS];
    __shared__ __align__(16) float    ssc[FP8 ? 2 : 1][3][FP8 ? KT : 4];
    __shared__ int                    srow[2][KT];
    __shared__ uint32_t               red[16];

    const int      tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int      h    = blockIdx.x % a.Hkv;
    const int      slot = blockIdx.x / a.Hkv;
    const AttnItem it   = attn_find<BQ, KT, NT>(a, slot, red);
    if (a.desc != nullptr && h == 0 && tid == 0)
        a.desc[slot] = it.b < 0 ? make_int4(ATT_NONE, 0, 0, 0) : make_int4(it.b, it.tile, it.chunk, it.chunks);
    if (it.b < 0) return;

    const int  c = lane & 31, half = lane >> 5;
    const int  r     = it.row0 + wave * 32 + c; // this lane's row
    const bool rin   = r < it.row0 + it.rows;
    const int  rtok  = rin ? r / a.G : 0;
    const int  tok   = it.tok0 + rtok;
    const int  hq    = h * a.G + (rin ? r - rtok * a.G : 0);
    const int  pos   = rin ? it.pos0 + rtok : -1; // rows past the tile see nothing
    const int  wlo   = a.window > 0 ? pos - a.window + 1 : INT_MIN;
    // positions of the wave's rows, for whole tiles that need no mask
    const int  wrow  = it.row0 + wave * 32;
    const int  wend  = min(wrow + 32, it.row0 + it.rows);
    const bool whole = wrow + 32 <= it.row0 + it.rows;
    const int  wpmin = it.pos0 + wrow / a.G, wpmax = it.pos0 + (wend - 1) / a.G;
    const bool wave_in = wrow < it.row0 + it.rows;

    uint4 qf[DP / 16];
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
        const int d = s * 16 + half * 8;
        qf[s]       = rin && d < a.D ? *reinterpret_cast<const uint4 *>(a.q + tok * a.q_st + hq * a.q_sh + d)
                                     : make_uint4(0, 0, 0, 0);
    }
    att_f16 o[DP / 32];
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) o[i][j] = 0.0f;
    float m = -INFINITY, l = 0.0f;

    uint4 kreg[NP], vreg[NP];
    float scl[2] = {0.0f, 1.0f}; // key and value scale of key `tid`
    auto  rows = [&](int t) { // pool rows of a key tile's keys
        if (tid < KT) srow[t & 1][tid] = t < it.t1 ? attn_key_row(a, it, h, attn_key0(it, t, KT) + tid) : -1;
    };
    auto load = [&](int t) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int p = i * NT + tid, key = p / CPR, e = (p % CPR) * EC;
            const int row = srow[t & 1][key];
            kreg[i] = vreg[i] = make_uint4(0, 0, 0, 0);
            if (row >= 0 && e < a.D) {
                const int64_t off = (static_cast<int64_t>(row) * a.D + e) * ES;
                kreg[i]           = *reinterpret_cast<const uint4 *>(a.kc + off);
                vreg[i]           = *reinterpret_cast<const uint4 *>(a.vc + off);
            }
        }
        if constexpr (FP8) {
            if (tid < KT) {
                const int row = srow[t & 1][tid];
                scl[0]        = row >= 0 ? a.ks[row] : 0.0f;
                scl[1]        = row >= 0 ? a.vs[row] : 1.0f;
            }
        }
    };
    auto stage = [&](int t) {
        uint16_t *K = sk[t & 1], *V = sv[t & 1];
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int p = i * NT + tid, key = p / CPR, e = (p % CPR) * EC;
            // 16-byte pieces of a key row in an order of its own, so that equal
            // pieces of consecutive keys lie in different banks
            if constexpr (FP8) {
                const int pc = e / 8;
                *reinterpret_cast<uint4 *>(K + key * DP + ((pc ^ (key & (KC - 1))) * 8)) =
                    att_cvt8<QT, KIND>(kreg[i].x, kreg[i].y);
                *reinterpret_cast<uint4 *>(K + key * DP + (((pc + 1) ^ (key & (KC - 1))) * 8)) =
                    att_cvt8<QT, KIND>(kreg[i].z, kreg[i].w);
                *reinterpret_cast<uint4 *>(V + key * VS + e)     = att_cvt8<QT, KIND>(vreg[i].x, vreg[i].y);
                *reinterpret_cast<uint4 *>(V + key * VS + e + 8) = att_cvt8<QT, KIND>(vreg[i].z, vreg[i].w);
            } else {
                *reinterpret_cast<uint4 *>(K + key * DP + (((e / 8) ^ (key & (KC - 1))) * 8)) = kreg[i];
                *reinterpret_cast<uint4 *>(V + key * VS + e)                                  = vreg[i];
            }
        }
        if constexpr (FP8) {
            if (tid < KT) {
                // no scale of the writer is below 2^-49; one of zero stands for values of zero
                const float vs = fmaxf(scl[1], 0x1p-100f);
                ssc[t & 1][0][tid] = scl[0] * a.scale_log2;
                ssc[t & 1][1][tid] = att_log2(vs);
                ssc[t & 1][2][tid] = 1.0f / vs;
            }
        }
    };

    rows(it.t0);
    __syncthreads();
    if (it.t0 < it.t1) load(it.t0);
    rows(it.t0 + 1);
    for (int t = it.t0; t < it.t1; ++t) {
        stage(t);
        __syncthreads();
        if (t + 1 < it.t1) load(t + 1);
        const int key0 = attn_key0(it, t, KT);
        if (wave_in && key0 <= wpmax) {
            const uint16_t *K = sk[t & 1], *V = sv[t & 1];
            att_f16 s[2];
#pragma unroll
            for (int b = 0; b < 2; ++b) {
#pragma unroll
                for (int j = 0; j < 16; ++j) s[b][j] = 0.0f;
                const int key = b * 32 + c;
#pragma unroll
                for (int k = 0; k < DP / 16; ++k) {
                    const uint4 kf =
                        *reinterpret_cast<const uint4 *>(K + key * DP + (((k * 2 + half) ^ (key & (KC - 1))) * 8));
                    s[b] = AttT<QT>::mfma32(kf, qf[k], s[b]);
                }
            }
            // logits; register j of block b holds key b * 32 + 8 (j / 4) + 4 half + j % 4
            float mx = m;
            float iv[2][16];
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int kk = b * 32 + 8 * g + 4 * half;
                    if constexpr (FP8) {
                        const float4 x = *reinterpret_cast<const float4 *>(&ssc[t & 1][0][kk]);
                        const float4 y = *reinterpret_cast<const float4 *>(&ssc[t & 1][1][kk]);
                        const float4 z = *reinterpret_cast<const float4 *>(&ssc[t & 1][2][kk]);
                        s[b][4 * g]     = fmaf(s[b][4 * g], x.x, y.x);
                        s[b][4 * g + 1] = fmaf(s[b][4 * g + 1], x.y, y.y);
                        s[b][4 * g + 2] = fmaf(s[b][4 * g + 2], x.z, y.z);
                        s[b][4 * g + 3] = fmaf(s[b][4 * g + 3], x.w, y.w);
                        iv[b][4 * g] = z.x; iv[b][4 * g + 1] = z.y; iv[b][4 * g + 2] = z.z; iv[b][4 * g + 3] = z.w;
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; ++j) s[b][4 * g + j] *= a.scale_log2;
                    }
                }
            if (!whole || key0 + KT - 1 > wpmin || (a.window > 0 && key0 < wpmax - a.window + 1)) {
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const int  key = key0 + b * 32 + 8 * (j / 4) + 4 * half + j % 4;
                        const bool see = key <= pos && (key >= wlo || key < a.sinks);
                        s[b][j]        = see ? s[b][j] : -INFINITY;
                    }
            }
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int j = 0; j < 16; ++j) mx = fmaxf(mx, s[b][j]);
            mx                = max_xor32(mx);
            const float base  = mx == -INFINITY ? 0.0f : mx; // nothing seen yet
            const float alpha = att_exp2(m - base);
            m                 = mx;
            l *= alpha;
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    s[b][j] = att_exp2(s[b][j] - base);
                    if constexpr (FP8) l = fmaf(s[b][j], iv[b][j], l);
                    else l += s[b][j];
                }
#pragma unroll
            for (int i = 0; i < DP / 32; ++i)
#pragma unroll
                for (int j = 0; j < 16; ++j) o[i][j] *= alpha;
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int st = 0; st < 2; ++st) {
                    const int   j0 = 8 * st;
                    const uint4 pf = make_uint4(AttT<QT>::pack(s[b][j0], s[b][j0 + 1]), AttT<QT>::pack(s[b][j0 + 2], s[b][j0 + 3]),
                                                AttT<QT>::pack(s[b][j0 + 4], s[b][j0 + 5]), AttT<QT>::pack(s[b][j0 + 6], s[b][j0 + 7]));
                    const int   kr = b * 32 + st * 16 + half * 4 + (lane & 15) / 4;
                    const int   dc = ((lane >> 4) & 1) * 16 + 4 * (lane & 3);
#pragma unroll
                    for (int i = 0; i < DP / 32; ++i) {
                        const uint2 v0 = att_tr16(V + kr * VS + i * 32 + dc), v1 = att_tr16(V + (kr + 8) * VS + i * 32 + dc);
                        o[i] = AttT<QT>::mfma32(make_uint4(v0.x, v0.y, v1.x, v1.y), pf, o[i]);
                    }
                }
        }
        rows(t + 2);
    }
    l = add_xor32(l);
    if (!rin) return;
    if (it.chunks == 1) {
        const float   inv = l > 0.0f || l != l ? 1.0f / l : 0.0f; // no key seen: zeros
        const int64_t at  = (static_cast<int64_t>(tok) * a.Hq + hq) * a.D;
#pragma unroll
        for (int i = 0; i < DP / 32; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int d = i * 32 + 8 * g + 4 * half;
                if (d < a.D)
                    *reinterpret_cast<uint2 *>(a.out + at + d) =
                        make_uint2(AttT<QT>::pack(o[i][4 * g] * inv, o[i][4 * g + 1] * inv),
                                   AttT<QT>::pack(o[i][4 * g + 2] * inv, o[i][4 * g + 3] * inv));
            }
        if (a.lse != nullptr && half == 0) a.lse[static_cast<int64_t>(tok) * a.Hq + hq] = (m + att_log2(l)) * 0.69314718055994531f;
    } else {
        const int64_t at = (static_cast<int64_t>(slot) * a.Hkv + h) * BQ + wave * 32 + c;
#pragma unroll
        for (int i = 0; i < DP / 32; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int d = i * 32 + 8 * g + 4 * half;
                if (d < a.D)
                    *reinterpret_cast<float4 *>(a.part_o + at * a.D + d) =
                        make_float4(o[i][4 * g], o[i][4 * g + 1], o[i][4 * g + 2], o[i][4 * g + 3]);
            }
        if (half == 0) a.part_ml[at] = make_float2(m, l);
    }
}

// ---------------------------------------------------------------------------
// narrow kernel: 16 rows, four waves on 32 keys each of a key tile of 128
// ---------------------------------------------------------------------------
template <int QT, int KIND, int DP>
__global__ __launch_bounds__(256, DP > 128 ? 1 : 2) void attn_narrow_kernel(AttnArgs a) {
    constexpr int  KT = 128, BQ = 16, WK = 32;
    constexpr bool FP8 = KIND != PTA_CACHE_16BIT;
    constexpr int  ES  = FP8 ? 1 : 2;
    constexpr int  EC  = 16 / ES;
    constexpr int  KP  = DP / 4 / EC;       // 16-byte pieces of a lane's quarter of a key row
    constexpr int  CPR = DP / EC;           // pieces of a value row
    constexpr int  VP  = WK * CPR / 64;     // value pieces of a lane
    constexpr int  VS  = DP + 16;           // elements of a staged value row: the transposed read's 16 rows
                                            // of 32 bytes then fall into different banks
    constexpr int  OS  = DP + 4;            // floats of a row of the waves' joined output
    constexpr int  SV_BYTES = 4 * WK * VS * 2, SO_BYTES = 4 * BQ * OS * 4;
    static_assert(KP >= 1, "a quarter row is a piece at least");
    __shared__ __align__(16) uint8_t smem[SV_BYTES > SO_BYTES ? SV_BYTES : SO_BYTES];
    __shared__ __align__(16) float   ssc[4][3][WK];
    __shared__ float2                sml[4][BQ];
    __shared__ uint32_t              red[16];

    const int      tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int      h    = blockIdx.x % a.Hkv;
    const int      slot = blockIdx.x / a.Hkv;
    const AttnItem it   = attn_find<BQ, KT, 256>(a, slot, red);
    if (a.desc != nullptr && h == 0 && tid == 0)
        a.desc[slot] = it.b < 0 ? make_int4(ATT_NONE, 0, 0, 0) : make_int4(it.b, it.tile, it.chunk, it.chunks);
    if (it.b < 0) return;

    const int  c = lane & 15, qd = lane >> 4;
    const int  r    = it.row0 + c;
    const bool rin  = c < it.rows;
    const int  rtok = rin ? r / a.G : 0;
    const int  tok  = it.tok0 + rtok;
    const int  hq   = h * a.G + (rin ? r - rtok * a.G : 0);
    const int  pos  = rin ? it.pos0 + rtok : -1;
    const int  wlo  = a.window > 0 ? pos - a.window + 1 : INT_MIN;

    // k-step s of the products over the head dimension takes elements
    // qd * DP / 4 + 8 s .. + 7 from quarter qd of the lanes: a lane's part of a
    // key row is one run of bytes
    uint4 qf[DP / 32];
#pragma unroll
    for (int s = 0; s < DP / 32; ++s) {
        const int d = qd * (DP / 4) + s * 8;
        qf[s]       = rin && d < a.D ? *reinterpret_cast<const uint4 *>(a.q + tok * a.q_st + hq * a.q_sh + d)
                                     : make_uint4(0, 0, 0, 0);
    }
    att_f4 o[DP / 16];
#pragma unroll
    for (int i = 0; i < DP / 16; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][j] = 0.0f;
    float m = -INFINITY, l = 0.0f;

    uint16_t *V = reinterpret_cast<uint16_t *>(smem) + wave * WK * VS;
    uint4     kreg[2][KP], vreg[VP];
    float     scl[2] = {0.0f, 1.0f};
    auto      row_of = [&](int t) { // pool row of key lane % 32 of this wave's part
        return t < it.t1 ? attn_key_row(a, it, h, attn_key0(it, t, KT) + wave * WK + (lane & 31)) : -1;
    };
    auto load = [&](int row) {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int kr = __shfl(row, b * 16 + c);
#pragma unroll
            for (int i = 0; i < KP; ++i) {
                const int e = qd * (DP / 4) + i * EC;
                kreg[b][i]  = make_uint4(0, 0, 0, 0);
                if (kr >= 0 && e < a.D)
                    kreg[b][i] = *reinterpret_cast<const uint4 *>(a.kc + (static_cast<int64_t>(kr) * a.D + e) * ES);
            }
        }
#pragma unroll
        for (int i = 0; i < VP; ++i) {
            const int p = i * 64 + lane, key = p / CPR, e = (p % CPR) * EC;
            const int vr = __shfl(row, key);
            vreg[i]      = make_uint4(0, 0, 0, 0);
            if (vr >= 0 && e < a.D)
                vreg[i] = *reinterpret_cast<const uint4 *>(a.vc + (static_cast<int64_t>(vr) * a.D + e) * ES);
        }
        if constexpr (FP8) {
            scl[0] = row >= 0 ? a.ks[row] : 0.0f;
            scl[1] = row >= 0 ? a.vs[row] : 1.0f;
        }
    };

    load(row_of(it.t0));
    int next = row_of(it.t0 + 1);
    for (int t = it.t0; t < it.t1; ++t) {
        // this tile's values to LDS, its keys as operands; then the next tile's loads
#pragma unroll
        for (int i = 0; i < VP; ++i) {
            const int p = i * 64 + lane, key = p / CPR, e = (p % CPR) * EC;
            if constexpr (FP8) {
                *reinterpret_cast<uint4 *>(V + key * VS + e)     = att_cvt8<QT, KIND>(vreg[i].x, vreg[i].y);
                *reinterpret_cast<uint4 *>(V + key * VS + e + 8) = att_cvt8<QT, KIND>(vreg[i].z, vreg[i].w);
            } else {
                *reinterpret_cast<uint4 *>(V + key * VS + e) = vreg[i];
            }
        }
        if constexpr (FP8) {
            if (lane < WK) {
                const float vs        = fmaxf(scl[1], 0x1p-100f); // no scale of the writer is below 2^-49; one of zero stands for values of zero
                ssc[wave][0][lane] = scl[0] * a.scale_log2;
                ssc[wave][1][lane] = att_log2(vs);
                ssc[wave][2][lane] = 1.0f / vs;
            }
        }
        uint4 kf[2][DP / 32];
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int s = 0; s < DP / 32; ++s) {
                if constexpr (FP8) {
                    const uint4 w = kreg[b][s / 2];
                    kf[b][s] = s % 2 == 0 ? att_cvt8<QT, KIND>(w.x, w.y) : att_cvt8<QT, KIND>(w.z, w.w);
                } else {
                    kf[b][s] = kreg[b][s];
                }
            }
        if (t + 1 < it.t1) {
            load(next);
            next = row_of(t + 2);
        }
        att_f4 s[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
#pragma unroll
            for (int j = 0; j < 4; ++j) s[b][j] = 0.0f;
#pragma unroll
            for (int k = 0; k < DP / 32; ++k) s[b] = AttT<QT>::mfma16(kf[b][k], qf[k], s[b]);
        }
        // the wave's own LDS writes are seen by its later reads once they are done
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        const int key0 = attn_key0(it, t, KT) + wave * WK;
        float     mx = m, iv[2][4];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int kk = b * 16 + 4 * qd;
            if constexpr (FP8) {
                const float4 x = *reinterpret_cast<const float4 *>(&ssc[wave][0][kk]);
                const float4 y = *reinterpret_cast<const float4 *>(&ssc[wave][1][kk]);
                const float4 z = *reinterpret_cast<const float4 *>(&ssc[wave][2][kk]);
                s[b][0] = fmaf(s[b][0], x.x, y.x); s[b][1] = fmaf(s[b][1], x.y, y.y);
                s[b][2] = fmaf(s[b][2], x.z, y.z); s[b][3] = fmaf(s[b][3], x.w, y.w);
                iv[b][0] = z.x; iv[b][1] = z.y; iv[b][2] = z.z; iv[b][3] = z.w;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) s[b][j] *= a.scale_log2;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int  key = key0 + kk + j;
                const bool see = key <= pos && (key >= wlo || key < a.sinks);
                s[b][j]        = see ? s[b][j] : -INFINITY;
                mx             = fmaxf(mx, s[b][j]);
            }
        }
        mx                = max_xor32(max_xor16(mx));
        const float base  = mx == -INFINITY ? 0.0f : mx;
        const float alpha = att_exp2(m - base);
        m                 = mx;
        l *= alpha;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s[b][j] = att_exp2(s[b][j] - base);
                if constexpr (FP8) l = fmaf(s[b][j], iv[b][j], l);
                else l += s[b][j];
            }
        const uint4 pf = make_uint4(AttT<QT>::pack(s[0][0], s[0][1]), AttT<QT>::pack(s[0][2], s[0][3]),
                                    AttT<QT>::pack(s[1][0], s[1][1]), AttT<QT>::pack(s[1][2], s[1][3]));
        const int   kr = 4 * qd + c / 4, dc = 4 * (c & 3);
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][j] *= alpha;
            const uint2 v0 = att_tr16(V + kr * VS + i * 16 + dc), v1 = att_tr16(V + (kr + 16) * VS + i * 16 + dc);
            o[i] = AttT<QT>::mfma16(make_uint4(v0.x, v0.y, v1.x, v1.y), pf, o[i]);
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
    l = add_xor32(add_xor16(l));
    // the four waves' parts join in LDS
    __syncthreads(); // the values' LDS becomes the outputs'
    float *so = reinterpret_cast<float *>(smem);
    if (qd == 0) sml[wave][c] = make_float2(m, l);
#pragma unroll
    for (int i = 0; i < DP / 16; ++i)
        *reinterpret_cast<float4 *>(so + (wave * BQ + c) * OS + i * 16 + 4 * qd) = make_float4(o[i][0], o[i][1], o[i][2], o[i][3]);
    __syncthreads();
    constexpr int TPR = 16, DPT = DP / TPR; // threads of a row, their elements
    const int     jr = tid / TPR, jd = (tid % TPR) * DPT;
    if (jr >= it.rows) return;
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; ++w) mm = fmaxf(mm, sml[w][jr].x);
    const float base = mm == -INFINITY ? 0.0f : mm;
    float       ll = 0.0f, acc[DPT];
#pragma unroll
    for (int e = 0; e < DPT; ++e) acc[e] = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const float f = att_exp2(sml[w][jr].x - base);
        ll            = fmaf(sml[w][jr].y, f, ll);
#pragma unroll
        for (int e = 0; e < DPT; ++e) acc[e] = fmaf(so[(w * BQ + jr) * OS + jd + e], f, acc[e]);
    }
    if (it.chunks == 1) {
        const int     rr = it.row0 + jr, rt = rr / a.G;
        const int64_t orow = static_cast<int64_t>(it.tok0 + rt) * a.Hq + h * a.G + (rr - rt * a.G);
        const float   inv  = ll > 0.0f || ll != ll ? 1.0f / ll : 0.0f;
#pragma unroll
        for (int e = 0; e < DPT; e += 4)
            if (jd + e < a.D)
                *reinterpret_cast<uint2 *>(a.out + orow * a.D + jd + e) =
                    make_uint2(AttT<QT>::pack(acc[e] * inv, acc[e + 1] * inv), AttT<QT>::pack(acc[e + 2] * inv, acc[e + 3] * inv));
        if (a.lse != nullptr && jd == 0) a.lse[orow] = (mm + att_log2(ll)) * 0.69314718055994531f;
    } else {
        const int64_t at = (static_cast<int64_t>(slot) * a.Hkv + h) * BQ + jr;
#pragma unroll
        for (int e = 0; e < DPT; e += 4)
            if (jd + e < a.D)
                *reinterpret_cast<float4 *>(a.part_o + at * a.D + jd + e) = make_float4(acc[e], acc[e + 1], acc[e + 2], acc[e + 3]);
        if (jd == 0) a.part_ml[at] = make_float2(mm, ll);
    }
}

// ---------------------------------------------------------------------------
// joins the chunks of a row tile: workgroup = (first slot of the tile, head)
// ---------------------------------------------------------------------------
template <int QT, int BQ> __global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a) {
    const int  h = blockIdx.x % a.Hkv, slot = blockIdx.x / a.Hkv;
    const int4 w = a.desc[slot]; // sequence, row tile, chunk, chunks
    if (w.x == ATT_NONE || w.z != 0 || w.w == 1) return;
    const AttnSeq s    = attn_seq(a, w.x);
    const int     row0 = w.y * BQ, rows = min(BQ, s.n * a.G - row0);
    const int     tpr = a.D / 4; // threads of a row
    for (int p = threadIdx.x; p < rows * tpr; p += 256) {
        const int jr = p / tpr, d = (p - jr * tpr) * 4;
        float     mm = -INFINITY;
        for (int c = 0; c < w.w; ++c) mm = fmaxf(mm, a.part_ml[(static_cast<int64_t>(slot + c) * a.Hkv + h) * BQ + jr].x);
        const float base = mm == -INFINITY ? 0.0f : mm;
        float       ll = 0.0f;
        float4      acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int c = 0; c < w.w; ++c) {
            const int64_t at = (static_cast<int64_t>(slot + c) * a.Hkv + h) * BQ + jr;
            const float2  ml = a.part_ml[at];
            const float   f  = att_exp2(ml.x - base);
            const float4  x  = *reinterpret_cast<const float4 *>(a.part_o + at * a.D + d);
            ll               = fmaf(ml.y, f, ll);
            acc.x = fmaf(x.x, f, acc.x); acc.y = fmaf(x.y, f, acc.y);
            acc.z = fmaf(x.z, f, acc.z); acc.w = fmaf(x.w, f, acc.w);
        }
        const int     rr = row0 + jr, rt = rr / a.G;
        const int64_t orow = static_cast<int64_t>(s.tok0 + rt) * a.Hq + h * a.G + (rr - rt * a.G);
        const float   inv  = ll > 0.0f || ll != ll ? 1.0f / ll : 0.0f;
        *reinterpret_cast<uint2 *>(a.out + orow * a.D + d) =
            make_uint2(AttT<QT>::pack(acc.x * inv, acc.y * inv), AttT<QT>::pack(acc.z * inv, acc.w * inv));
        if (a.lse != nullptr && d == 0) a.lse[orow] = (mm + att_log2(ll)) * 0.69314718055994531f;
    }
}

// Launches the kernels of one type of queries (paged_attention_inst_*.hip).
// wide: rows of the row tile are 128 (wide) or 16 (narrow).
template <int QT> void attn_launch(const AttnArgs &a, int kind, bool wide, hipStream_t st);
extern template void attn_launch<PTA_BF16>(const AttnArgs &, int, bool, hipStream_t);
extern template void attn_launch<PTA_F16>(const AttnArgs &, int, bool, hipStream_t);

constexpr int ATT_WIDE_ROWS = 128, ATT_WIDE_KEYS = 64, ATT_NARROW_ROWS = 16, ATT_NARROW_KEYS = 128;

} // namespace pta
