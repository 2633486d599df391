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
// P stays in [0, 1], in the wide form, whose m may lag behind the maximum, below
// 2^8, however large or small the scales are, which fp16 needs.  It is rounded
// once, to the 16 bits that the matrix instructions take; logits, m, l and O are
// fp32.
//
// The query heads of one key / value head are rows of one matrix, r = i * G + g
// (G = Hq / Hkv), so a key is read once for all of them.  Both products are
// computed transposed: S^T = K Q^T has keys as rows and queries as columns, so
// the softmax statistics of a query are values of one lane (its column), and
// the registers of S^T are the operand of O^T = V^T P^T as they are: the
// contraction runs over the keys in the order in which S^T holds them, and V
// comes from LDS through the transposing read in that order.
//
// Two forms share this: the wide one (32 rows a wave, keys and values staged in LDS
// for all waves) where a sequence has many rows, the narrow one (16 rows, keys
// straight into registers, every wave on keys of its own) where it has few and the
// cache's bytes bound the call.  The keys of a row tile may be split over several
// workgroups; a last kernel joins their parts.
#pragma once

#include <climits>
#include <type_traits>
#include <utility>

#include "common.h"

namespace pta {

// on lambdas of a kernel: one that is called captures its arrays in memory
#define PTA_INLINE __attribute__((always_inline))

constexpr int ATT_WIDE_ROWS = 128, ATT_WIDE_KEYS = 64, ATT_NARROW_ROWS = 16, ATT_NARROW_KEYS = 128;

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
    float          *part_o;  // [parts, Hkv, BQ, D] (wide), [split, Tq, Hq, D] or [split, B, Hkv, 16, D] (narrow)
    float2         *part_ml; // the same without D
    int4           *desc;    // [slots]: sequence, row tile, its first part (-1: none, or another chunk's), chunks (wide)
    int             B, Tq, Hq, Hkv, G, D;
    int             num_pages, page, max_pages;
    uint32_t        page_mul, page_shift; // j / page = mulhi(j, page_mul) >> page_shift for j < 2^31; page_mul 0: j >> page_shift
    int             window, sinks; // window 0: none
    float           scale_log2;
    int             slots;      // wide: work items per key / value head that the grid holds
    int             split_goal; // wide; 0: row tiles are never split
    int             split;      // narrow: chunks of a sequence
    int             part_seq, part_step; // narrow: parts go by sequence, not by token; rows of a chunk's parts
    int             rows_min, rows_max; // sequences of this launch: rows_min < n G <= rows_max
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
    static __device__ __forceinline__ float dot(uint32_t x, uint32_t y) { // of two pairs
        return fmaf(__uint_as_float(x << 16), __uint_as_float(y << 16), __uint_as_float(x & 0xffff0000u) * __uint_as_float(y & 0xffff0000u));
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
    static __device__ __forceinline__ float dot(uint32_t x, uint32_t y) { // of two pairs
        return fmaf(f16_bits_to_f32(x & 0xffffu), f16_bits_to_f32(y & 0xffffu), f16_bits_to_f32(x >> 16) * f16_bits_to_f32(y >> 16));
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

// f(0), f(1), ..., f(N - 1) with constants: arrays indexed by them stay in registers
template <class F, int... I> __device__ __forceinline__ void att_each(F &&f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F> __device__ __forceinline__ void att_each(F &&f) {
    att_each(f, std::make_integer_sequence<int, N>{});
}

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

// the lane's number, opaque to the compiler
__device__ __forceinline__ int att_lane() {
    int r;
    asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=&v"(r));
    return r;
}

__device__ __forceinline__ float att_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float att_log2(float x) { return __builtin_amdgcn_logf(x); }

// The two values of a value scale: a scale of zero (values of zero) counts as 2^-100.
// A NaN stays in the logits, where a row that does not see the key replaces it, and
// not in the factor of the row's sum, which multiplies that row's zero.
constexpr float ATT_LEAST_SCALE = 0x1p-100f;
__device__ __forceinline__ float att_clamp_scale(float vs) { return fmaxf(vs, ATT_LEAST_SCALE); }
__device__ __forceinline__ float att_log2_scale(float vs) { return att_log2(vs < ATT_LEAST_SCALE ? ATT_LEAST_SCALE : vs); }

// 1 / l of a row; one that sees no key (its position is below 0) becomes zeros.
// Logits of -inf alone give l = 0 and 0 / 0, as the formula does.
__device__ __forceinline__ float att_inverse(float l, bool none) { return none ? 0.0f : 1.0f / l; }
// Among parts that are joined, such a row has m = 0 and l = 0, the others m = -inf
// where they have seen nothing yet.  The join could read the lengths instead, but then
// takes 81 scalar registers for 80, and 8.4 us for 6.8 (64 sequences, 64 heads of 128,
// four chunks).
__device__ __forceinline__ float att_part_max(float m, bool none) { return none ? 0.0f : m; }

// max(a, b, c), NaN dropped; the plain form quiets operands first
__device__ __forceinline__ float att_max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

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
    int part;                   // number of the chunk among those of split row tiles
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
    const int64_t rows = static_cast<int64_t>(s.n) * a.G;
    if (rows <= a.rows_min || rows > a.rows_max) s.n = 0; // another launch's
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

// The list of key tiles of an item whose rows and positions are set: its fields,
// and its length.
template <int KT> __device__ __forceinline__ int attn_keys(const AttnArgs &a, AttnItem &it, int len) {
    const int pmin = it.pos0 + it.row0 / a.G, pmax = it.pos0 + (it.row0 + it.rows - 1) / a.G;
    it.kend = max(0, min(pmax + 1, len));
    it.lo   = min(a.window > 0 ? max(0, pmin - a.window + 1) : 0, it.kend);
    // sink tiles that the window's tiles do not cover
    const int first = it.lo / KT, last = (it.kend + KT - 1) / KT;
    it.n_sink  = min(a.window > 0 ? (min(a.sinks, it.kend) + KT - 1) / KT : 0, first);
    it.lo_tile = first;
    return it.n_sink + max(0, last - first);
}

// Finds the item of slot `slot`; all threads of the workgroup call it (`red`:
// 16 words of LDS).  Items are numbered sequence by sequence, row tile by row
// tile, chunk by chunk; a row tile's k key tiles make ceil(k / C) equal chunks, C
// such that all items of a head fit the grid: sum over the row tiles of
// ceil(k / C) <= sum(k) / C + tiles.  A tile is split where k > C, into less than
// 2 k / C chunks: less than twice the split goal in all have parts.
template <int BQ, int KT, int NTHR> __device__ AttnItem attn_find(const AttnArgs &a, int slot, uint32_t *red) {
    constexpr int NW = NTHR / 64;
    const int     tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // inclusive prefix sums over the workgroup, two side by side
    auto scan = [&](uint32_t(&v)[2], uint32_t(&total)[2]) PTA_INLINE {
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t o0 = __shfl_up(v[0], d), o1 = __shfl_up(v[1], d);
            if (lane >= d) {
                v[0] += o0;
                v[1] += o1;
            }
        }
        __syncthreads();
        if (lane == 63) {
            red[wave]      = v[0];
            red[12 + wave] = v[1];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            uint32_t before = 0;
            total[i]        = 0;
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                if (w < wave) before += red[12 * i + w];
                total[i] += red[12 * i + w];
            }
            v[i] += before;
        }
    };
    AttnItem it;
    it.b            = -1;
    const AttnSeq s0 = tid < a.B ? attn_seq(a, tid) : AttnSeq{0, 0, 0};
    int   C = INT_MAX;
    if (a.split_goal > 0) {
        // sums past 32 bits only make C larger than needed: in floating point
        float w = 0.0f, some = 0.0f; // `some`: of up to 256 sequences, so that few roundings add up
        for (int b0 = 0; b0 < a.B; b0 += NTHR) {
            const int b = b0 + tid;
            if (b < a.B) {
                const AttnSeq s = b0 == 0 ? s0 : attn_seq(a, b);
                const float   r = static_cast<float>((static_cast<int64_t>(s.n) * a.G + BQ - 1) / BQ);
                some += r * static_cast<float>(attn_tiles<KT>(a, s, BQ));
            }
            if (b0 / NTHR % 256 == 255) {
                w += some;
                some = 0.0f;
            }
        }
        w += some;
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) w += __shfl_xor(w, d);
        if (lane == 0) red[8 + wave] = __float_as_uint(w);
        __syncthreads();
        w = 0.0f;
#pragma unroll
        for (int i = 0; i < NW; ++i) w += __uint_as_float(red[8 + i]);
        w = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(w)));
        // above the quotient by more than the sum's rounding: the grid holds all items
        C = static_cast<int>(fminf(w * 1.001f / static_cast<float>(a.split_goal), 1e9f)) + 1;
    }
    uint32_t seen = 0, split = 0; // items of the sequences before, those among them that have parts
    for (int b0 = 0; b0 < a.B; b0 += NTHR) {
        const int b = b0 + tid;
        AttnSeq   s = {0, 0, 0};
        uint32_t  tiles = 0, chunks = 1;
        if (b < a.B) {
            s      = b0 == 0 ? s0 : attn_seq(a, b);
            tiles  = static_cast<uint32_t>((static_cast<int64_t>(s.n) * a.G + BQ - 1) / BQ);
            const int k = attn_tiles<KT>(a, s, BQ);
            chunks      = k > C ? (k - 1) / C + 1 : 1;
        }
        uint32_t       incl[2], total[2];
        const uint32_t mine = tiles * chunks;
        incl[0] = mine;
        incl[1] = chunks > 1 ? mine : 0;
        scan(incl, total);
        if (static_cast<uint32_t>(slot) < seen + total[0]) {
            const uint32_t at = static_cast<uint32_t>(slot) - seen;
            __syncthreads();
            if (at < incl[0] && at >= incl[0] - mine) {
                red[0] = b;
                red[1] = at - (incl[0] - mine);
                red[6] = split + incl[1] - mine; // the sequence's first, if it is split
                red[2] = chunks;
                red[3] = s.n;
                red[4] = s.len;
                red[5] = s.tok0;
            }
            __syncthreads();
            it.b      = __builtin_amdgcn_readfirstlane(red[0]);
            it.chunks = __builtin_amdgcn_readfirstlane(red[2]);
            const int at_b = __builtin_amdgcn_readfirstlane(red[1]);
            it.tile   = at_b / it.chunks;
            it.chunk  = at_b - it.tile * it.chunks;
            it.part   = __builtin_amdgcn_readfirstlane(red[6]) + at_b;
            break;
        }
        seen += total[0];
        split += total[1];
    }
    if (it.b < 0) return it;
    const int n = __builtin_amdgcn_readfirstlane(red[3]), len = __builtin_amdgcn_readfirstlane(red[4]);
    it.tok0 = __builtin_amdgcn_readfirstlane(red[5]);
    it.pos0 = len - n; // below 0 where more tokens came than the length says: those see nothing
    it.row0 = it.tile * BQ;
    it.rows = min(BQ, n * a.G - it.row0);
    const int64_t k = attn_keys<KT>(a, it, len);
    it.t0 = static_cast<int>(k * it.chunk / it.chunks);
    it.t1 = static_cast<int>(k * (it.chunk + 1) / it.chunks);
    // all of it is the workgroup's, but came through vector loads: into scalar registers
    for (int *f : {&it.row0, &it.rows, &it.tok0, &it.pos0, &it.kend, &it.lo, &it.n_sink, &it.lo_tile, &it.t0, &it.t1})
        *f = __builtin_amdgcn_readfirstlane(*f);
    return it;
}

__device__ __forceinline__ int attn_key0(const AttnItem &it, int t, int KT) {
    return (t < it.n_sink ? t : it.lo_tile + t - it.n_sink) * KT;
}

__device__ __forceinline__ int attn_page_of(const AttnArgs &a, int j) {
    const uint32_t u = static_cast<uint32_t>(j);
    return static_cast<int>((a.page_mul ? __umulhi(u, a.page_mul) : u) >> a.page_shift);
}
// Page of key j, or -1 where there is none: past the keys, or hidden from every
// row by the window
__device__ __forceinline__ int attn_key_page(const AttnArgs &a, const AttnItem &it, int j) {
    if (j >= it.kend || (j < it.lo && j >= a.sinks)) return -1;
    return a.table[it.b * a.table_st + attn_page_of(a, j)];
}
// Pool row of key j for head h (row = (page * Hkv + h) * page_size + offset), or
// -1 where its page is none of the pool's
__device__ __forceinline__ int attn_page_row(const AttnArgs &a, int h, int j, int pg) {
    if (pg < 0 || pg >= a.num_pages) return -1;
    return (pg * a.Hkv + h) * a.page + (j - attn_page_of(a, j) * a.page);
}

// ---------------------------------------------------------------------------
// wide kernel: 4 waves of 32 rows, key tiles of 64 in LDS
// ---------------------------------------------------------------------------
// Pipeline, one barrier an iteration.  Iteration t interleaves, one matrix
// instruction a step, what the matrix pipe and the vector unit can do side by
// side (a matrix instruction that has to wait for the pipe holds up the vector
// instructions of both waves of the SIMD, so each is followed by about its own
// length of others):
//   S(t + 1) = K(t + 1) Q^T      beside three quarters of tile t's exponentials
//   O += V(t)^T P(t)             beside the last quarter, the logits and maxima of
//                                tile t + 1, and the staging of keys t + 2 and values t + 1
// Each register is loaded with keys t + 3 or values t + 2 once it is staged; the
// loads stay in flight over the barrier.  The softmax's reference m follows the
// running maximum only when a tile exceeds it by 2^8: P then stays below 2^8 and
// most tiles rescale nothing.
//
// Bound by what the vector unit has to do beside the matrix pipe: of the pipe's time
// for a tile of 128 elements a head (4 waves x 64 instructions) the exponentials,
// conversions, scales and staging take about as much again.  2048 new tokens over
// 16384 of 32 / 8 heads of 128, e4m3: 655 us, 790 TFLOP/s, against 419 us at the
// rate of a large library matrix product.  Keys and values go through LDS, converted
// once for all four waves; a wave's registers hold O (64 of 256 a lane at 128
// elements) and Q (32).  Two workgroups a CU hide some of each other's waits.
constexpr float ATT_SLACK = 8.0f;

// bits of a 16-bit type's infinity
template <int QT> constexpr uint32_t att_inf16() { return QT == PTA_BF16 ? 0x7f80u : 0x7c00u; }

// Operand of values with infinities and NaN taken out, and where they are: `plus`
// is 1 for +inf and NaN, `minus` for -inf and NaN.
template <int QT> __device__ __forceinline__ void att_split_special(uint4 v, uint4 &fin, uint4 &plus, uint4 &minus) {
    constexpr uint32_t INF = att_inf16<QT>(), ONE = QT == PTA_BF16 ? 0x3f80u : 0x3c00u;
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t       f[4], p[4], m[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[i] = p[i] = m[i] = 0;
#pragma unroll
        for (int h = 0; h < 32; h += 16) {
            const uint32_t e = w[i] >> h & 0xffffu, mag = e & 0x7fffu;
            if (mag < INF) f[i] |= e << h;
            if (mag > INF || e == INF) p[i] |= ONE << h;
            if (mag > INF || e == (INF | 0x8000u)) m[i] |= ONE << h;
        }
    }
    fin   = make_uint4(f[0], f[1], f[2], f[3]);
    plus  = make_uint4(p[0], p[1], p[2], p[3]);
    minus = make_uint4(m[0], m[1], m[2], m[3]);
}

// 1 where a probability of the operand is not zero
template <int QT> __device__ __forceinline__ uint4 att_nonzero(uint4 v) {
    constexpr uint32_t ONE = QT == PTA_BF16 ? 0x3f80u : 0x3c00u;
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t       r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = ((w[i] & 0xffffu) ? ONE : 0u) | ((w[i] >> 16) ? ONE << 16 : 0u);
    return make_uint4(r[0], r[1], r[2], r[3]);
}

// Whether a 16-byte piece of cache values holds infinities or NaN
template <int QT, int KIND> __device__ __forceinline__ bool att_has_special(uint4 v) {
    // exponents of all ones, and for e4m3 the NaN code: adding the distance to the
    // sign bit carries into it
    constexpr uint32_t MAG = KIND == PTA_CACHE_16BIT ? 0x7fff7fffu : 0x7f7f7f7fu;
    constexpr uint32_t TOP = KIND == PTA_CACHE_16BIT ? 0x80008000u : 0x80808080u;
    constexpr uint32_t ADD = KIND == PTA_CACHE_16BIT ? (QT == PTA_BF16 ? 0x00800080u : 0x04000400u)
                                                     : (KIND == PTA_E4M3 ? 0x01010101u : 0x04040404u);
    return ((((v.x & MAG) + ADD) | ((v.y & MAG) + ADD) | ((v.z & MAG) + ADD) | ((v.w & MAG) + ADD)) & TOP) != 0;
}

// Cache elements i .. i + 3 in fp32
template <int QT, int KIND> __device__ __forceinline__ void att_values4(const uint8_t *pool, int64_t i, float (&v)[4]) {
    if constexpr (KIND == PTA_CACHE_16BIT) {
        const uint2 w = *reinterpret_cast<const uint2 *>(pool + 2 * i);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t h = (j < 2 ? w.x : w.y) >> (16 * (j & 1)) & 0xffffu;
            v[j]             = QT == PTA_BF16 ? bf16_bits_to_f32(h) : f16_bits_to_f32(h);
        }
    } else {
        const int w = *reinterpret_cast<const int *>(pool + i);
        if constexpr (KIND == PTA_E4M3) {
            v[0] = __builtin_amdgcn_cvt_f32_fp8(w, 0); v[1] = __builtin_amdgcn_cvt_f32_fp8(w, 1);
            v[2] = __builtin_amdgcn_cvt_f32_fp8(w, 2); v[3] = __builtin_amdgcn_cvt_f32_fp8(w, 3);
        } else {
            v[0] = __builtin_amdgcn_cvt_f32_bf8(w, 0); v[1] = __builtin_amdgcn_cvt_f32_bf8(w, 1);
            v[2] = __builtin_amdgcn_cvt_f32_bf8(w, 2); v[3] = __builtin_amdgcn_cvt_f32_bf8(w, 3);
        }
    }
}

template <int KIND, int DP> struct AttnWideLds {
    static constexpr int KT = ATT_WIDE_KEYS;
    static constexpr int KS = DP + 8;  // elements of a staged key row: 16 rows' equal pieces lie in different banks
    static constexpr int VS = DP + 32; // of a value row: the transposed read's 8 rows of 64 bytes do; odd keys have
                                       // the halves of every 32 bytes exchanged, for the writes' sake
    static constexpr bool FP8 = KIND != PTA_CACHE_16BIT;
    alignas(16) uint16_t sk[2][KT * KS];
    alignas(16) uint16_t sv[2][KT * VS];
    alignas(16) float ssc[FP8 ? 3 : 1][3][FP8 ? KT : 4]; // scale log2e ks, log2 vs, 1 / vs by tile % 3
    int      srow[8][KT];
    int      shole[8];    // by tile % 8: some key has no row
    int      sspec[2][4]; // by tile % 2 and wave: values with infinities or NaN
    uint32_t red[16];
};

template <int QT, int KIND, int DP>
__device__ __forceinline__ void attn_wide(const AttnArgs &a, int block, AttnWideLds<KIND, DP> &lds) {
    constexpr int  KT = ATT_WIDE_KEYS, BQ = ATT_WIDE_ROWS, NT = 256;
    constexpr bool FP8 = KIND != PTA_CACHE_16BIT;
    constexpr int  ES  = FP8 ? 1 : 2;       // bytes of a cache element
    constexpr int  EC  = 16 / ES;           // elements of a 16-byte piece
    constexpr int  CPR = DP / EC;           // pieces of a row
    constexpr int  NP  = KT * CPR / NT;     // pieces of a thread and pool
    constexpr int  KS = AttnWideLds<KIND, DP>::KS, VS = AttnWideLds<KIND, DP>::VS;
    static_assert(KT * CPR % NT == 0, "pieces");
    auto &sk = lds.sk; auto &sv = lds.sv; auto &ssc = lds.ssc; auto &srow = lds.srow;
    auto &shole = lds.shole; auto &sspec = lds.sspec; auto &red = lds.red;

    int            tid = threadIdx.x, lane = tid & 63;
    const int      wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int      h    = block % a.Hkv;
    const int      slot = block / a.Hkv;
    const AttnItem it   = attn_find<BQ, KT, NT>(a, slot, red);
    if (a.desc != nullptr && h == 0 && tid == 0)
        a.desc[slot] = it.b < 0 || it.chunks == 1 || it.chunk > 0 ? make_int4(0, 0, -1, 0) : make_int4(it.b, it.tile, it.part, it.chunks);
    if (it.b < 0) return;

    int  page_id     = -1;
    auto fetch_pages = [&](int t) PTA_INLINE { // t: the wave's tile
        page_id = t < it.t1 ? attn_key_page(a, it, attn_key0(it, t, KT) + lane) : -1;
    };
    fetch_pages(it.t0 + wave);
    int c = lane & 31, half = lane >> 5;
    uint4     qf[DP / 16];
    int       pos = -1; // of this lane's row; rows past the tile see nothing
    {
        const int  r  = it.row0 + wave * 32 + c;
        const bool in = r < it.row0 + it.rows;
        const int  rt = in ? r / a.G : 0, hq = h * a.G + (in ? r - rt * a.G : 0);
        if (in) pos = it.pos0 + rt;
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) {
            const int d = s * 16 + half * 8;
            qf[s]       = in && d < a.D ? *reinterpret_cast<const uint4 *>(a.q + (it.tok0 + rt) * a.q_st + hq * a.q_sh + d)
                                        : make_uint4(0, 0, 0, 0);
        }
    }
    // positions of the wave's rows
    const int  wrow = it.row0 + wave * 32, wend = min(wrow + 32, it.row0 + it.rows);
    const bool full = wrow + 32 <= it.row0 + it.rows;
    const int  wpmin = it.pos0 + wrow / a.G, wpmax = it.pos0 + (wend - 1) / a.G;
    // the wave's tiles: keys past its last row's are other waves'
    int tend = it.t0;
    if (wend > wrow && wpmax >= 0) {
        const int last = wpmax / KT + 1; // key tiles up to its last key
        tend = last <= it.n_sink ? last : last > it.lo_tile ? it.n_sink + last - it.lo_tile : it.n_sink;
        tend = max(it.t0, min(tend, it.t1));
    }
    tend = __builtin_amdgcn_readfirstlane(tend);
    // tiles in which not every row sees every key
    const int  bpmin  = it.pos0 + it.row0 / a.G;
    const bool full_block = it.rows == BQ;
    auto edge = [&](int t, int pmin, int pmax) PTA_INLINE {
        const int key0 = attn_key0(it, t, KT);
        return key0 + KT - 1 > pmin || (a.window > 0 && key0 < pmax - a.window + 1);
    };

    att_f16 o[DP / 32];
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) o[i][j] = 0.0f;
    float m = -INFINITY, l = 0.0f, mx = -INFINITY;

    uint4 kreg[NP], vreg[NP];
    float kscl = 0.0f, vscl = 1.0f; // of key `tid`, as old as kreg
    // Pool rows of four key tiles' keys, one tile a wave, every fourth iteration; from
    // their pages, which were fetched four iterations before
    auto rows = [&](int t) PTA_INLINE {
        const int row     = attn_page_row(a, h, attn_key0(it, t, KT) + lane, page_id);
        srow[t & 7][lane] = row;
        const uint64_t no = __ballot(row < 0);
        if (lane == 0) shole[t & 7] = no != 0;
    };
    // Keys without a row read row 0 and become zeros when they are staged.  At an
    // iteration's begin kreg, krow are of tile t + 2, vreg is of tile t + 1; each
    // register is loaded again (t + 3, t + 2) as soon as it is staged, which leaves
    // the loads a whole iteration.
    int  krow[NP], nrow[NP], srow_n = 0, khole = 0, vhole = 0, nhole = 0;
    auto piece = [&](const uint8_t *pool, int i, int row) PTA_INLINE {
        const int e = ((i * NT + tid) % CPR) * EC;
        return *reinterpret_cast<const uint4 *>(pool + (static_cast<int64_t>(max(row, 0)) * a.D + (e < a.D ? e : 0)) * ES);
    };
    auto next_rows = [&](int t) PTA_INLINE { // of the tile whose keys are loaded next
#pragma unroll
        for (int i = 0; i < NP; ++i) nrow[i] = srow[t & 7][(i * NT + tid) / CPR];
        nhole = shole[t & 7];
        if constexpr (FP8) srow_n = srow[t & 7][lane];
    };
    auto load_key = [&](int i) PTA_INLINE { kreg[i] = piece(a.kc, i, nrow[i]); };
    auto load_value = [&](int i) PTA_INLINE { vreg[i] = piece(a.vc, i, krow[i]); };
    auto load_scale = [&]() PTA_INLINE {
        if constexpr (FP8) {
            kscl = a.ks[max(srow_n, 0)];
            vscl = a.vs[max(srow_n, 0)];
        }
    };
    auto shift_rows = [&]() PTA_INLINE {
#pragma unroll
        for (int i = 0; i < NP; ++i) krow[i] = nrow[i];
        vhole = khole;
        khole = __builtin_amdgcn_readfirstlane(nhole);
    };
    auto holes = [&](int hole, int t, uint4(&r)[NP]) PTA_INLINE {
        if (a.D != DP || hole) {
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const int e = ((i * NT + tid) % CPR) * EC;
                if (srow[t & 7][(i * NT + tid) / CPR] < 0 || e >= a.D) r[i] = make_uint4(0, 0, 0, 0);
            }
        }
    };
    // tiles [calm0, calm1): every row sees every key
    int calm0 = it.n_sink, calm1 = it.n_sink;
    if (full_block) {
        const int first = a.window > 0 ? max(0, it.kend - a.window + KT - 1) / KT : 0; // key0 >= the last row's window's begin
        const int last  = (bpmin + 1) / KT;                                            // key0 + KT - 1 <= the first row's position
        calm0           = it.n_sink + max(0, first - it.lo_tile);
        calm1           = max(calm0, it.n_sink + last - it.lo_tile);
    }
    // what is rare about the keys of tile t + 2 and the values of tile t + 1, ahead of their staging
    auto ready = [&](int t) PTA_INLINE {
        holes(khole, t + 2, kreg);
        holes(vhole, t + 1, vreg);
        if (t + 1 >= it.t0 && t + 1 < it.t1 && edge(t + 1, bpmin, it.kend - 1)) {
            bool sp = false;
#pragma unroll
            for (int i = 0; i < NP; ++i)
                if (att_has_special<QT, KIND>(vreg[i])) {
                    sp      = true;
                    vreg[i] = make_uint4(0, 0, 0, 0); // slow() reads the cache's
                }
            const uint64_t any = __ballot(sp);
            if (lane == 0) sspec[(t + 1) & 1][wave] = any != 0;
        }
    };
    auto put = [&](uint16_t *row, int e, int odd, const uint4 &r) PTA_INLINE { // odd: 8, or 0
        if constexpr (FP8) {
            *reinterpret_cast<uint4 *>(row + (e ^ odd))       = att_cvt8<QT, KIND>(r.x, r.y);
            *reinterpret_cast<uint4 *>(row + (e ^ 8 ^ odd)) = att_cvt8<QT, KIND>(r.z, r.w);
        } else {
            *reinterpret_cast<uint4 *>(row + (e ^ odd)) = r;
        }
    };
    // The registers are opaque where they are staged: their conversions would
    // otherwise go to the iteration's begin, and the wait for the loads with them
    auto here = [&](uint4 &r) PTA_INLINE { asm volatile("" : "+v"(r.x), "+v"(r.y), "+v"(r.z), "+v"(r.w)); };
    auto stage_key = [&](int t, int i) PTA_INLINE {
        const int p = i * NT + tid;
        here(kreg[i]);
        put(&sk[0][0] + (t & 1) * (KT * KS) + (p / CPR) * KS, (p % CPR) * EC, 0, kreg[i]);
    };
    auto stage_value = [&](int t, int i) PTA_INLINE {
        const int p = i * NT + tid;
        here(vreg[i]);
        put(&sv[0][0] + (t & 1) * (KT * VS) + (p / CPR) * VS, (p % CPR) * EC, (p / CPR & 1) * 8, vreg[i]);
    };
    auto stage_scale = [&](int t) PTA_INLINE { // the waves share the three tables
        if constexpr (FP8) {
            asm volatile("" : "+v"(kscl), "+v"(vscl));
            const bool  no = srow[t & 7][lane] < 0;
            const float vs = no ? 1.0f : vscl;
            const float w  = wave == 0 ? (no ? 0.0f : kscl) * a.scale_log2 : wave == 1 ? att_log2_scale(vs) : __builtin_amdgcn_rcpf(att_clamp_scale(vs));
            ssc[(t + 3) % 3][min(wave, 2)][lane] = w; // the fourth writes what the third does
        }
    };
    auto stage_keys = [&](int t) PTA_INLINE {
#pragma unroll
        for (int i = 0; i < NP; ++i) stage_key(t, i);
        stage_scale(t);
    };
    // a quarter of the staging of iteration t
    auto stage = [&](int t, auto p_c) PTA_INLINE {
        constexpr int p = decltype(p_c)::value;
#pragma unroll
        for (int i = 0; i < 2 * NP; ++i)
            if (i * 4 / (2 * NP) == p) {
                if (i < NP) {
                    stage_value(t + 1, i);
                    load_value(i);
                } else {
                    stage_key(t + 2, i - NP);
                    load_key(i - NP);
                }
            }
        if (p == 3) {
            stage_scale(t + 2);
            load_scale();
        }
    };
    auto stage_all = [&](int t) PTA_INLINE { att_each<4>([&](auto p) PTA_INLINE { stage(t, p); }); };
    // operand of step i: of K(t + 1) (key block i / (DP / 16), k-step i % (DP / 16)), then of
    // V(t) (keys 16 j .. + 15, columns 32 (i % (DP / 32)) .. + 31)
    constexpr int   NQ = DP / 8; // steps of one product
    auto key_op = [&](int t, int i) PTA_INLINE {
        const uint16_t *klane = &sk[0][0] + c * KS + half * 8;
        return *reinterpret_cast<const uint4 *>(klane + (t & 1) * (KT * KS) + i / (DP / 16) * 32 * KS + i % (DP / 16) * 16);
    };
    auto value_op = [&](int t, int i) PTA_INLINE {
        const uint16_t *vlane = &sv[0][0] + (half * 4 + (lane & 15) / 4) * VS + ((lane >> 4) & 1) * 16 + ((4 * (lane & 3)) ^ (8 * ((lane >> 2) & 1)));
        const uint16_t *V = vlane + (t & 1) * (KT * VS) + i / (DP / 32) * 16 * VS + i % (DP / 32) * 32;
        const uint2     v0 = att_tr16(V), v1 = att_tr16(V + 8 * VS);
        return make_uint4(v0.x, v0.y, v1.x, v1.y);
    };
    // register 4 g + j of key block kb holds key kb * 32 + 8 g + 4 half + j; a chunk is one g
    auto key_of = [&](int kb, int g) PTA_INLINE { return kb * 32 + 8 * g + 4 * half; };
    auto scale_of = [&](int t, int which, int ch) PTA_INLINE { // of chunk ch's keys
        if constexpr (FP8) return *reinterpret_cast<const float4 *>(&ssc[t % 3][which][key_of(ch / 4, ch % 4)]);
        else return make_float4(1.f, 1.f, 1.f, 1.f);
    };

    att_f16  u[2];       // base-2 logits of the current tile
    uint32_t pf[4][4];   // its probabilities, operands of the second product
    // exponentials of registers 2 i, 2 i + 1
    auto exps = [&](auto i_c, float base, float z0, float z1) PTA_INLINE {
        constexpr int i = decltype(i_c)::value, kb = i / 8, j = i % 8 * 2;
        const float e0 = att_exp2(u[kb][j] - base), e1 = att_exp2(u[kb][j + 1] - base);
        if constexpr (FP8) l = fmaf(e1, z1, fmaf(e0, z0, l));
        else l += e0 + e1;
        uint32_t w = AttT<QT>::pack(e0, e1);
        asm volatile("" : "+v"(w), "+v"(l)); // here, and not where the product uses it
        pf[i / 4][i % 4] = w;
    };
    // chunk ch of the logits from the products s, with their maximum
    auto logits = [&](auto ch_c, const att_f16(&s)[2], const float4 &x, const float4 &y) PTA_INLINE {
        constexpr int ch = decltype(ch_c)::value, kb = ch / 4, g = ch % 4;
        float         r[4];
        if constexpr (FP8) {
            r[0] = fmaf(s[kb][4 * g], x.x, y.x);
            r[1] = fmaf(s[kb][4 * g + 1], x.y, y.y);
            r[2] = fmaf(s[kb][4 * g + 2], x.z, y.z);
            r[3] = fmaf(s[kb][4 * g + 3], x.w, y.w);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) r[j] = s[kb][4 * g + j] * a.scale_log2;
        }
        asm volatile("" : "+v"(r[0]), "+v"(r[1]), "+v"(r[2]), "+v"(r[3])); // here, and not behind the tile
        mx = att_max3(ch == 0 ? r[0] : mx, r[0], r[1]);
        mx = att_max3(mx, r[2], r[3]);
#pragma unroll
        for (int j = 0; j < 4; ++j) u[kb][4 * g + j] = r[j];
    };
    auto mask = [&](int t) PTA_INLINE {
        const int key0 = attn_key0(it, t, KT), wlo = a.window > 0 ? pos - a.window + 1 : INT_MIN;
        mx             = -INFINITY;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const int  key = key0 + key_of(kb, j / 4) + j % 4;
                const bool see = (key <= pos) & ((key >= wlo) | (key < a.sinks));
                u[kb][j]       = see ? u[kb][j] : -INFINITY;
                mx             = fmaxf(mx, u[kb][j]);
                if (j % 4 == 3) __builtin_amdgcn_sched_barrier(0); // or all comparisons come first, in SGPRs that spill
            }
    };
    // moves the reference where a tile's maximum has left it behind
    auto rescale = [&]() PTA_INLINE {
        mx             = max_xor32(mx);
        const bool far = mx > m + ATT_SLACK || (m == -INFINITY && mx > m);
        if (!__any(far)) return;
        const float n     = fmaxf(m, mx);
        const float alpha = n == -INFINITY ? 1.0f : att_exp2(m - n);
        m                 = n;
        l *= alpha;
#pragma unroll
        for (int i = 0; i < DP / 32; ++i)
#pragma unroll
            for (int j = 0; j < 16; ++j) o[i][j] *= alpha;
    };
    // Tile t key by key, for a tile in which some values are infinite or NaN and some
    // rows do not see them: 0 * inf must not reach those.  The tile's logits become
    // -inf, so that nothing of it is counted twice.
    auto slow = [&](int t) PTA_INLINE {
        const int key0 = attn_key0(it, t, KT), wlo = a.window > 0 ? pos - a.window + 1 : INT_MIN;
#pragma unroll 1
        for (int j = 0; j < KT; ++j) {
            const int       row = __builtin_amdgcn_readfirstlane(srow[t & 7][j]), key = key0 + j;
            const uint16_t *K   = &sk[0][0] + (t & 1) * (KT * KS) + j * KS + half * 8;
            float           x   = 0.0f;
#pragma unroll
            for (int s = 0; s < DP / 16; ++s) {
                const uint4 kw = *reinterpret_cast<const uint4 *>(K + s * 16), qw = qf[s];
                x += AttT<QT>::dot(kw.x, qw.x) + AttT<QT>::dot(kw.y, qw.y) + AttT<QT>::dot(kw.z, qw.z) + AttT<QT>::dot(kw.w, qw.w);
            }
            x        = add_xor32(x);
            float iv = 1.0f;
            if constexpr (FP8) {
                x  = fmaf(x, ssc[t % 3][0][j], ssc[t % 3][1][j]);
                iv = ssc[t % 3][2][j];
            } else {
                x *= a.scale_log2;
            }
            if (!(key <= pos && (key >= wlo || key < a.sinks))) continue;
            const float n = fmaxf(m, x), base = n == -INFINITY ? 0.0f : n;
            const float f = att_exp2(m - base), p = att_exp2(x - base);
            m = n;
            // each half of the wave sums its own keys: this one is the first half's
            l = fmaf(half == 0 ? p : 0.0f, iv, l * f);
#pragma unroll
            for (int i = 0; i < DP / 32; ++i)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    // outputs past D are not stored: what is in bounds does
                    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    if (row >= 0) att_values4<QT, KIND>(a.vc, static_cast<int64_t>(row) * a.D + min(i * 32 + 8 * g + 4 * half, a.D - 4), v);
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[i][4 * g + e] = fmaf(p, v[e], o[i][4 * g + e] * f);
                    __builtin_amdgcn_sched_barrier(0);
                }
        }
        mx = -INFINITY;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int j = 0; j < 16; ++j) u[kb][j] = -INFINITY;
    };
    // Tile t's exponentials and second product, with the first product and the
    // logits of tile t + 1 (behind the last tile: of what is in its place, for
    // nothing) and the staging in between.  A scheduling barrier closes each step;
    // operands and scales are read several steps ahead.
    auto tile = [&](int t) PTA_INLINE {
        att_f16 s[2];
        constexpr int R = 3; // operands in flight
        uint4   op[R];
        float4  z[2], x, y;
        const float base = m == -INFINITY ? 0.0f : m; // nothing seen yet
        z[0] = scale_of(t, 2, 0);
#pragma unroll
        for (int i = 0; i < R; ++i) op[i] = key_op(t + 1, i);
        z[1] = scale_of(t, 2, 1);
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int j = 0; j < 16; ++j) s[kb][j] = 0.0f;
        auto exp_pair = [&](auto i_c) PTA_INLINE { // pair i of 16, two a chunk
            constexpr int i = decltype(i_c)::value, ch = i / 2;
            const float4  w = z[ch & 1];
            exps(i_c, base, i % 2 ? w.z : w.x, i % 2 ? w.w : w.y);
            if (i % 2 && ch < 6) z[ch & 1] = scale_of(t, 2, ch + 2);
        };
        auto logit_chunk = [&](auto ch_c) PTA_INLINE {
            constexpr int ch = decltype(ch_c)::value;
            logits(ch_c, s, x, y);
            if (ch < 7) {
                x = scale_of(t + 1, 0, ch + 1);
                y = scale_of(t + 1, 1, ch + 1);
            }
        };
        att_each<NQ>([&](auto i_c) PTA_INLINE {
            constexpr int i = decltype(i_c)::value, kb = i / (DP / 16), k = i % (DP / 16);
            s[kb] = AttT<QT>::mfma32(op[i % R], qf[k], s[kb]);
            op[i % R] = i + R < NQ ? key_op(t + 1, i + R) : value_op(t, i + R - NQ);
            // pairs 0 .. 11 over the steps
            att_each<(i + 1) * 12 / NQ - i * 12 / NQ>([&](auto q) PTA_INLINE {
                exp_pair(std::integral_constant<int, i * 12 / NQ + decltype(q)::value>{});
            });
            if (i == NQ - 2) {
                x = scale_of(t + 1, 0, 0);
                y = scale_of(t + 1, 1, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        });
        // the rest: pairs 12 .. 15 (E) before the last quarter of the product needs them,
        // a chunk of logits (L) after its pairs are through, staging (S)
        constexpr int E = 0, L = 1, S = 2;
        constexpr int kind[16] = {E, L, S, E, L, L, E, S, L, E, L, S, L, L, S, L};
        constexpr int which[16] = {12, 0, 0, 13, 1, 2, 14, 1, 3, 15, 4, 2, 5, 6, 3, 7};
        att_each<NQ>([&](auto i_c) PTA_INLINE {
            constexpr int i = decltype(i_c)::value, ks = i / (DP / 32), d = i % (DP / 32);
            o[d] = AttT<QT>::mfma32(op[(i + NQ) % R], make_uint4(pf[ks][0], pf[ks][1], pf[ks][2], pf[ks][3]), o[d]);
            if (i + R < NQ) op[(i + NQ) % R] = value_op(t, i + R);
            att_each<(i + 1) * 16 / NQ - i * 16 / NQ>([&](auto q) PTA_INLINE {
                constexpr int w = i * 16 / NQ + decltype(q)::value;
                using W = std::integral_constant<int, which[w]>;
                if constexpr (kind[w] == E) exp_pair(W{});
                else if constexpr (kind[w] == L) logit_chunk(W{});
                else stage(t, W{});
            });
            __builtin_amdgcn_sched_barrier(0);
        });
    };

    rows(it.t0 + wave);
    fetch_pages(it.t0 + 4 + wave);
    __syncthreads();
    if (it.t0 < it.t1) {
        // tile t0 whole and the keys of t0 + 1 into LDS; then the state of an iteration's begin
        const int t = it.t0;
        auto load_keys = [&](int tt) PTA_INLINE {
            next_rows(tt);
#pragma unroll
            for (int i = 0; i < NP; ++i) load_key(i);
            load_scale();
            shift_rows();
        };
        load_keys(t);
#pragma unroll
        for (int i = 0; i < NP; ++i) load_value(i);
        holes(khole, t, kreg);
        stage_keys(t);
        load_keys(t + 1);
        ready(t - 1);
        next_rows(t + 2);
        stage_all(t - 1); // values t, keys t + 1; loads values t + 1, keys t + 2
        shift_rows();
        __syncthreads();
        if (t < tend) {
            att_f16 s[2];
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
                for (int j = 0; j < 16; ++j) s[kb][j] = 0.0f;
#pragma unroll
                for (int k = 0; k < DP / 16; ++k) s[kb] = AttT<QT>::mfma32(key_op(t, kb * (DP / 16) + k), qf[k], s[kb]);
                __builtin_amdgcn_sched_barrier(0);
            }
            att_each<8>([&](auto ch) PTA_INLINE { logits(ch, s, scale_of(t, 0, ch), scale_of(t, 1, ch)); });
            if (!full || edge(t, wpmin, wpmax)) mask(t);
        }
        // the first iteration overwrites these keys: a wave without rows begins at once
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    }
    for (int t = it.t0; t < it.t1; ++t) {
        // the lane's number anew: what derives from it (addresses in LDS and of the
        // pieces) is then made again in an iteration instead of kept in registers,
        // which all have a use: a spilled one's reload would wait for every load in flight
        lane = att_lane();
        c    = lane & 31;
        half = lane >> 5;
        tid  = wave * 64 + lane;
        next_rows(t + 3);
        const bool calm = t >= calm0 && t + 1 < calm1 && (khole | vhole) == 0 && a.D == DP;
        if (!calm) {
            ready(t);
            // the same for all waves
            if (edge(t, bpmin, it.kend - 1) && (sspec[t & 1][0] | sspec[t & 1][1] | sspec[t & 1][2] | sspec[t & 1][3])) {
                if (t < tend) slow(t);
                // it reads the keys' LDS, which this iteration's staging overwrites
                asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            }
        }
        if (t < tend) {
            rescale();
            tile(t);
            if (!calm && (!full || edge(t + 1, wpmin, wpmax))) mask(t + 1);
        } else {
            stage_all(t);
        }
        shift_rows();
        if (((t - it.t0) & 3) == 0) { // tiles t + 4 .. t + 7; the slots of t - 4 .. t - 1
            rows(t + 4 + wave);
            fetch_pages(t + 8 + wave);
        }
        // the loads stay in flight over the barrier
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    }
    l           = add_xor32(l);
    const int r = it.row0 + wave * 32 + c;
    if (r >= it.row0 + it.rows) return;
    if (it.chunks == 1) {
        const float   inv = att_inverse(l, pos < 0);
        const int     rt  = r / a.G;
        const int64_t row = static_cast<int64_t>(it.tok0 + rt) * a.Hq + h * a.G + (r - rt * a.G);
#pragma unroll
        for (int i = 0; i < DP / 32; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int d = i * 32 + 8 * g + 4 * half;
                if (d < a.D)
                    *reinterpret_cast<uint2 *>(a.out + row * a.D + d) = make_uint2(
                        AttT<QT>::pack(o[i][4 * g] * inv, o[i][4 * g + 1] * inv), AttT<QT>::pack(o[i][4 * g + 2] * inv, o[i][4 * g + 3] * inv));
            }
        if (a.lse != nullptr && half == 0) a.lse[row] = (m + att_log2(l)) * 0.69314718055994531f;
    } else {
        const int64_t at = (static_cast<int64_t>(it.part) * a.Hkv + h) * BQ + wave * 32 + c;
#pragma unroll
        for (int i = 0; i < DP / 32; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int d = i * 32 + 8 * g + 4 * half;
                if (d < a.D)
                    *reinterpret_cast<float4 *>(a.part_o + at * a.D + d) = make_float4(o[i][4 * g], o[i][4 * g + 1], o[i][4 * g + 2], o[i][4 * g + 3]);
            }
        if (half == 0) a.part_ml[at] = make_float2(att_part_max(m, pos < 0), l);
    }
}

// ---------------------------------------------------------------------------
// narrow kernel: 16 rows, four waves on 32 keys each of a key tile of 128
// ---------------------------------------------------------------------------
// Workgroup = (head, chunk, sequence), without a search: every sequence has the
// same number of chunks, of a size of its own.  Its row tiles, mostly one, go one
// after the other.  A wave keeps ST tiles of
// keys and values in flight in registers.
//
// Bound by the cache's reads in flight: 64 sequences of up to 16384 tokens, 64 / 8
// heads of 128, e4m3, take 251 to 256 us, 4.9 TB/s, what a large copy reaches (a linear
// read 6.9), and with the join 261; the wide kernel takes 730 for them, since 120 of
// its 128 rows are empty.
// With a search for the work item on the device (as in the wide kernel) and one
// tile in flight instead of two that was 284.
template <int DP> struct AttnNarrowLds {
    static constexpr int WK = 32, BQ = ATT_NARROW_ROWS;
    static constexpr int VS = DP + 16; // elements of a staged value row: the transposed read's 16 rows
                                       // of 32 bytes then fall into different banks
    static constexpr int OS = DP + 4;  // floats of a row of the waves' joined output
    static constexpr int SV_BYTES = 4 * WK * VS * 2, SO_BYTES = 4 * BQ * OS * 4;
    alignas(16) uint8_t smem[SV_BYTES > SO_BYTES ? SV_BYTES : SO_BYTES];
    alignas(16) float ssc[4][3][WK];
    float2 sml[4][BQ];
};

template <int QT, int KIND, int DP>
__device__ __forceinline__ void attn_narrow(const AttnArgs &a, int block, AttnNarrowLds<DP> &lds) {
    constexpr int  KT = ATT_NARROW_KEYS, BQ = ATT_NARROW_ROWS, WK = 32;
    constexpr bool FP8 = KIND != PTA_CACHE_16BIT;
    constexpr int  ES  = FP8 ? 1 : 2;
    constexpr int  EC  = 16 / ES;
    constexpr int  ST  = DP * ES <= 128 ? 2 : 1;
    constexpr int  KP  = DP / 4 / EC;       // 16-byte pieces of a lane's quarter of a key row
    constexpr int  CPR = DP / EC;           // pieces of a value row
    constexpr int  VP  = WK * CPR / 64;     // value pieces of a lane
    constexpr int  VS = AttnNarrowLds<DP>::VS, OS = AttnNarrowLds<DP>::OS;
    static_assert(KP >= 1, "a quarter row is a piece at least");
    auto &smem = lds.smem; auto &ssc = lds.ssc; auto &sml = lds.sml;

    const int     tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int     h = block % a.Hkv, w0 = block / a.Hkv, chunk = w0 % a.split, b = w0 / a.split;
    const AttnSeq sq   = attn_seq(a, b);
    const int     n    = __builtin_amdgcn_readfirstlane(sq.n), len = __builtin_amdgcn_readfirstlane(sq.len);
    const int     tok0 = __builtin_amdgcn_readfirstlane(sq.tok0);
    const int     c = lane & 15, qd = lane >> 4;
    uint16_t     *V = reinterpret_cast<uint16_t *>(smem) + wave * WK * VS;

    for (int row0 = 0; row0 < n * a.G; row0 += BQ) {
        AttnItem it;
        it.b    = b;
        it.row0 = row0;
        it.rows = min(BQ, n * a.G - it.row0);
        it.pos0 = len - n;
        const int total = attn_keys<KT>(a, it, len);
        const int per   = (total + a.split - 1) / a.split;
        it.t0           = min(chunk * per, total);
        it.t1           = min(it.t0 + per, total);

        const int  r    = it.row0 + c;
        const bool rin  = c < it.rows;
        const int  rtok = rin ? r / a.G : 0;
        const int  hq   = h * a.G + (rin ? r - rtok * a.G : 0);
        const int  pos  = rin ? it.pos0 + rtok : -1;
        const int  wlo  = a.window > 0 ? pos - a.window + 1 : INT_MIN;
        const bool mixed = a.window > 0 || it.row0 / a.G != (it.row0 + it.rows - 1) / a.G; // rows may see different keys

        uint4    kreg[ST][2][KP], vreg[ST][VP];
        float    scl[ST][2];
        int      krow[ST], page_id = -1;
        uint64_t hole[ST];
        auto     key = [&](int t) PTA_INLINE { return attn_key0(it, t, KT) + wave * WK + (lane & 31); };
        auto     fetch_page = [&](int t) PTA_INLINE { page_id = t < it.t1 ? attn_key_page(a, it, key(t)) : -1; };
        // loads tile t, whose pages were fetched before; keys without a row read row 0
        // and become zeros when they are used
        auto     load = [&](int t, uint4(&kr)[2][KP], uint4(&vr)[VP], float(&sc)[2], int &row, uint64_t &no) PTA_INLINE {
            row = t < it.t1 ? attn_page_row(a, h, key(t), page_id) : -1;
            no  = __ballot(row < 0);
            const int at = max(row, 0);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const uint8_t *p = a.kc + static_cast<int64_t>(__shfl(at, k * 16 + c)) * a.D * ES;
#pragma unroll
                for (int i = 0; i < KP; ++i) {
                    const int e = qd * (DP / 4) + i * EC;
                    kr[k][i]    = *reinterpret_cast<const uint4 *>(p + (e < a.D ? e : 0) * ES);
                }
            }
#pragma unroll
            for (int i = 0; i < VP; ++i) {
                const int p = i * 64 + lane, e = (p % CPR) * EC;
                vr[i]       = *reinterpret_cast<const uint4 *>(a.vc + (static_cast<int64_t>(__shfl(at, p / CPR)) * a.D + (e < a.D ? e : 0)) * ES);
            }
            if constexpr (FP8) {
                sc[0] = a.ks[at];
                sc[1] = a.vs[at];
            }
        };
        fetch_page(it.t0);
        // k-step s of the products over the head dimension takes elements
        // qd * DP / 4 + 8 s .. + 7 from quarter qd of the lanes: a lane's part of a
        // key row is one run of bytes
        uint4 qf[DP / 32];
#pragma unroll
        for (int s = 0; s < DP / 32; ++s) {
            const int d = qd * (DP / 4) + s * 8;
            qf[s]       = rin && d < a.D ? *reinterpret_cast<const uint4 *>(a.q + (tok0 + rtok) * a.q_st + hq * a.q_sh + d)
                                         : make_uint4(0, 0, 0, 0);
        }
        att_f4 o[DP / 16];
#pragma unroll
        for (int i = 0; i < DP / 16; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][j] = 0.0f;
        float m = -INFINITY, l = 0.0f;

        att_each<ST>([&](auto u_c) PTA_INLINE {
            constexpr int u = decltype(u_c)::value;
            load(it.t0 + u, kreg[u], vreg[u], scl[u], krow[u], hole[u]);
            fetch_page(it.t0 + u + 1);
        });
        for (int tt = it.t0; tt < it.t1; tt += ST)
            att_each<ST>([&](auto u_c) PTA_INLINE {
                constexpr int u = decltype(u_c)::value;
                const int     t = tt + u;
                if (u > 0 && t >= it.t1) return;
                if (a.D != DP || hole[u] != 0) {
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const bool no = __shfl(krow[u], k * 16 + c) < 0;
#pragma unroll
                        for (int i = 0; i < KP; ++i)
                            if (no || qd * (DP / 4) + i * EC >= a.D) kreg[u][k][i] = make_uint4(0, 0, 0, 0);
                    }
#pragma unroll
                    for (int i = 0; i < VP; ++i) {
                        const int p = i * 64 + lane;
                        if (__shfl(krow[u], p / CPR) < 0 || (p % CPR) * EC >= a.D) vreg[u][i] = make_uint4(0, 0, 0, 0);
                    }
                    if (krow[u] < 0) {
                        scl[u][0] = 0.0f;
                        scl[u][1] = 1.0f;
                    }
                }
                bool special = false;
                if (mixed) {
#pragma unroll
                    for (int i = 0; i < VP; ++i) special |= att_has_special<QT, KIND>(vreg[u][i]);
                    special = __any(special);
                }
                // this tile's values to LDS, its keys as operands; then the loads of the tile after next
#pragma unroll
                for (int i = 0; i < VP; ++i) {
                    const int p = i * 64 + lane, ky = p / CPR, e = (p % CPR) * EC;
                    if constexpr (FP8) {
                        *reinterpret_cast<uint4 *>(V + ky * VS + e)     = att_cvt8<QT, KIND>(vreg[u][i].x, vreg[u][i].y);
                        *reinterpret_cast<uint4 *>(V + ky * VS + e + 8) = att_cvt8<QT, KIND>(vreg[u][i].z, vreg[u][i].w);
                    } else {
                        *reinterpret_cast<uint4 *>(V + ky * VS + e) = vreg[u][i];
                    }
                }
                if constexpr (FP8) {
                    if (lane < WK) {
                        ssc[wave][0][lane] = scl[u][0] * a.scale_log2;
                        ssc[wave][1][lane] = att_log2_scale(scl[u][1]);
                        ssc[wave][2][lane] = 1.0f / att_clamp_scale(scl[u][1]);
                    }
                }
                uint4 kf[2][DP / 32];
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int s = 0; s < DP / 32; ++s) {
                        if constexpr (FP8) {
                            const uint4 w = kreg[u][k][s / 2];
                            kf[k][s] = s % 2 == 0 ? att_cvt8<QT, KIND>(w.x, w.y) : att_cvt8<QT, KIND>(w.z, w.w);
                        } else {
                            kf[k][s] = kreg[u][k][s];
                        }
                    }
                load(t + ST, kreg[u], vreg[u], scl[u], krow[u], hole[u]);
                fetch_page(t + ST + 1);
                att_f4 s[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[k][j] = 0.0f;
#pragma unroll
                    for (int i = 0; i < DP / 32; ++i) s[k] = AttT<QT>::mfma16(kf[k][i], qf[i], s[k]);
                }
                // the wave's own LDS writes are seen by its later reads once they are done
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                __builtin_amdgcn_wave_barrier();
                __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
                const int key0 = attn_key0(it, t, KT) + wave * WK;
                float     mx = m, iv[2][4];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int kk = k * 16 + 4 * qd;
                    if constexpr (FP8) {
                        const float4 x = *reinterpret_cast<const float4 *>(&ssc[wave][0][kk]);
                        const float4 y = *reinterpret_cast<const float4 *>(&ssc[wave][1][kk]);
                        const float4 z = *reinterpret_cast<const float4 *>(&ssc[wave][2][kk]);
                        s[k][0] = fmaf(s[k][0], x.x, y.x); s[k][1] = fmaf(s[k][1], x.y, y.y);
                        s[k][2] = fmaf(s[k][2], x.z, y.z); s[k][3] = fmaf(s[k][3], x.w, y.w);
                        iv[k][0] = z.x; iv[k][1] = z.y; iv[k][2] = z.z; iv[k][3] = z.w;
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; ++j) s[k][j] *= a.scale_log2;
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int  ky  = key0 + kk + j;
                        const bool see = (ky <= pos) & ((ky >= wlo) | (ky < a.sinks));
                        s[k][j]        = see ? s[k][j] : -INFINITY;
                        mx             = fmaxf(mx, s[k][j]);
                    }
                }
                mx                = max_xor32(max_xor16(mx));
                const float base  = mx == -INFINITY ? 0.0f : mx;
                const float alpha = att_exp2(m - base);
                m                 = mx;
                l *= alpha;
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        s[k][j] = att_exp2(s[k][j] - base);
                        if constexpr (FP8) l = fmaf(s[k][j], iv[k][j], l);
                        else l += s[k][j];
                    }
                const uint4 pf = make_uint4(AttT<QT>::pack(s[0][0], s[0][1]), AttT<QT>::pack(s[0][2], s[0][3]),
                                            AttT<QT>::pack(s[1][0], s[1][1]), AttT<QT>::pack(s[1][2], s[1][3]));
                const int   kr = 4 * qd + c / 4, dc = 4 * (c & 3);
#pragma unroll
                for (int i = 0; i < DP / 16; ++i) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[i][j] *= alpha;
                    const uint2 v0 = att_tr16(V + kr * VS + i * 16 + dc), v1 = att_tr16(V + (kr + 16) * VS + i * 16 + dc);
                    const uint4 vf = make_uint4(v0.x, v0.y, v1.x, v1.y);
                    if (!special) {
                        o[i] = AttT<QT>::mfma16(vf, pf, o[i]);
                    } else {
                        // infinities and NaN that only some rows see: 0 * inf must not reach the
                        // others.  Finite values go as ever; then a count of the special ones that
                        // a row sees decides.
                        uint4  fin, plus, minus;
                        att_f4 np = {0.f, 0.f, 0.f, 0.f}, nm = {0.f, 0.f, 0.f, 0.f};
                        att_split_special<QT>(vf, fin, plus, minus);
                        const uint4 seen = att_nonzero<QT>(pf);
                        o[i] = AttT<QT>::mfma16(fin, pf, o[i]);
                        np   = AttT<QT>::mfma16(plus, seen, np);
                        nm   = AttT<QT>::mfma16(minus, seen, nm);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            if (np[j] > 0.0f) o[i][j] += INFINITY;
                            if (nm[j] > 0.0f) o[i][j] -= INFINITY;
                        }
                    }
                }
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                __builtin_amdgcn_wave_barrier();
                __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            });
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
        if (jr < it.rows) {
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
            const int     rr = it.row0 + jr, rt = rr / a.G;
            const int64_t orow = static_cast<int64_t>(tok0 + rt) * a.Hq + h * a.G + (rr - rt * a.G);
            if (a.split == 1) {
                const float inv = att_inverse(ll, it.pos0 + rt < 0);
#pragma unroll
                for (int e = 0; e < DPT; e += 4)
                    if (jd + e < a.D)
                        *reinterpret_cast<uint2 *>(a.out + orow * a.D + jd + e) =
                            make_uint2(AttT<QT>::pack(acc[e] * inv, acc[e + 1] * inv), AttT<QT>::pack(acc[e + 2] * inv, acc[e + 3] * inv));
                if (a.lse != nullptr && jd == 0) a.lse[orow] = (mm + att_log2(ll)) * 0.69314718055994531f;
            } else {
                const int64_t at = static_cast<int64_t>(chunk) * a.part_step + (a.part_seq ? (b * a.Hkv + h) * BQ + rr : orow);
#pragma unroll
                for (int e = 0; e < DPT; e += 4)
                    if (jd + e < a.D)
                        *reinterpret_cast<float4 *>(a.part_o + at * a.D + jd + e) = make_float4(acc[e], acc[e + 1], acc[e + 2], acc[e + 3]);
                if (jd == 0) a.part_ml[at] = make_float2(att_part_max(mm, it.pos0 + rt < 0), ll);
            }
        }
        __syncthreads(); // the outputs' LDS becomes the values' of the next row tile
    }
}

// ---------------------------------------------------------------------------
// the kernels: one form alone, or in one launch the wide form's workgroups, which
// take longest, and behind them the narrow form's
// ---------------------------------------------------------------------------
// Their last `pads` workgroups take the tokens that no sequence owns, ahead of the
// first and behind the last: zeros and -inf, like tokens that see no key.
__device__ __forceinline__ void attn_pad(const AttnArgs &a, int part, int parts) {
    const int     first = min(max(a.cu[0], 0), a.Tq), last = min(max(a.cu[a.B], first), a.Tq);
    const int     per = a.Hq * (a.D / 8); // 16-byte pieces of a token
    const int64_t tokens = a.Tq - (last - first);
    for (int64_t p = part * 256 + threadIdx.x; p < tokens * per; p += parts * 256) {
        const int64_t t = p / per, row = t < first ? t : t - first + last;
        reinterpret_cast<uint4 *>(a.out)[row * per + (p - t * per)] = make_uint4(0, 0, 0, 0);
    }
    if (a.lse == nullptr) return;
    for (int64_t p = part * 256 + threadIdx.x; p < tokens * a.Hq; p += parts * 256) {
        const int64_t t = p / a.Hq, row = t < first ? t : t - first + last;
        a.lse[row * a.Hq + (p - t * a.Hq)] = -INFINITY;
    }
}

template <int QT, int KIND, int DP> __global__ __launch_bounds__(256, DP <= 128 ? 2 : 1) void attn_wide_kernel(AttnArgs a, int pads) {
    __shared__ AttnWideLds<KIND, DP> lds;
    const int block = blockIdx.x, work = gridDim.x - pads;
    if (block < work) attn_wide<QT, KIND, DP>(a, block, lds);
    else attn_pad(a, block - work, pads);
}
template <int QT, int KIND, int DP> __global__ __launch_bounds__(256, DP <= 128 ? 2 : 1) void attn_narrow_kernel(AttnArgs a, int pads) {
    __shared__ AttnNarrowLds<DP> lds;
    const int block = blockIdx.x, work = gridDim.x - pads;
    if (block < work) attn_narrow<QT, KIND, DP>(a, block, lds);
    else attn_pad(a, block - work, pads);
}
template <int QT, int KIND, int DP>
__global__ __launch_bounds__(256, DP <= 128 ? 2 : 1) void attn_both_kernel(AttnArgs w, AttnArgs n, int w_blocks, int pads) {
    __shared__ union Lds {
        AttnWideLds<KIND, DP> w;
        AttnNarrowLds<DP>     n;
        __device__ Lds() {}
    } lds;
    const int block = blockIdx.x, work = gridDim.x - pads;
    if (block < w_blocks) attn_wide<QT, KIND, DP>(w, block, lds.w);
    else if (block < work) attn_narrow<QT, KIND, DP>(n, block - w_blocks, lds.n);
    else attn_pad(n, block - work, pads);
}

// ---------------------------------------------------------------------------
// joins the chunks of both kernels: o = sum_c 2^(m_c - m) O_c / sum_c 2^(m_c - m) l_c
// ---------------------------------------------------------------------------
// An element is 4 values of a row; Q threads share its chunks, which a thread adds
// one after the other.  Bound by that chain of reads and the parts' bytes, 4 D + 8 a
// row and chunk: a batch of chunks of up to 256 tokens, 32 heads of 128, takes 10 us.
// The narrow form's parts have one thread an element where chunks are few (four
// threads: 17 us), four beyond four chunks; the wide form's always one, which a row
// tile of a hundred chunks pays for (35 tokens over 21119, 8 / 2 heads: 103 us a call).
template <int QT, int Q> __device__ __forceinline__ void attn_join(const AttnArgs &a, const AttnSeq &s, int h, int row0, int rows,
                                                                   bool by_token, int64_t at0, int64_t stride, int count, int part, int parts) {
    constexpr int N = 256 / Q; // elements of a workgroup at a time
    __shared__ float4 sacc[Q][N];
    __shared__ float2 sml[Q][N];
    const int tpr = a.D / 4, lane = threadIdx.x % N, quarter = threadIdx.x / N;
    for (int64_t p0 = part * N; p0 < static_cast<int64_t>(rows) * tpr; p0 += parts * N) {
        const int64_t p = p0 + lane;
        const bool    in = p < static_cast<int64_t>(rows) * tpr;
        const int     jr = in ? static_cast<int>(p / tpr) : rows - 1, d = in ? static_cast<int>(p - static_cast<int64_t>(jr) * tpr) * 4 : 0;
        const int     rr = row0 + jr, rt = rr / a.G;
        const int64_t orow = static_cast<int64_t>(s.tok0 + rt) * a.Hq + h * a.G + (rr - rt * a.G);
        const int64_t first = by_token ? orow : at0 + jr;
        float         mm = -INFINITY, ll = 0.0f;
        float4        acc = make_float4(0.f, 0.f, 0.f, 0.f);
        auto add = [&](const float2 &ml, const float4 &x) PTA_INLINE {
            const float n = fmaxf(mm, ml.x), base = n == -INFINITY ? 0.0f : n;
            const float f = att_exp2(mm - base), g = att_exp2(ml.x - base);
            mm    = n;
            ll    = fmaf(ml.y, g, ll * f);
            acc.x = fmaf(x.x, g, acc.x * f); acc.y = fmaf(x.y, g, acc.y * f);
            acc.z = fmaf(x.z, g, acc.z * f); acc.w = fmaf(x.w, g, acc.w * f);
        };
        for (int c0 = quarter; c0 < count; c0 += 4 * Q) {
            float2 ml[4];
            float4 x[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int64_t at = min(c0 + Q * u, count - 1) * stride + first;
                ml[u]            = a.part_ml[at];
                x[u]             = *reinterpret_cast<const float4 *>(a.part_o + at * a.D + d);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (c0 + Q * u >= count) break;
                add(ml[u], x[u]);
            }
        }
        if constexpr (Q > 1) {
            __syncthreads();
            sacc[quarter][lane] = acc;
            sml[quarter][lane]  = make_float2(mm, ll);
            __syncthreads();
        }
        if (quarter != 0 || !in) continue;
        if constexpr (Q > 1) {
#pragma unroll
            for (int u = 1; u < Q; ++u) add(sml[u][lane], sacc[u][lane]);
        }
        const float inv = att_inverse(ll, ll == 0.0f && mm > -INFINITY);
        *reinterpret_cast<uint2 *>(a.out + orow * a.D + d) =
            make_uint2(AttT<QT>::pack(acc.x * inv, acc.y * inv), AttT<QT>::pack(acc.z * inv, acc.w * inv));
        if (a.lse != nullptr && d == 0) a.lse[orow] = (mm + att_log2(ll)) * 0.69314718055994531f;
    }
}

// Workgroups of the narrow kernel's sequences (head, part, sequence), then of the
// wide kernel's slots (head, part, slot).
constexpr int ATT_JOIN_PARTS = 8;

template <int QT, int QN> __global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs n, AttnArgs w, int n_blocks, int n_parts) {
    if (static_cast<int>(blockIdx.x) < n_blocks) {
        const int     h = blockIdx.x % n.Hkv, g = blockIdx.x / n.Hkv;
        const AttnSeq s = attn_seq(n, g / n_parts);
        attn_join<QT, QN>(n, s, h, 0, s.n * n.G, !n.part_seq, (static_cast<int64_t>(g / n_parts) * n.Hkv + h) * ATT_NARROW_ROWS, n.part_step,
                          n.split, g % n_parts, n_parts);
    } else {
        const int  x = blockIdx.x - n_blocks, h = x % w.Hkv, g = x / w.Hkv, slot = g / ATT_JOIN_PARTS;
        const int4 d = w.desc[slot]; // sequence, row tile, first part, chunks
        if (d.z < 0) return;
        const AttnSeq s    = attn_seq(w, d.x);
        const int     row0 = d.y * ATT_WIDE_ROWS;
        attn_join<QT, 1>(w, s, h, row0, min(ATT_WIDE_ROWS, s.n * w.G - row0), false, (static_cast<int64_t>(d.z) * w.Hkv + h) * ATT_WIDE_ROWS,
                      static_cast<int64_t>(w.Hkv) * ATT_WIDE_ROWS, d.w, g % ATT_JOIN_PARTS, ATT_JOIN_PARTS);
    }
}

// One call's launches for one type of queries (paged_attention_inst_*.hip).
struct AttnCall {
    AttnArgs narrow, wide;
    bool     has_narrow, has_wide;
    int      narrow_join_parts; // workgroups of a sequence's head that join its chunks
    int      pads;              // workgroups for the tokens of no sequence
};
template <int QT> void attn_launch(const AttnCall &c, int kind, hipStream_t st);
extern template void attn_launch<PTA_BF16>(const AttnCall &, int, hipStream_t);
extern template void attn_launch<PTA_F16>(const AttnCall &, int, hipStream_t);

} // namespace pta
