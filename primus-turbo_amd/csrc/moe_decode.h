// SwiGLU experts for the few tokens of a decoding step, in two kernels:
//
//   a_te = p_te * silu(Wg_e x_t) * (Wu_e x_t)        p_te = sum of token t's probs for expert e
//   y_t  = sum_e Wd_e a_te
//
// with the weights as they were quantized once (e4m3 / e5m2 with one scale for
// the tensor, for each row or for each 128 x 128 block) or in 16 bits.  What the
// call cannot do without is every reached expert's weights once; at up to 64
// tokens their read bounds it, so no weight is read twice and nothing but x, a
// and y moves beside them.
//
// The weights are the first operand of the matrix instructions (rows: output
// features), the tokens the second (16 columns; up to 4 column tiles), so all
// tokens of a step go along with one read of the weights.  fp8 converts exactly
// to the tokens' 16-bit type; the scales are applied to fp32 sums.  The
// contraction takes a step's elements in the order in which a lane has them in
// one run of 32 bytes: a row's step is one 128-byte line.
//
// a is rounded to the tokens' type between the kernels, its probability
// included, as a layer that runs its two products apart does.  Sums over an
// expert's and over the experts' products are fp32, in an order that depends on
// the sizes and the routing alone.
#pragma once

#include "paged_attention.h"

namespace pta {

constexpr int MOE_TG = 64, MOE_MAX_E = 1024, MOE_MAX_K = 32, MOE_NT = 256;

enum MoeScale { MOE_NONE = 0, MOE_TENSOR = 1, MOE_ROW = 2, MOE_BLOCK = 3 };

struct MoeArgs {
    const uint16_t *x;
    int64_t         x_st;
    const uint8_t  *w1, *w2; // [E, 2I, H], [E, H, I]
    const float    *s1, *s2;
    const void     *idx;     // [T, k] int32 or int64
    int             idx_i64;
    const float    *probs;   // [T, k]
    uint16_t       *act;     // [groups, S, TG, I]
    uint16_t       *y;       // [T, H]
    int             T, E, k, I, H, S, TG;
    int             by_entry; // slots are entries of the index rows (few tokens) instead of experts
    int             scale;    // MoeScale
};

__device__ __forceinline__ int moe_expert(const MoeArgs &a, int64_t at) {
    const int64_t e = a.idx_i64 ? reinterpret_cast<const int64_t *>(a.idx)[at]
                                : static_cast<int64_t>(reinterpret_cast<const int32_t *>(a.idx)[at]);
    return e >= 0 && e < a.E ? static_cast<int>(e) : -1;
}

// 32 bytes of a lane's part of a weight row's step as operands
template <int XT, int KIND> struct MoeFrag {
    static constexpr int ES = KIND == PTA_CACHE_16BIT ? 2 : 1, EL = 32 / ES, NS = EL / 8, STEP = 4 * EL;
    uint4                w[2];
    __device__ __forceinline__ void load(const uint8_t *row, int k, int K) { // row null: zeros
        w[0] = w[1] = make_uint4(0, 0, 0, 0);
        if (row != nullptr) {
            if (k < K) w[0] = *reinterpret_cast<const uint4 *>(row + static_cast<int64_t>(k) * ES);
            if (k + EL / 2 < K) w[1] = *reinterpret_cast<const uint4 *>(row + static_cast<int64_t>(k) * ES + 16);
        }
    }
    __device__ __forceinline__ uint4 get(int s) const {
        if constexpr (ES == 2) return w[s];
        else return s % 2 == 0 ? att_cvt8<XT, KIND>(w[s / 2].x, w[s / 2].y) : att_cvt8<XT, KIND>(w[s / 2].z, w[s / 2].w);
    }
};

template <int NS> struct MoeTok {
    uint4 v[NS];
    __device__ __forceinline__ void load(const uint16_t *row, int k, int K) { // row null: zeros
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            v[s] = make_uint4(0, 0, 0, 0);
            if (row != nullptr && k + 8 * s < K) v[s] = *reinterpret_cast<const uint4 *>(row + k + 8 * s);
        }
    }
};

// ---------------------------------------------------------------------------
// gate and up products: workgroup = (32 features, slot, group of 64 tokens);
// the waves take every fourth step
// ---------------------------------------------------------------------------
template <int XT, int KIND, int NC> __global__ __launch_bounds__(MOE_NT, 2) void moe_up_kernel(MoeArgs a) {
    using F = MoeFrag<XT, KIND>;
    __shared__ float    sred[4][NC][4][256]; // wave, column tile, row tile, 16 x 16
    __shared__ float    sprob[MOE_TG];
    __shared__ uint64_t smask;
    __shared__ int      sexp;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int slot = blockIdx.y, g = blockIdx.z, t0 = g * MOE_TG, tl = min(MOE_TG, a.T - t0);

    if (wave == 0) {
        int e = slot;
        if (a.by_entry) e = slot < tl * a.k ? moe_expert(a, static_cast<int64_t>(t0) * a.k + slot) : -1;
        float p    = 0.0f;
        int   mine = -1; // the token's first entry for this expert
        if (lane < tl && e >= 0) {
            for (int j = a.k - 1; j >= 0; --j) {
                const int64_t at = static_cast<int64_t>(t0 + lane) * a.k + j;
                if (moe_expert(a, at) == e) {
                    mine = lane * a.k + j;
                    p += a.probs[at];
                }
            }
        }
        const uint64_t mask = __ballot(mine >= 0);
        // an expert that several entries name belongs to the first
        const int first = mask ? __shfl(mine, __ffsll(static_cast<unsigned long long>(mask)) - 1) : -1;
        sprob[lane]     = p;
        if (lane == 0) {
            smask = mask;
            sexp  = mask && (!a.by_entry || first == slot) ? e : -1;
        }
    }
    __syncthreads();
    const int      e    = sexp;
    const uint64_t mask = smask;
    if (e < 0) return;

    const int      c = lane & 15, qd = lane >> 4, i0 = blockIdx.x * 32;
    const int      K = a.H, steps = (K + F::STEP - 1) / F::STEP;
    const int64_t  rowb = static_cast<int64_t>(K) * F::ES;
    const uint8_t *row[4]; // gate rows, then up rows
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int i = i0 + (r & 1) * 16 + c;
        row[r]      = i < a.I ? a.w1 + (static_cast<int64_t>(e) * 2 * a.I + (r >> 1) * a.I + i) * rowb : nullptr;
    }
    const uint16_t *tok[NC];
    bool            tile[NC]; // some token of the tile goes to this expert
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        tok[n]  = mask >> (n * 16 + c) & 1 ? a.x + (t0 + n * 16 + c) * a.x_st : nullptr;
        tile[n] = (mask >> (n * 16) & 0xffff) != 0;
    }
    att_f4 acc[NC][4];
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[n][r][j] = 0.0f;

    const bool     block = a.scale == MOE_BLOCK;
    const int      nkb = (K + 127) / 128, nrb = (2 * a.I + 127) / 128;
    const float   *bs = block ? a.s1 + static_cast<int64_t>(e) * nrb * nkb : nullptr;
    F              wf[4], wn[4];
    MoeTok<F::NS>  xf[NC], xn[NC];
    auto           fetch = [&](int st, F(&w)[4], MoeTok<F::NS>(&x)[NC]) {
        const int k = st * F::STEP + qd * F::EL;
#pragma unroll
        for (int r = 0; r < 4; ++r) w[r].load(row[r], k, K);
#pragma unroll
        for (int n = 0; n < NC; ++n)
            if (tile[n]) x[n].load(tok[n], k, K);
    };
    if (wave < steps) fetch(wave, wf, xf);
    for (int st = wave; st < steps; st += 4) {
        const bool more = st + 4 < steps;
        if (more) fetch(st + 4, wn, xn);
        att_f4 part[NC][4];
#pragma unroll
        for (int n = 0; n < NC; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int j = 0; j < 4; ++j) part[n][r][j] = 0.0f;
#pragma unroll
        for (int s = 0; s < F::NS; ++s)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint4 wv = wf[r].get(s);
#pragma unroll
                for (int n = 0; n < NC; ++n)
                    if (tile[n]) part[n][r] = AttT<XT>::mfma16(wv, xf[n].v[s], part[n][r]);
            }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            // 16 rows lie in one block: I is a multiple of 16
            const int ib = i0 + (r & 1) * 16;
            float     sc = 1.0f;
            if (block && ib < a.I) sc = bs[static_cast<int64_t>(((r >> 1) * a.I + ib) / 128) * nkb + st];
#pragma unroll
            for (int n = 0; n < NC; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[n][r][j] = fmaf(part[n][r][j], sc, acc[n][r][j]);
        }
        if (more) {
#pragma unroll
            for (int r = 0; r < 4; ++r) wf[r] = wn[r];
#pragma unroll
            for (int n = 0; n < NC; ++n) xf[n] = xn[n];
        }
    }
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) // [token][feature]: a lane's four features in a row
            *reinterpret_cast<float4 *>(&sred[wave][n][r][c * 16 + 4 * qd]) =
                make_float4(acc[n][r][0], acc[n][r][1], acc[n][r][2], acc[n][r][3]);
    __syncthreads();
    // 8 features of one token a thread
    for (int p = tid; p < NC * 16 * 4; p += MOE_NT) {
        const int tt = p >> 2, f = (p & 3) * 8, n = tt >> 4; // token, first feature
        const int i = i0 + f;
        if (!(mask >> tt & 1) || i >= a.I) continue;
        const int at = (tt & 15) * 16 + (f & 15), u = f >> 4;
        float     v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float gate = 0.0f, up = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                gate += sred[w][n][u][at + j];
                up += sred[w][n][2 + u][at + j];
            }
            if (a.scale == MOE_TENSOR) {
                gate *= a.s1[0];
                up *= a.s1[0];
            } else if (a.scale == MOE_ROW) {
                gate *= a.s1[static_cast<int64_t>(e) * 2 * a.I + i + j];
                up *= a.s1[static_cast<int64_t>(e) * 2 * a.I + a.I + i + j];
            }
            v[j] = gate / (1.0f + att_exp2(gate * -1.4426950408889634f)) * up * sprob[tt];
        }
        *reinterpret_cast<uint4 *>(a.act + ((static_cast<int64_t>(g) * a.S + slot) * a.TG + tt) * a.I + i) =
            make_uint4(AttT<XT>::pack(v[0], v[1]), AttT<XT>::pack(v[2], v[3]), AttT<XT>::pack(v[4], v[5]), AttT<XT>::pack(v[6], v[7]));
    }
}

// ---------------------------------------------------------------------------
// down product and the sum over experts: workgroup = (32 features, group of 64
// tokens); the waves take every fourth step of the list of all reached experts'
// steps
// ---------------------------------------------------------------------------
template <int XT, int KIND, int NC> __global__ __launch_bounds__(MOE_NT, 2) void moe_down_kernel(MoeArgs a) {
    using F = MoeFrag<XT, KIND>;
    __shared__ float              sred[4][NC][2][256];
    __shared__ unsigned long long smask[MOE_MAX_E]; // tokens of a slot
    __shared__ int                sfirst[MOE_MAX_E]; // by entry: an expert's slot; afterwards: list of reached slots
    __shared__ int                sexp[MOE_MAX_E];   // expert of a listed slot
    __shared__ int                scount;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int g = blockIdx.y, t0 = g * MOE_TG, tl = min(MOE_TG, a.T - t0), n_ent = tl * a.k;
    const int64_t ent0 = static_cast<int64_t>(t0) * a.k;

    for (int i = tid; i < a.S; i += MOE_NT) smask[i] = 0;
    if (a.by_entry) {
        for (int i = tid; i < a.E; i += MOE_NT) sfirst[i] = INT_MAX;
        __syncthreads();
        for (int i = tid; i < n_ent; i += MOE_NT) {
            const int e = moe_expert(a, ent0 + i);
            if (e >= 0) atomicMin(&sfirst[e], i);
        }
    }
    __syncthreads();
    for (int i = tid; i < n_ent; i += MOE_NT) {
        const int e = moe_expert(a, ent0 + i);
        if (e >= 0) atomicOr(&smask[a.by_entry ? sfirst[e] : e], 1ull << (i / a.k));
    }
    __syncthreads();
    if (wave == 0) {
        int n = 0;
        for (int s0 = 0; s0 < a.S; s0 += 64) {
            const int      s  = s0 + lane;
            const bool     in = s < a.S && smask[s] != 0;
            const uint64_t b  = __ballot(in);
            if (in) {
                const int at = n + __popcll(b & ((1ull << lane) - 1));
                sexp[at]     = a.by_entry ? moe_expert(a, ent0 + s) : s;
                sfirst[at]   = s;
            }
            n += __popcll(b);
        }
        if (lane == 0) scount = n;
    }
    __syncthreads();

    const int c = lane & 15, qd = lane >> 4, h0 = blockIdx.x * 32;
    const int K = a.I, steps = (K + F::STEP - 1) / F::STEP, items = scount * steps;
    const int nkb = (K + 127) / 128, nrb = (a.H + 127) / 128;
    const int64_t rowb = static_cast<int64_t>(K) * F::ES;
    att_f4 acc[NC][2];
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[n][r][j] = 0.0f;
    F             wf[2], wn[2];
    MoeTok<F::NS> xf[NC], xn[NC];
    auto          fetch = [&](int it, F(&w)[2], MoeTok<F::NS>(&x)[NC]) {
        const int      li = it / steps, st = it - li * steps, e = sexp[li], s = sfirst[li];
        const uint64_t mask = smask[s];
        const int      k    = st * F::STEP + qd * F::EL;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int h = h0 + r * 16 + c;
            w[r].load(h < a.H ? a.w2 + (static_cast<int64_t>(e) * a.H + h) * rowb : nullptr, k, K);
        }
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            const int tt = n * 16 + c;
            x[n].load(mask >> tt & 1 ? a.act + ((static_cast<int64_t>(g) * a.S + s) * a.TG + tt) * a.I : nullptr, k, K);
        }
    };
    if (wave < items) fetch(wave, wf, xf);
    for (int it = wave; it < items; it += 4) {
        const bool more = it + 4 < items;
        if (more) fetch(it + 4, wn, xn);
        const int      li = it / steps, st = it - li * steps, e = sexp[li];
        const uint64_t mask = smask[sfirst[li]];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int hb = h0 + r * 16;
            float     sc[4] = {1.0f, 1.0f, 1.0f, 1.0f};
            if (a.scale == MOE_TENSOR) sc[0] = sc[1] = sc[2] = sc[3] = a.s2[0];
            else if (a.scale == MOE_BLOCK) {
                if (hb < a.H) sc[0] = sc[1] = sc[2] = sc[3] = a.s2[(static_cast<int64_t>(e) * nrb + hb / 128) * nkb + st];
            } else if (a.scale == MOE_ROW) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (hb + 4 * qd + j < a.H) sc[j] = a.s2[static_cast<int64_t>(e) * a.H + hb + 4 * qd + j];
            }
            att_f4 part[NC];
#pragma unroll
            for (int n = 0; n < NC; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) part[n][j] = 0.0f;
#pragma unroll
            for (int s = 0; s < F::NS; ++s) {
                const uint4 wv = wf[r].get(s);
#pragma unroll
                for (int n = 0; n < NC; ++n)
                    if (mask >> (n * 16) & 0xffff) part[n] = AttT<XT>::mfma16(wv, xf[n].v[s], part[n]);
            }
            // a token that does not go to this expert has nothing of it, not even 0 * NaN
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                const bool in = mask >> (n * 16 + c) & 1;
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[n][r][j] = in ? fmaf(part[n][j], sc[j], acc[n][r][j]) : acc[n][r][j];
            }
        }
        if (more) {
#pragma unroll
            for (int r = 0; r < 2; ++r) wf[r] = wn[r];
#pragma unroll
            for (int n = 0; n < NC; ++n) xf[n] = xn[n];
        }
    }
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
        for (int r = 0; r < 2; ++r)
            *reinterpret_cast<float4 *>(&sred[wave][n][r][c * 16 + 4 * qd]) =
                make_float4(acc[n][r][0], acc[n][r][1], acc[n][r][2], acc[n][r][3]);
    __syncthreads();
    for (int p = tid; p < NC * 16 * 4; p += MOE_NT) {
        const int tt = p >> 2, f = (p & 3) * 8, n = tt >> 4;
        if (tt >= tl || h0 + f >= a.H) continue;
        const int at = (tt & 15) * 16 + (f & 15), r = f >> 4;
        float     v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[j] = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; ++w) v[j] += sred[w][n][r][at + j];
        }
        *reinterpret_cast<uint4 *>(a.y + static_cast<int64_t>(t0 + tt) * a.H + h0 + f) =
            make_uint4(AttT<XT>::pack(v[0], v[1]), AttT<XT>::pack(v[2], v[3]), AttT<XT>::pack(v[4], v[5]), AttT<XT>::pack(v[6], v[7]));
    }
}

} // namespace pta
