// SwiGLU experts for the few tokens of a decoding step, in two kernels:
//
//   a_te = p_te * silu(Wg_e x_t) * (Wu_e x_t)        p_te = sum of token t's probs for expert e
//   y_t  = sum_e Wd_e a_te
//
// with the weights as they were quantized once (e4m3 / e5m2 with one scale for
// the tensor, for each row or for each 128 x 128 block) or in 16 bits.  What the
// call cannot do without is every reached expert's weights once; at up to 64
// tokens their read bounds it, so no weight is read twice from memory and nothing but x, a
// and y moves beside them.
//
// The weights are the first operand of the matrix instructions (rows: output
// features), the tokens that go to the expert the second (column tiles of 16, up
// to 4), so all of them go along with one read of the weights.  fp8 converts
// exactly to the tokens' 16-bit type; the scales are applied to fp32 sums.  A
// step is 128 bytes of every row, two 16-byte pieces a lane with the 4 lanes of a
// row side by side; the contraction takes the elements in that order.
//
// Measured, 32 experts of 2048 x 7168, top 8, e4m3: one token 79 us (352 MB, up 48 at
// 4.8 TB/s, down 31 at 3.7), 64 tokens 347 (1.41 GB: up 217 at 4.3 TB/s, down 137 at
// 3.4); a linear read reaches 6.9.  Up to 16 tokens the down product takes 16 rows a workgroup and a ring of
// four (more workgroups where latency counts), beyond 32 rows, whose tokens' operands
// are then used twice.
//
// Loads are unconditional (rows, columns and pieces that do not exist read ones
// that do, and their products are not stored or meet a zero), so that a ring of
// register stages keeps several steps in flight.
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
    uint16_t       *act;     // [groups, rows, I]: an expert's tokens one after the other
    uint16_t       *y;       // [T, H]
    int             T, E, k, I, H, S, TG;
    int             by_entry; // slots are entries of the index rows (few tokens) instead of experts
    int             rows;     // of a group in act
    int             packed;   // an expert's rows begin behind the entries of those before; else at slot * TG
    int             scale;    // MoeScale
};

__device__ __forceinline__ int moe_expert(const MoeArgs &a, int64_t at) {
    const int64_t e = a.idx_i64 ? reinterpret_cast<const int64_t *>(a.idx)[at]
                                : static_cast<int64_t>(reinterpret_cast<const int32_t *>(a.idx)[at]);
    return e >= 0 && e < a.E ? static_cast<int>(e) : -1;
}

// A step of one weight row: two pieces of 16 bytes
template <int XT, int KIND> struct MoeFrag {
    static constexpr int ES = KIND == PTA_CACHE_16BIT ? 2 : 1, EP = 16 / ES, NS = 2 * EP / 8, STEP = 8 * EP;
    uint4                w[2];
    __device__ __forceinline__ void load(const uint8_t *row, int k0, int qd, int K) {
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            const int k = k0 + p * 4 * EP + qd * EP;
            w[p]        = *reinterpret_cast<const uint4 *>(row + static_cast<int64_t>(k < K ? k : 0) * ES);
        }
    }
    __device__ __forceinline__ uint4 get(int s) const {
        if constexpr (ES == 2) return w[s];
        else return s % 2 == 0 ? att_cvt8<XT, KIND>(w[s / 2].x, w[s / 2].y) : att_cvt8<XT, KIND>(w[s / 2].z, w[s / 2].w);
    }
    __device__ __forceinline__ void cut(int k0, int qd, int K) {
#pragma unroll
        for (int p = 0; p < 2; ++p)
            if (k0 + p * 4 * EP + qd * EP >= K) w[p] = make_uint4(0, 0, 0, 0);
    }
    // first element of operand s in the step, for quarter qd
    static __device__ __forceinline__ int elem(int s, int qd) { return ES == 2 ? s * 32 + qd * 8 : (s / 2) * 64 + qd * 16 + (s % 2) * 8; }
};

// The same step of one token row.  Elements past K become zeros where they are
// used (an instruction after the load would wait for it), of weights too: what
// was read in their place may be infinite.
template <class F> struct MoeTok {
    uint4 v[F::NS];
    __device__ __forceinline__ void load(const uint16_t *row, int k0, int qd, int K) {
#pragma unroll
        for (int s = 0; s < F::NS; ++s) {
            const int k = k0 + F::elem(s, qd);
            v[s]        = *reinterpret_cast<const uint4 *>(row + (k < K ? k : 0));
        }
    }
    __device__ __forceinline__ void cut(int k0, int qd, int K) {
#pragma unroll
        for (int s = 0; s < F::NS; ++s)
            if (k0 + F::elem(s, qd) >= K) v[s] = make_uint4(0, 0, 0, 0);
    }
};

template <class F, int RT, int NC> struct MoeStage {
    F         w[RT];
    MoeTok<F> x[NC];
    float     sc[RT]; // block scales
    __device__ __forceinline__ void cut(int k0, int qd, int K) {
#pragma unroll
        for (int r = 0; r < RT; ++r) w[r].cut(k0, qd, K);
#pragma unroll
        for (int n = 0; n < NC; ++n) x[n].cut(k0, qd, K);
    }
};

__device__ __forceinline__ int moe_uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// ---------------------------------------------------------------------------
// gate and up products: workgroup = (32 features, slot, group of 64 tokens);
// the waves take every fourth step
// ---------------------------------------------------------------------------
struct MoeUpShared {
    float    red[4 * 4 * 4 * 256]; // wave, column tile, row tile, 16 x 16
    float    prob[MOE_TG];
    int      tok[MOE_TG]; // the expert's tokens
    int      n, expert, row0; // row0: its first row in act
};

// One pass over K: PR pairs of (gate, up) row tiles from pair p0 on, NC column tiles.
template <int XT, int KIND, int PR, int NC, int RING>
__device__ __forceinline__ void moe_up_pass(const MoeArgs &a, MoeUpShared &sh, int p0, int i0, int t0) {
    using F = MoeFrag<XT, KIND>;
    const int      lane = threadIdx.x & 63, wave = moe_uniform(threadIdx.x >> 6), c = lane & 15, qd = lane >> 4;
    const int      e = moe_uniform(sh.expert);
    const int      K = a.H, steps = (K + F::STEP - 1) / F::STEP;
    const int64_t  rowb = static_cast<int64_t>(K) * F::ES;
    const uint8_t *row[2 * PR]; // gate rows, then up rows
#pragma unroll
    for (int r = 0; r < 2 * PR; ++r) {
        const int i = min(i0 + (p0 + r % PR) * 16 + c, a.I - 1);
        row[r]      = a.w1 + (static_cast<int64_t>(e) * 2 * a.I + (r / PR) * a.I + i) * rowb;
    }
    const uint16_t *tok[NC];
#pragma unroll
    for (int n = 0; n < NC; ++n) tok[n] = a.x + (t0 + sh.tok[min(n * 16 + c, sh.n - 1)]) * a.x_st;
    const bool block = a.scale == MOE_BLOCK;
    const int  nkb = (K + 127) / 128, nrb = (2 * a.I + 127) / 128;
    const float *bs[2 * PR]; // 16 rows lie in one block: I is a multiple of 16
#pragma unroll
    for (int r = 0; r < 2 * PR; ++r) {
        const int i = min(i0 + (p0 + r % PR) * 16, a.I - 16) + (r / PR) * a.I;
        bs[r]       = block ? a.s1 + (static_cast<int64_t>(e) * nrb + i / 128) * nkb : nullptr;
    }
    att_f4 acc[NC][2 * PR];
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
        for (int r = 0; r < 2 * PR; ++r)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[n][r][j] = 0.0f;
    MoeStage<F, 2 * PR, NC> ring[RING];
    auto fetch = [&](MoeStage<F, 2 * PR, NC> &g, int st) PTA_INLINE {
#pragma unroll
        for (int r = 0; r < 2 * PR; ++r) {
            g.w[r].load(row[r], st * F::STEP, qd, K);
            g.sc[r] = block ? bs[r][min(st, steps - 1)] : 1.0f;
        }
#pragma unroll
        for (int n = 0; n < NC; ++n) g.x[n].load(tok[n], st * F::STEP, qd, K);
    };
#pragma unroll
    for (int u = 0; u < RING; ++u) fetch(ring[u], wave + 4 * u);
    for (int st0 = wave; st0 < steps; st0 += 4 * RING) {
#pragma unroll
        for (int u = 0; u < RING; ++u) {
            // steps past the last, too, whose operands are all cut to zeros: with a
            // branch around them the loads in flight could not be counted, and every round
            // would wait for all of them
            const int st = st0 + 4 * u;
            if ((st + 1) * F::STEP > K) ring[u].cut(st * F::STEP, qd, K);
#pragma unroll
            for (int r = 0; r < 2 * PR; ++r) {
                att_f4 part[NC];
#pragma unroll
                for (int n = 0; n < NC; ++n)
#pragma unroll
                    for (int j = 0; j < 4; ++j) part[n][j] = 0.0f;
#pragma unroll
                for (int s = 0; s < F::NS; ++s) {
                    const uint4 wv = ring[u].w[r].get(s);
#pragma unroll
                    for (int n = 0; n < NC; ++n) part[n] = AttT<XT>::mfma16(wv, ring[u].x[n].v[s], part[n]);
                }
#pragma unroll
                for (int n = 0; n < NC; ++n)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[n][r][j] = fmaf(part[n][j], ring[u].sc[r], acc[n][r][j]);
            }
            fetch(ring[u], st + 4 * RING);
        }
    }
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
        for (int r = 0; r < 2 * PR; ++r) // [token][feature]: a lane's four features in a row
            *reinterpret_cast<float4 *>(&sh.red[(((wave * 4 + n) * 4) + (r / PR) * 2 + p0 + r % PR) * 256 + c * 16 + 4 * qd]) =
                make_float4(acc[n][r][0], acc[n][r][1], acc[n][r][2], acc[n][r][3]);
}

template <int XT, int KIND, bool MANY> __global__ __launch_bounds__(MOE_NT, 2) void moe_up_kernel(MoeArgs a) {
    __shared__ __align__(16) MoeUpShared sh;
    const int tid = threadIdx.x, lane = tid & 63, wave = moe_uniform(tid >> 6);
    const int slot = blockIdx.y, g = blockIdx.z, t0 = g * MOE_TG, tl = min(MOE_TG, a.T - t0);

    if (wave == 0) {
        int e = slot;
        if (a.by_entry) e = slot < tl * a.k ? moe_expert(a, static_cast<int64_t>(t0) * a.k + slot) : -1;
        float p    = 0.0f;
        int   mine = -1; // the token's first entry for this expert
        int   below = 0; // entries for experts before it
        if (lane < tl && e >= 0) {
            for (int j = a.k - 1; j >= 0; --j) {
                const int64_t at = static_cast<int64_t>(t0 + lane) * a.k + j;
                const int     ej = moe_expert(a, at);
                if (a.packed) below += __popcll(__ballot(static_cast<unsigned>(ej) < static_cast<unsigned>(e)));
                if (ej == e) {
                    mine = lane * a.k + j;
                    p += a.probs[at];
                }
            }
        }
        const uint64_t mask = __ballot(mine >= 0);
        // an expert that several entries name belongs to the first
        const int first = mask ? __shfl(mine, __ffsll(static_cast<unsigned long long>(mask)) - 1) : -1;
        if (mine >= 0) {
            const int at = __popcll(mask & ((1ull << lane) - 1));
            sh.prob[at]  = p;
            sh.tok[at]   = lane;
        }
        if (lane == 0) {
            sh.n      = __popcll(mask);
            sh.expert = mask && (!a.by_entry || first == slot) ? e : -1;
            sh.row0   = a.packed ? below : slot * a.TG;
        }
    }
    __syncthreads();
    const int e = moe_uniform(sh.expert), n_tok = moe_uniform(sh.n), i0 = blockIdx.x * 32;
    if (e < 0) return;
    if (!MANY || n_tok <= 16) {
        moe_up_pass<XT, KIND, 2, 1, 3>(a, sh, 0, i0, t0);
    } else if (n_tok <= 32) {
        moe_up_pass<XT, KIND, 2, 2, 2>(a, sh, 0, i0, t0);
    } else {
        // a pair of row tiles at a time: the tokens' operands fill the registers
        moe_up_pass<XT, KIND, 1, 4, 2>(a, sh, 0, i0, t0);
        moe_up_pass<XT, KIND, 1, 4, 2>(a, sh, 1, i0, t0);
    }
    __syncthreads();
    // 8 features of one token a thread
    for (int p = tid; p < n_tok * 4; p += MOE_NT) {
        const int tt = p >> 2, f = (p & 3) * 8, n = tt >> 4; // token, first feature
        const int i = i0 + f;
        if (i >= a.I) continue;
        const int at = (tt & 15) * 16 + (f & 15), u = f >> 4;
        float     v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float gate = 0.0f, up = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                gate += sh.red[((w * 4 + n) * 4 + u) * 256 + at + j];
                up += sh.red[((w * 4 + n) * 4 + 2 + u) * 256 + at + j];
            }
            if (a.scale == MOE_TENSOR) {
                gate *= a.s1[0];
                up *= a.s1[0];
            } else if (a.scale == MOE_ROW) {
                gate *= a.s1[static_cast<int64_t>(e) * 2 * a.I + i + j];
                up *= a.s1[static_cast<int64_t>(e) * 2 * a.I + a.I + i + j];
            }
            v[j] = gate / (1.0f + att_exp2(gate * -1.4426950408889634f)) * up * sh.prob[tt];
        }
        *reinterpret_cast<uint4 *>(a.act + (static_cast<int64_t>(g) * a.rows + sh.row0 + tt) * a.I + i) =
            make_uint4(AttT<XT>::pack(v[0], v[1]), AttT<XT>::pack(v[2], v[3]), AttT<XT>::pack(v[4], v[5]), AttT<XT>::pack(v[6], v[7]));
    }
}

// ---------------------------------------------------------------------------
// down product and the sum over experts: workgroup = (16 RT features, group of
// 64 tokens); the waves take every fourth step of the list of all reached
// experts' steps.  An expert with more tokens than the NC column tiles hold is
// listed again for the rest, its weights then come from the caches.  Each wave sums
// into an LDS table of its own, [token][feature], whenever it is done with an entry:
// the tokens of a column differ from expert to expert.
// ---------------------------------------------------------------------------
template <int XT, int KIND, bool ROW, int RT, int NC, int RING>
__global__ __launch_bounds__(MOE_NT, NC == 1 ? 2 : 1) void moe_down_kernel(MoeArgs a) {
    using F = MoeFrag<XT, KIND>;
    constexpr int                 NT = MOE_NT, NW = NT / 64, RS = RT * 16 + 4; // floats of a token's row
    constexpr int                 TOKS = NC == 1 ? 16 : MOE_TG, PART = NC * 16, LIST = MOE_MAX_E + MOE_TG * MOE_MAX_K / PART;
    __shared__ __align__(16) float ssum[NW][TOKS][RS];
    __shared__ unsigned long long smask[MOE_MAX_E];  // tokens of a slot
    __shared__ int                sfirst[LIST]; // by entry: an expert's slot; afterwards: list of reached slots
    __shared__ short              sexp[LIST], scnt[LIST], sfrom[LIST]; // of the list: expert, tokens, the first of them
    __shared__ int                srow[LIST];        // of the list: first row in act
    __shared__ int                sbefore[MOE_MAX_E]; // packed: an expert's entries, then those of the experts before it
    __shared__ int                stok[NW][PART]; // a wave's tokens of the expert it sums
    __shared__ int                scount;
    const int tid = threadIdx.x, lane = tid & 63, wave = moe_uniform(tid >> 6);
    const int g = blockIdx.y, t0 = g * MOE_TG, tl = min(MOE_TG, a.T - t0), n_ent = tl * a.k;
    const int64_t ent0 = static_cast<int64_t>(t0) * a.k;

    for (int i = tid; i < a.S; i += NT) smask[i] = 0;
    if (a.packed)
        for (int i = tid; i < a.E; i += NT) sbefore[i] = 0;
    for (int i = tid; i < NW * TOKS * RS; i += NT) (&ssum[0][0][0])[i] = 0.0f;
    if (a.by_entry) {
        for (int i = tid; i < a.E; i += NT) sfirst[i] = INT_MAX;
        __syncthreads();
        for (int i = tid; i < n_ent; i += NT) {
            const int e = moe_expert(a, ent0 + i);
            if (e >= 0) atomicMin(&sfirst[e], i);
        }
    }
    __syncthreads();
    for (int i = tid; i < n_ent; i += NT) {
        const int e = moe_expert(a, ent0 + i);
        if (e >= 0) atomicOr(&smask[a.by_entry ? sfirst[e] : e], 1ull << (i / a.k));
        if (e >= 0 && a.packed) atomicAdd(&sbefore[e], 1);
    }
    __syncthreads();
    if (wave == 0) {
        int n = 0;
        if (a.packed) {
            int before = 0;
            for (int e0 = 0; e0 < a.E; e0 += 64) {
                const int mine = e0 + lane < a.E ? sbefore[e0 + lane] : 0;
                int       sum  = mine;
#pragma unroll
                for (int d = 1; d < 64; d <<= 1) {
                    const int o = __shfl_up(sum, d);
                    if (lane >= d) sum += o;
                }
                if (e0 + lane < a.E) sbefore[e0 + lane] = before + sum - mine;
                before += __shfl(sum, 63);
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        }
        for (int s0 = 0; s0 < a.S; s0 += 64) {
            const int      s   = s0 + lane;
            const int      cnt = s < a.S ? __popcll(smask[s]) : 0;
            const uint64_t below = (1ull << lane) - 1;
            int            at = n, e = s, row0 = s * a.TG;
            if (cnt > 0) {
                if (a.by_entry) e = moe_expert(a, ent0 + s);
                if (a.packed) row0 = sbefore[e];
            }
#pragma unroll
            for (int q = 0; q < TOKS; q += PART) at += __popcll(__ballot(cnt > q) & below);
#pragma unroll
            for (int q = 0; q < TOKS; q += PART) {
                if (cnt > q) {
                    sexp[at]   = static_cast<short>(e);
                    srow[at]   = row0 + q;
                    sfirst[at] = s;
                    sfrom[at]  = static_cast<short>(q);
                    scnt[at]   = static_cast<short>(min(cnt - q, PART));
                    ++at;
                }
                n += __popcll(__ballot(cnt > q));
            }
        }
        if (lane == 0) scount = n;
    }
    __syncthreads();

    const int c = lane & 15, qd = lane >> 4, h0 = blockIdx.x * (RT * 16);
    const int K = a.I, steps = (K + F::STEP - 1) / F::STEP, items = moe_uniform(scount) * steps;
    const int nkb = (K + 127) / 128, nrb = (a.H + 127) / 128;
    const int64_t rowb = static_cast<int64_t>(K) * F::ES;
    const bool    block = a.scale == MOE_BLOCK;
    att_f4 acc[NC][RT];
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[n][r][j] = 0.0f;
    MoeStage<F, RT, NC> ring[RING];
    float4              rs[RING][RT]; // row scales
    int64_t             hoff[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) hoff[r] = min(h0 + r * 16 + c, a.H - 1) * rowb;
    const float one = a.scale == MOE_TENSOR ? a.s2[0] : 1.0f;
    auto fetch = [&](MoeStage<F, RT, NC> &q, float4(&qs)[RT], int it) PTA_INLINE {
        // past the last: the last expert's tables, and a step past K
        const int li = it < items ? it / steps : items / steps - 1, st = it < items ? it - li * steps : steps, k0 = st * F::STEP;
        const int e = moe_uniform(sexp[li]), n_tok = moe_uniform(scnt[li]);
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            q.w[r].load(a.w2 + static_cast<int64_t>(e) * a.H * rowb + hoff[r], k0, qd, K);
            q.sc[r] = block ? a.s2[(static_cast<int64_t>(e) * nrb + min(h0 + r * 16, a.H - 16) / 128) * nkb + min(st, steps - 1)] : 1.0f;
        }
        if constexpr (ROW) { // in every step: a load in a branch would drain the ring
#pragma unroll
            for (int r = 0; r < RT; ++r)
                qs[r] = *reinterpret_cast<const float4 *>(a.s2 + static_cast<int64_t>(e) * a.H + min(h0 + r * 16, a.H - 16) + 4 * qd);
        }
        const uint16_t *act = a.act + (static_cast<int64_t>(g) * a.rows + moe_uniform(srow[li])) * a.I;
#pragma unroll
        for (int n = 0; n < NC; ++n) q.x[n].load(act + static_cast<int64_t>(min(n * 16 + c, n_tok - 1)) * a.I, k0, qd, K);
    };
    if (wave < items) {
#pragma unroll
        for (int u = 0; u < RING; ++u) fetch(ring[u], rs[u], wave + NW * u);
    }
    for (int it0 = wave; it0 < items; it0 += NW * RING) {
#pragma unroll
        for (int u = 0; u < RING; ++u) {
            const int it = it0 + NW * u;
            const int li = it < items ? it / steps : items / steps - 1, st = it < items ? it - li * steps : steps, n_tok = moe_uniform(scnt[li]);
            if ((st + 1) * F::STEP > K) ring[u].cut(st * F::STEP, qd, K);
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                const float sc = ring[u].sc[r];
#pragma unroll
                for (int n = 0; n < NC; ++n) {
                    att_f4 part;
#pragma unroll
                    for (int j = 0; j < 4; ++j) part[j] = 0.0f;
#pragma unroll
                    for (int s = 0; s < F::NS; ++s) part = AttT<XT>::mfma16(ring[u].w[r].get(s), ring[u].x[n].v[s], part);
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[n][r][j] = fmaf(part[j], sc, acc[n][r][j]);
                }
            }
            float4 s4[RT];
#pragma unroll
            for (int r = 0; r < RT; ++r) s4[r] = ROW ? rs[u][r] : make_float4(one, one, one, one);
            fetch(ring[u], rs[u], it + NW * RING);
            if (st + NW >= steps) { // the wave's last step of this expert
                const uint64_t mask = smask[sfirst[li]];
                const int      nth  = __popcll(mask & ((1ull << lane) - 1)) - sfrom[li];
                if ((mask >> lane & 1) && nth >= 0 && nth < n_tok) stok[wave][nth] = lane;
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                __builtin_amdgcn_wave_barrier();
                __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
                for (int n = 0; n < NC; ++n) {
                    const bool in = n * 16 + c < n_tok;
                    const int  tt = in ? stok[wave][n * 16 + c] : 0;
#pragma unroll
                    for (int r = 0; r < RT; ++r) {
                        if (in) {
                            float4 *p = reinterpret_cast<float4 *>(&ssum[wave][tt][r * 16 + 4 * qd]);
                            float4  v = *p;
                            v.x = fmaf(acc[n][r][0], s4[r].x, v.x); v.y = fmaf(acc[n][r][1], s4[r].y, v.y);
                            v.z = fmaf(acc[n][r][2], s4[r].z, v.z); v.w = fmaf(acc[n][r][3], s4[r].w, v.w);
                            *p = v;
                        }
#pragma unroll
                        for (int j = 0; j < 4; ++j) acc[n][r][j] = 0.0f;
                    }
                }
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                __builtin_amdgcn_wave_barrier();
                __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            }
        }
    }
    __syncthreads();
    for (int p = tid; p < tl * RT * 2; p += NT) {
        const int tt = p / (RT * 2), f = (p % (RT * 2)) * 8;
        if (h0 + f >= a.H) continue;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[j] = ssum[0][tt][f + j];
#pragma unroll
            for (int w = 1; w < NW; ++w) v[j] += ssum[w][tt][f + j];
        }
        *reinterpret_cast<uint4 *>(a.y + static_cast<int64_t>(t0 + tt) * a.H + h0 + f) =
            make_uint4(AttT<XT>::pack(v[0], v[1]), AttT<XT>::pack(v[2], v[3]), AttT<XT>::pack(v[4], v[5]), AttT<XT>::pack(v[6], v[7]));
    }
}

} // namespace pta
