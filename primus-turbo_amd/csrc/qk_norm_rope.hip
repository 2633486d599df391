// Norms of queries and keys for each head and the rotation by their positions,
// in one pass; its backward pass; and the form that puts new tokens' keys and
// values into the paged cache at once.
//
// A row x is the D values of one token and head, w its head's weights, p the
// token's position:
//
//   r = (sum x^2 / D + eps)^(-1/2),   n = x r w       (without weights: n = x)
//   y_a = n_a cos - n_b sin,  y_b = n_a sin + n_b cos  for the pairs (a, b) of the
//         first R elements, cos and sin of row p of the tables; y = n beyond
//
// and with the gradient g of y, h = x r, g' = g turned by -angle:
//
//   dw = sum over rows g' h,   dx = r (g' w - h sum(g' w h) / D)
//
// A group of LPR lanes has a row; a lane has both elements of its pairs, so the
// rotation stays in the lane and the sums take log2(LPR) DPP steps.  Where the
// sizes allow, that is 8 elements of either half, 16 bytes each.
//
// All of it is fp32 between the loads and the one rounding of what is stored.
//
// Bound by memory: each row is read once and written once, the angles' tables come from the
// caches.  8192 tokens of 32 and 8 heads of 128, bf16, inputs and outputs not in the caches:
// forward 34 us (4.9 TB/s; a large copy 5.2), backward 52 (4.8) and 3 for the joined sums,
// cache write to e4m3 37 (5.1); fp32, over and over the same tensors, forward 62 (bf16 28) and
// backward 103 (45).  A row a group of lanes, no loop over rows in the forward
// pass: with two or four heads a lane, whose loads are in flight together, 36 and 37 us (the
// chip has enough rows in flight, and more small workgroups spread loads and stores better).
#include <algorithm>
#include <climits>

#include "common.h"

namespace pta {
namespace {

constexpr int QR_NT = 256;

struct QRArgs {
    const void    *x[3];         // queries, keys, values (cache write)
    int64_t        xt[3], xh[3]; // element strides: token, head
    const void    *g[2];         // gradients of the outputs
    int64_t        gt[2], gh[2];
    void          *y[2];         // outputs, or gradients of the inputs: [T, H, D]
    const void    *w[2];         // weights or null
    int            w_dt[2];
    float         *part[2];      // backward: [blocks, D] sums for the weights' gradients, or null
    int            H[2]; // heads
    const float   *cos, *sin;    // [positions, half]
    const void    *pos;
    int            pos_i64;
    int64_t        positions;
    uint32_t       T;
    int            D, half;
    float          eps, inv_d;
    uint32_t       blocks[2];    // backward: workgroups of the queries, of the keys
    uint8_t       *cache[2];
    float         *scale[2];
    const void    *slots;
    int            slots_i64;
    uint32_t       page, nslots;
};

// x[i] by comparisons: an index that the compiler does not know would put the arguments into memory
template <class T> __device__ __forceinline__ T qr_of(const T (&x)[2], int i) { return i ? x[1] : x[0]; }
template <class T> __device__ __forceinline__ T qr_of(const T (&x)[3], int i) { return i == 0 ? x[0] : i == 1 ? x[1] : x[2]; }

// ---- V elements of a type ----------------------------------------------------
template <int DT> constexpr int qr_bytes() { return InTraits<DT>::bytes; }

// As words: one 16-byte access, two (8 fp32), or a smaller one
template <int N> struct QRWords;
template <> struct QRWords<2> { typedef uint16_t type; };
template <> struct QRWords<4> { typedef uint32_t type; };
template <> struct QRWords<8> { typedef uint32_t type __attribute__((ext_vector_type(2))); };
template <> struct QRWords<16> { typedef uint32_t type __attribute__((ext_vector_type(4))); };
template <> struct QRWords<32> { typedef uint32_t type __attribute__((ext_vector_type(8), aligned(16))); };
template <int DT, int V> using QRRaw = typename QRWords<V * qr_bytes<DT>()>::type;

template <int DT, int V> __device__ __forceinline__ QRRaw<DT, V> qr_load(const void *base, int64_t i) {
    return *reinterpret_cast<const QRRaw<DT, V> *>(reinterpret_cast<const uint8_t *>(base) + i * qr_bytes<DT>());
}
template <int N, class W> __device__ __forceinline__ uint32_t qr_word(const W &w, int i) {
    if constexpr (N <= 4) return w;
    else return w[i];
}
template <int DT, int V> __device__ __forceinline__ void qr_values(const QRRaw<DT, V> &r, float (&v)[V]) {
    constexpr int N = V * qr_bytes<DT>();
#pragma unroll
    for (int i = 0; i < V; ++i) {
        if constexpr (DT == PTA_F32) {
            v[i] = __uint_as_float(qr_word<N>(r, i));
        } else {
            const uint32_t w = qr_word<N>(r, i / 2);
            if constexpr (DT == PTA_BF16) v[i] = __uint_as_float(i % 2 ? w & 0xffff0000u : w << 16);
            else v[i] = f16_bits_to_f32(i % 2 ? w >> 16 : w & 0xffffu);
        }
    }
}
// Two values of a 16-bit type, rounded
template <int DT> __device__ __forceinline__ uint32_t qr_pair(float a, float b) {
    if constexpr (DT == PTA_BF16) {
        typedef __bf16 pair __attribute__((ext_vector_type(2)));
        pair           r;
        r[0] = static_cast<__bf16>(a);
        r[1] = static_cast<__bf16>(b);
        return __builtin_bit_cast(uint32_t, r);
    } else {
        typedef _Float16 pair __attribute__((ext_vector_type(2)));
        pair             r;
        // opaque: a product fused with its rounding to fp16 differs from fp32, then fp16
        asm("" : "+v"(a), "+v"(b));
        r[0] = static_cast<_Float16>(a);
        r[1] = static_cast<_Float16>(b);
        return __builtin_bit_cast(uint32_t, r);
    }
}
template <int DT, int V> __device__ __forceinline__ QRRaw<DT, V> qr_round(const float (&v)[V]) {
    constexpr int N = V * qr_bytes<DT>();
    QRRaw<DT, V>  r;
    if constexpr (DT == PTA_F32) {
        if constexpr (V == 1) r = __float_as_uint(v[0]);
        else
#pragma unroll
            for (int i = 0; i < V; ++i) r[i] = __float_as_uint(v[i]);
    } else if constexpr (N <= 4) {
        r = static_cast<QRRaw<DT, V>>(qr_pair<DT>(v[0], v[V - 1]));
    } else {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) r[i] = qr_pair<DT>(v[2 * i], v[2 * i + 1]);
    }
    return r;
}
template <int DT, int V> __device__ __forceinline__ void qr_store(void *base, int64_t i, const float (&v)[V]) {
    *reinterpret_cast<QRRaw<DT, V> *>(reinterpret_cast<uint8_t *>(base) + i * qr_bytes<DT>()) = qr_round<DT, V>(v);
}

// sum and max over groups of LPR lanes (4, 8 or 16)
template <int LPR> __device__ __forceinline__ float qr_sum(float v) {
    v += dpp_f<PTA_DPP_QUAD_XOR1>(v);
    v += dpp_f<PTA_DPP_QUAD_XOR2>(v);
    if constexpr (LPR >= 8) v += dpp_f<PTA_DPP_ROW_HALF_MIRROR>(v);
    if constexpr (LPR >= 16) v += dpp_f<PTA_DPP_ROW_MIRROR>(v);
    return v;
}
template <int LPR> __device__ __forceinline__ float qr_max(float v) {
    v = fmaxf(v, dpp_f<PTA_DPP_QUAD_XOR1>(v));
    v = fmaxf(v, dpp_f<PTA_DPP_QUAD_XOR2>(v));
    if constexpr (LPR >= 8) v = fmaxf(v, dpp_f<PTA_DPP_ROW_HALF_MIRROR>(v));
    if constexpr (LPR >= 16) v = fmaxf(v, dpp_f<PTA_DPP_ROW_MIRROR>(v));
    return v;
}

// ---- a lane's part of a row ----------------------------------------------------
// P pieces of two runs of V elements at `at`: both halves' (pairs (i, i + half)), or
// two neighbouring runs (pairs (2 i, 2 i + 1)); beyond the rotated elements any two.
template <int V, int P> struct QRLane {
    int   at[P][2];
    bool  in[P], turned[P];
    float c[P][V], s[P][V]; // of pair j; (1, 0) where the token has no angles
};

template <int V, int LPR> constexpr int qr_pieces() { return V == 8 ? 1 : 128 / (V * LPR); }

template <bool NB, int V, int LPR>
__device__ __forceinline__ QRLane<V, qr_pieces<V, LPR>()> qr_lane(const QRArgs &a, int l) {
    constexpr int P = qr_pieces<V, LPR>();
    QRLane<V, P>  k;
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const int e = (p * LPR + l) * V; // number of its first pair
        k.in[p]     = 2 * e < a.D;
        k.turned[p] = e < a.half; // all of the piece's pairs or none
        if constexpr (NB) {
            k.at[p][0] = 2 * e;
            k.at[p][1] = 2 * e + V;
        } else {
            k.at[p][0] = e < a.half ? e : a.half + e;
            k.at[p][1] = e < a.half ? e + a.half : a.D / 2 + e;
        }
        // lanes beyond the row read its first elements; their sums are left out, nothing of theirs is stored
        if (!k.in[p]) k.at[p][0] = k.at[p][1] = 0;
    }
    return k;
}

// Angles of a token; false where its position has none.
template <int V, int LPR, int P> __device__ __forceinline__ bool qr_angles(const QRArgs &a, uint32_t t, int l, QRLane<V, P> &k) {
    const int64_t pos = a.pos_i64 ? reinterpret_cast<const int64_t *>(a.pos)[t]
                                  : static_cast<int64_t>(reinterpret_cast<const int32_t *>(a.pos)[t]);
    const bool    in  = pos >= 0 && pos < a.positions;
    const float  *c = a.cos + (in ? pos : 0) * a.half, *s = a.sin + (in ? pos : 0) * a.half;
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const int e = (p * LPR + l) * V;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            k.c[p][j] = 1.0f;
            k.s[p][j] = 0.0f;
        }
        if (!in) continue;
        if (e + V <= a.half) {
            typedef float vec __attribute__((ext_vector_type(4)));
            if constexpr (V % 4 == 0) {
                // V = 4, 8: half and the tables' alignment allow 16-byte loads
#pragma unroll
                for (int j = 0; j < V; j += 4) {
                    const vec x = *reinterpret_cast<const vec *>(c + e + j), y = *reinterpret_cast<const vec *>(s + e + j);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        k.c[p][j + i] = x[i];
                        k.s[p][j + i] = y[i];
                    }
                }
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    k.c[p][j] = c[e + j];
                    k.s[p][j] = s[e + j];
                }
            }
        }
    }
    return in;
}

// Turns the lane's pairs by the angles, BACK: by their negatives.  The products are fused
// here and not left to the compiler, so that every form of the kernels gives the same bits.
// Beyond the rotated elements two that are not a pair would meet here: they are left alone,
// since an angle of 0 would make a NaN of one beside an infinity.
template <bool NB, bool BACK, int V, int P> __device__ __forceinline__ void qr_turn(const QRLane<V, P> &k, float (&v)[P][2][V]) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
        if (!k.turned[p]) continue;
        if constexpr (V > 1 && NB) {
            // the 2 V elements are V pairs of neighbours
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int j = 0; j < V; j += 2) {
                    const float c = k.c[p][r * (V / 2) + j / 2], s = BACK ? -k.s[p][r * (V / 2) + j / 2] : k.s[p][r * (V / 2) + j / 2];
                    const float x = v[p][r][j], y = v[p][r][j + 1];
                    v[p][r][j]     = fmaf(x, c, -(y * s));
                    v[p][r][j + 1] = fmaf(x, s, y * c);
                }
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float c = k.c[p][j], s = BACK ? -k.s[p][j] : k.s[p][j];
                const float x = v[p][0][j], y = v[p][1][j];
                v[p][0][j] = fmaf(x, c, -(y * s));
                v[p][1][j] = fmaf(x, s, y * c);
            }
        }
    }
}

template <int DT, int V, int P> __device__ __forceinline__ void qr_weights_of(const void *b, const QRLane<V, P> &k, float (&w)[P][2][V]) {
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
        for (int r = 0; r < 2; ++r)
            qr_values<DT, V>(qr_load<DT, V>(b, k.at[p][r]), w[p][r]);
}
template <int V, int P> __device__ __forceinline__ void qr_weights(const QRArgs &a, int which, const QRLane<V, P> &k, float (&w)[P][2][V]) {
    const void *b = qr_of(a.w, which);
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int j = 0; j < V; ++j) w[p][r][j] = 0.0f;
    if (b == nullptr) return;
    if (qr_of(a.w_dt, which) == PTA_BF16) qr_weights_of<PTA_BF16, V, P>(b, k, w);
    else if (qr_of(a.w_dt, which) == PTA_F16) qr_weights_of<PTA_F16, V, P>(b, k, w);
    else qr_weights_of<PTA_F32, V, P>(b, k, w);
}

template <int DT, int V, int P>
__device__ __forceinline__ void qr_load_row(const void *x, int64_t at, const QRLane<V, P> &k, QRRaw<DT, V> (&raw)[P][2]) {
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
        for (int r = 0; r < 2; ++r)
            raw[p][r] = qr_load<DT, V>(x, at + k.at[p][r]);
}
template <int DT, int V, int P> __device__ __forceinline__ void qr_row(const QRRaw<DT, V> (&raw)[P][2], float (&v)[P][2][V]) {
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
        for (int r = 0; r < 2; ++r) qr_values<DT, V>(raw[p][r], v[p][r]);
}

// 1 / rms of a row
template <int LPR, int V, int P> __device__ __forceinline__ float qr_rsqrt(const QRArgs &a, const QRLane<V, P> &k, const float (&v)[P][2][V]) {
    float ss = 0.0f;
#pragma unroll
    for (int p = 0; p < P; ++p) {
        float x = 0.0f;
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int j = 0; j < V; ++j) x = fmaf(v[p][r][j], v[p][r][j], x);
        ss += k.in[p] ? x : 0.0f;
    }
    return rsqrtf(fmaf(qr_sum<LPR>(ss), a.inv_d, a.eps));
}

// ---- forward, and cache write ------------------------------------------------
// NB: pairs of neighbours.  KIND: -1 queries and keys to y; a cache kind: queries to y, keys and values to their slots
template <int KIND, int DT, int V, int P, int LPR>
__device__ __forceinline__ void qr_put(const QRArgs &a, int which, int64_t row, int l, const QRLane<V, P> &k, const float (&v)[P][2][V]) {
    if constexpr (KIND == PTA_CACHE_16BIT) {
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
            for (int r = 0; r < 2; ++r)
                if (k.in[p] && row >= 0) qr_store<DT, V>(qr_of(a.cache, which), row * a.D + k.at[p][r], v[p][r]);
    } else {
        // ROWWISE quantization of the fp32 values, as kv_cache_write's of the rounded ones
        float m = 0.0f;
#pragma unroll
        for (int p = 0; p < P; ++p) {
            float x = 0.0f;
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int j = 0; j < V; ++j) x = fmaxf(x, fabsf(__builtin_canonicalizef(v[p][r][j])));
            m = fmaxf(m, k.in[p] ? x : 0.0f);
        }
        const float sc = scale_from_amax<KIND>(qr_max<LPR>(m), 1e-12f);
        if (row < 0) return;
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                if (!k.in[p]) continue;
                uint8_t *y = qr_of(a.cache, which) + row * a.D + k.at[p][r];
                if constexpr (V % 4 == 0) {
#pragma unroll
                    for (int j = 0; j < V; j += 8) {
                        if constexpr (V == 8) *reinterpret_cast<uint2 *>(y) = make_uint2(quant4<KIND>(&v[p][r][0], sc), quant4<KIND>(&v[p][r][4], sc));
                        else *reinterpret_cast<uint32_t *>(y) = quant4<KIND>(&v[p][r][0], sc);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < V; ++j) y[j] = cvt1_fp8<KIND>(qclamp<KIND>(v[p][r][j], sc));
                }
            }
        if (l == 0) qr_of(a.scale, which)[row] = 1.0f / sc;
    }
}

template <int KIND, int DT, bool NB, int V, int LPR> __global__ __launch_bounds__(QR_NT) void qr_forward_kernel(QRArgs a) {
    constexpr int  P   = qr_pieces<V, LPR>();
    const int      l   = threadIdx.x % LPR;
    const uint32_t row = blockIdx.x * (QR_NT / LPR) + threadIdx.x / LPR;
    const uint32_t per = a.H[0] + a.H[1] + (KIND >= 0 ? a.H[1] : 0);
    const uint32_t t   = row / per;
    if (t >= a.T) return;
    int which = 0, h = static_cast<int>(row - t * per);
    if (h >= a.H[0]) {
        h -= a.H[0];
        which = 1;
        if (KIND >= 0 && h >= a.H[1]) {
            h -= a.H[1];
            which = 2;
        }
    }
    QRLane<V, P> k = qr_lane<NB, V, LPR>(a, l);
    QRRaw<DT, V> raw[P][2];
    qr_load_row<DT, V, P>(qr_of(a.x, which), static_cast<int64_t>(t) * qr_of(a.xt, which) + h * qr_of(a.xh, which), k, raw);
    int64_t slot_row = 0;
    if (KIND >= 0 && which > 0) {
        const int64_t s = a.slots_i64 ? reinterpret_cast<const int64_t *>(a.slots)[t]
                                      : static_cast<int64_t>(reinterpret_cast<const int32_t *>(a.slots)[t]);
        if (s < 0 || s >= a.nslots) return; // all lanes of the group
        const uint32_t pg = static_cast<uint32_t>(s) / a.page;
        slot_row = (static_cast<int64_t>(pg) * a.H[1] + h) * a.page + (static_cast<uint32_t>(s) - pg * a.page);
    }
    float v[P][2][V];
    if (KIND >= 0 && which == 2) {
        qr_row<DT, V, P>(raw, v);
        qr_put<KIND, DT, V, P, LPR>(a, 1, slot_row, l, k, v);
        return;
    }
    float      w[P][2][V];
    const bool in = qr_angles<V, LPR, P>(a, t, l, k);
    qr_weights<V, P>(a, which, k, w);
    if (!in) {
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
            for (int i = 0; i < 2; ++i) raw[p][i] = {};
    }
    qr_row<DT, V, P>(raw, v);
    if (qr_of(a.w, which) != nullptr && in) { // zeros stay zeros, whatever eps and the weights are
        const float r = qr_rsqrt<LPR, V, P>(a, k, v);
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < V; ++j) v[p][i][j] = v[p][i][j] * r * w[p][i][j];
    }
    qr_turn<NB, false, V, P>(k, v);
    if (KIND >= 0 && which == 1) {
        qr_put<KIND < 0 ? 0 : KIND, DT, V, P, LPR>(a, 0, slot_row, l, k, v);
        return;
    }
    const int64_t at = (static_cast<int64_t>(t) * qr_of(a.H, which) + h) * a.D;
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (k.in[p]) qr_store<DT, V>(qr_of(a.y, which), at + k.at[p][i], v[p][i]);
}

// ---- backward ------------------------------------------------------------------
// The first blocks[0] workgroups take the queries, the others the keys, each every
// blocks[]-th run of items, so that the weights' gradients are sums in registers,
// then in LDS, then one row of `part` a workgroup: no atomics, the same bits every time.
template <int DT, bool NB, int V, int LPR> __global__ __launch_bounds__(QR_NT) void qr_backward_kernel(QRArgs a) {
    constexpr int  P = qr_pieces<V, LPR>(), GROUPS = QR_NT / LPR, DMAX = 2 * V * P * LPR;
    __shared__ float sums[GROUPS * DMAX];
    const int      which = blockIdx.x >= a.blocks[0], grp = threadIdx.x / LPR, l = threadIdx.x % LPR;
    const uint32_t block = which ? blockIdx.x - a.blocks[0] : blockIdx.x;
    const int      H = qr_of(a.H, which);
    const uint32_t rows = a.T * H, step = qr_of(a.blocks, which) * GROUPS;
    const bool     norm = qr_of(a.w, which) != nullptr;
    QRLane<V, P>   k = qr_lane<NB, V, LPR>(a, l);
    float          w[P][2][V], dw[P][2][V];
    qr_weights<V, P>(a, which, k, w);
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) dw[p][i][j] = 0.0f;
    for (uint32_t row = block * GROUPS + grp; row < rows; row += step) {
        const uint32_t t = row / H, h = row - t * H;
        QRRaw<DT, V>   rx[P][2], rg[P][2];
        qr_load_row<DT, V, P>(qr_of(a.g, which), static_cast<int64_t>(t) * qr_of(a.gt, which) + h * qr_of(a.gh, which), k, rg);
        if (norm) qr_load_row<DT, V, P>(qr_of(a.x, which), static_cast<int64_t>(t) * qr_of(a.xt, which) + h * qr_of(a.xh, which), k, rx);
        const bool in = qr_angles<V, LPR, P>(a, t, l, k);
        if (!in) { // zeros give zeros, and nothing to the weights
#pragma unroll
            for (int p = 0; p < P; ++p)
#pragma unroll
                for (int i = 0; i < 2; ++i) rg[p][i] = {};
        }
        float g[P][2][V];
        qr_row<DT, V, P>(rg, g);
        qr_turn<NB, true, V, P>(k, g);
        if (norm && in) {
            float v[P][2][V], dot = 0.0f;
            qr_row<DT, V, P>(rx, v);
            const float r = qr_rsqrt<LPR, V, P>(a, k, v);
#pragma unroll
            for (int p = 0; p < P; ++p) {
                float x = 0.0f;
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        v[p][i][j] *= r;
                        dw[p][i][j] = fmaf(g[p][i][j], v[p][i][j], dw[p][i][j]);
                        g[p][i][j] *= w[p][i][j];
                        x = fmaf(g[p][i][j], v[p][i][j], x);
                    }
                dot += k.in[p] ? x : 0.0f;
            }
            dot = qr_sum<LPR>(dot) * a.inv_d;
#pragma unroll
            for (int p = 0; p < P; ++p)
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < V; ++j) g[p][i][j] = r * (g[p][i][j] - v[p][i][j] * dot);
        }
        const int64_t at = static_cast<int64_t>(row) * a.D;
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (k.in[p]) qr_store<DT, V>(qr_of(a.y, which), at + k.at[p][i], g[p][i]);
    }
    if (qr_of(a.part, which) == nullptr) return;
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (k.in[p])
#pragma unroll
                for (int j = 0; j < V; ++j) sums[grp * DMAX + k.at[p][i] + j] = dw[p][i][j];
    __syncthreads();
    for (int d = threadIdx.x; d < a.D; d += QR_NT) {
        float s = 0.0f;
#pragma unroll 8
        for (int i = 0; i < GROUPS; ++i) s += sums[i * DMAX + d];
        qr_of(a.part, which)[static_cast<int64_t>(block) * a.D + d] = s;
    }
}

// Sums the workgroups' rows: 8 columns by 128 runs of rows a workgroup.
struct QRSums {
    const float *part[2];
    void        *dw[2];
    int          dt[2];
    int          rows[2], D;
};
__global__ __launch_bounds__(1024) void qr_sums_kernel(QRSums a) {
    __shared__ float s[128][9];
    const int which = blockIdx.y, c = threadIdx.x % 8, run = threadIdx.x / 8, d = blockIdx.x * 8 + c;
    if (qr_of(a.dw, which) == nullptr) return;
    float acc = 0.0f;
    if (d < a.D) {
#pragma unroll 8
        for (int i = run; i < qr_of(a.rows, which); i += 128) acc += qr_of(a.part, which)[static_cast<int64_t>(i) * a.D + d];
    }
    s[run][c] = acc;
    __syncthreads();
    if (run >= 8) return; // one wave: 16 rows each, then the 8 sums of a column, which lie 8 lanes apart
#pragma unroll
    for (int i = 1; i < 16; ++i) acc += s[run + 8 * i][c];
#pragma unroll
    for (int o = 8; o < 64; o <<= 1) acc += __shfl_xor(acc, o);
    if (run != 0 || d >= a.D) return;
    if (qr_of(a.dt, which) == PTA_F32) reinterpret_cast<float *>(qr_of(a.dw, which))[d] = acc;
    else reinterpret_cast<uint16_t *>(qr_of(a.dw, which))[d] = qr_of(a.dt, which) == PTA_BF16 ? f32_to_bf16_bits(acc) : f32_to_f16_bits(acc);
}

// ---- host ----------------------------------------------------------------------
struct QRShape {
    int V, lpr; // run of elements, lanes of a row
};

bool qr_fits(const void *p, int64_t st, int64_t sh, int V, int bytes) {
    return reinterpret_cast<uintptr_t>(p) % std::min(V * bytes, 16) == 0 && st * bytes % std::min(V * bytes, 16) == 0 &&
           sh * bytes % std::min(V * bytes, 16) == 0;
}

int qr_check(int dtype, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t rot, int64_t positions, float eps) {
    PTA_CHECK_ARG(dtype == PTA_F32 || dtype == PTA_F16 || dtype == PTA_BF16, "unknown type %d", dtype);
    PTA_CHECK_ARG(T >= 0 && Hq >= 0 && Hkv >= 0 && positions >= 0, "bad sizes");
    PTA_CHECK_ARG(D >= 2 && D <= 256 && D % 2 == 0, "head_dim must be even and at most 256 (got %lld)", static_cast<long long>(D));
    PTA_CHECK_ARG(rot >= 2 && rot <= D && rot % 2 == 0, "rotated elements must be even and at most head_dim (got %lld)",
                  static_cast<long long>(rot));
    PTA_CHECK_ARG(Hq <= INT_MAX / 4 && Hkv <= INT_MAX / 4 && T <= (INT_MAX - 1024) / std::max<int64_t>(1, Hq + 2 * Hkv),
                  "too many rows for one call");
    PTA_CHECK_ARG(eps >= 0.0f && eps - eps == 0.0f, "eps must be finite and not negative");
    return PTA_OK;
}

// Longest run that the sizes and every tensor's alignment allow
template <class Ok> QRShape qr_shape(const QRArgs &a, Ok ok) {
    for (int V : {8, 4, 2}) {
        if (a.D % (2 * V) || a.half % V || !ok(V)) continue;
        if (V >= 4 && (a.half % 4 || !aligned16(a.cos) || !aligned16(a.sin))) continue;
        if (!qr_fits(a.w[0], 0, 0, V, a.w_dt[0] == PTA_F32 ? 4 : 2) || !qr_fits(a.w[1], 0, 0, V, a.w_dt[1] == PTA_F32 ? 4 : 2)) continue;
        return {V, V < 8 ? 16 : a.D <= 64 ? 4 : a.D <= 128 ? 8 : 16};
    }
    return {1, 16};
}

void qr_fill(QRArgs &a, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, const float *cos, const float *sin, int64_t positions,
             int64_t rot, const void *pos, int pos_i64, const void *wq, int wq_dt, const void *wk, int wk_dt, float eps) {
    a.T = static_cast<uint32_t>(T);
    a.H[0] = static_cast<int>(Hq); a.H[1] = static_cast<int>(Hkv);
    a.D = static_cast<int>(D); a.half = static_cast<int>(rot / 2);
    a.cos = cos; a.sin = sin; a.positions = positions; a.pos = pos; a.pos_i64 = pos_i64;
    a.w[0] = wq; a.w[1] = wk; a.w_dt[0] = wq_dt; a.w_dt[1] = wk_dt;
    a.eps = eps; a.inv_d = 1.0f / static_cast<float>(D);
}

bool qr_weight_type(const void *w, int dt) { return w == nullptr || dt == PTA_F32 || dt == PTA_F16 || dt == PTA_BF16; }

#define PTA_QR_SHAPE(S, F)                                                                         \
    do {                                                                                           \
        if (S.V == 8 && S.lpr == 4) F(8, 4);                                                       \
        else if (S.V == 8 && S.lpr == 8) F(8, 8);                                                  \
        else if (S.V == 8) F(8, 16);                                                               \
        else if (S.V == 4) F(4, 16);                                                               \
        else if (S.V == 2) F(2, 16);                                                               \
        else F(1, 16);                                                                             \
    } while (0)

template <int KIND, int DT, bool NB> void qr_forward(QRArgs &a, QRShape s, hipStream_t st) {
    const int64_t  rows = static_cast<int64_t>(a.T) * (a.H[0] + a.H[1] + (KIND >= 0 ? a.H[1] : 0));
    const unsigned grid = static_cast<unsigned>(cdiv(rows, QR_NT / s.lpr));
    if (grid == 0) return;
#define PTA_QRF(V, LPR) qr_forward_kernel<KIND, DT, NB, V, LPR><<<grid, QR_NT, 0, st>>>(a)
    PTA_QR_SHAPE(s, PTA_QRF);
#undef PTA_QRF
}

// Workgroups of the backward pass for the queries and the keys, each with the same
// number of runs of rows: at most QR_BACK a CU of both (8192 tokens of 32 and 8 heads of 128
// with the sums: 54.7 us with three or four, 58 with two or eight, 63 with 16).
constexpr int QR_BACK = 4;
void qr_back_blocks(int64_t T, int64_t Hq, int64_t Hkv, int64_t (&blocks)[2]) {
    const int64_t H[2] = {Hq, Hkv}, most = QR_BACK * device_cu_count();
    for (int i = 0; i < 2; ++i) {
        // runs of the fewest rows: how many a workgroup takes goes by alignment, which the size query does not know
        const int64_t runs = cdiv(T * H[i], QR_NT / 16), share = std::max<int64_t>(1, most * H[i] / std::max<int64_t>(1, Hq + Hkv));
        blocks[i]          = runs == 0 ? 0 : cdiv(runs, cdiv(runs, share));
    }
}

template <int DT, bool NB> void qr_backward(QRArgs &a, QRShape s, hipStream_t st) {
    const unsigned grid = a.blocks[0] + a.blocks[1];
    if (grid == 0) return;
#define PTA_QRB(V, LPR) qr_backward_kernel<DT, NB, V, LPR><<<grid, QR_NT, 0, st>>>(a)
    PTA_QR_SHAPE(s, PTA_QRB);
#undef PTA_QRB
}

template <int KIND, int DT> void qr_forward(QRArgs &a, QRShape s, int interleaved, hipStream_t st) {
    if (interleaved) qr_forward<KIND, DT, true>(a, s, st);
    else qr_forward<KIND, DT, false>(a, s, st);
}
template <int DT> void qr_backward(QRArgs &a, QRShape s, int interleaved, hipStream_t st) {
    if (interleaved) qr_backward<DT, true>(a, s, st);
    else qr_backward<DT, false>(a, s, st);
}

} // namespace
} // namespace pta

using namespace pta;

extern "C" int pta_qk_norm_rope(const void *q, const void *k, int dtype, int64_t num_tokens, int64_t Hq, int64_t Hkv, int64_t D,
                                int64_t q_stride_t, int64_t q_stride_h, int64_t k_stride_t, int64_t k_stride_h, const float *cos,
                                const float *sin, int64_t num_positions, int64_t rot_dim, const void *positions, int positions_i64,
                                const void *q_weight, int q_weight_dtype, const void *k_weight, int k_weight_dtype, float eps,
                                int interleaved, void *q_out, void *k_out, pta_stream_t stream) {
    clear_error();
    if (int rc = qr_check(dtype, num_tokens, Hq, Hkv, D, rot_dim, num_positions, eps)) return rc;
    PTA_CHECK_ARG(qr_weight_type(q_weight, q_weight_dtype) && qr_weight_type(k_weight, k_weight_dtype), "unknown weight type");
    if (num_tokens == 0 || Hq + Hkv == 0) return PTA_OK;
    PTA_CHECK_ARG((Hq == 0 || (q && q_out)) && (Hkv == 0 || (k && k_out)) && positions && (num_positions == 0 || (cos && sin)), "null pointer");
    PTA_CHECK_ARG(aligned16(q_out) && aligned16(k_out), "outputs must be 16-byte aligned");
    QRArgs a = {};
    qr_fill(a, num_tokens, Hq, Hkv, D, cos, sin, num_positions, rot_dim, positions, positions_i64, q_weight, q_weight_dtype, k_weight,
            k_weight_dtype, eps);
    a.x[0] = q; a.x[1] = k;
    a.xt[0] = q_stride_t; a.xt[1] = k_stride_t;
    a.xh[0] = q_stride_h; a.xh[1] = k_stride_h;
    a.y[0] = q_out; a.y[1] = k_out;
    const int     b = dtype == PTA_F32 ? 4 : 2;
    const QRShape s = qr_shape(a, [&](int V) {
        return qr_fits(q, q_stride_t, q_stride_h, V, b) && qr_fits(k, k_stride_t, k_stride_h, V, b);
    });
    const hipStream_t st = as_stream(stream);
    if (dtype == PTA_BF16) qr_forward<-1, PTA_BF16>(a, s, interleaved, st);
    else if (dtype == PTA_F16) qr_forward<-1, PTA_F16>(a, s, interleaved, st);
    else qr_forward<-1, PTA_F32>(a, s, interleaved, st);
    PTA_CHECK_LAUNCH();
    return PTA_OK;
}

extern "C" size_t pta_qk_norm_rope_backward_workspace_size(int64_t num_tokens, int64_t Hq, int64_t Hkv, int64_t D) {
    if (num_tokens <= 0 || Hq < 0 || Hkv < 0 || D <= 0) return 0;
    int64_t blocks[2];
    qr_back_blocks(num_tokens, Hq, Hkv, blocks);
    return static_cast<size_t>((blocks[0] + blocks[1]) * D * 4);
}

extern "C" int pta_qk_norm_rope_backward(const void *q_grad_out, const void *k_grad_out, int64_t gq_stride_t, int64_t gq_stride_h,
                                         int64_t gk_stride_t, int64_t gk_stride_h, const void *q, const void *k, int dtype,
                                         int64_t num_tokens, int64_t Hq, int64_t Hkv, int64_t D, int64_t q_stride_t, int64_t q_stride_h,
                                         int64_t k_stride_t, int64_t k_stride_h, const float *cos, const float *sin,
                                         int64_t num_positions, int64_t rot_dim, const void *positions, int positions_i64,
                                         const void *q_weight, int q_weight_dtype, const void *k_weight, int k_weight_dtype, float eps,
                                         int interleaved, void *q_grad, void *k_grad, void *q_weight_grad, void *k_weight_grad,
                                         void *workspace, size_t workspace_bytes, pta_stream_t stream) {
    clear_error();
    if (int rc = qr_check(dtype, num_tokens, Hq, Hkv, D, rot_dim, num_positions, eps)) return rc;
    PTA_CHECK_ARG(qr_weight_type(q_weight, q_weight_dtype) && qr_weight_type(k_weight, k_weight_dtype), "unknown weight type");
    PTA_CHECK_ARG((q_weight || !q_weight_grad) && (k_weight || !k_weight_grad), "a weight's gradient without the weight");
    const bool rows = num_tokens > 0 && Hq + Hkv > 0;
    PTA_CHECK_ARG(!rows || ((Hq == 0 || (q_grad_out && q_grad && (q || !q_weight))) &&
                            (Hkv == 0 || (k_grad_out && k_grad && (k || !k_weight))) && positions && (num_positions == 0 || (cos && sin))),
                  "null pointer");
    PTA_CHECK_ARG(aligned16(q_grad) && aligned16(k_grad), "outputs must be 16-byte aligned");
    QRArgs a = {};
    qr_fill(a, num_tokens, Hq, Hkv, D, cos, sin, num_positions, rot_dim, positions, positions_i64, q_weight, q_weight_dtype, k_weight,
            k_weight_dtype, eps);
    a.x[0] = q; a.x[1] = k;
    a.xt[0] = q_stride_t; a.xt[1] = k_stride_t;
    a.xh[0] = q_stride_h; a.xh[1] = k_stride_h;
    a.g[0] = q_grad_out; a.g[1] = k_grad_out;
    a.gt[0] = gq_stride_t; a.gt[1] = gk_stride_t;
    a.gh[0] = gq_stride_h; a.gh[1] = gk_stride_h;
    a.y[0] = q_grad; a.y[1] = k_grad;
    int64_t blocks[2] = {0, 0};
    if (rows) qr_back_blocks(num_tokens, Hq, Hkv, blocks);
    a.blocks[0] = static_cast<uint32_t>(blocks[0]); a.blocks[1] = static_cast<uint32_t>(blocks[1]);
    const size_t need = static_cast<size_t>((blocks[0] + blocks[1]) * D * 4);
    const bool   sums = q_weight_grad || k_weight_grad;
    PTA_CHECK_ARG(!sums || need == 0 || (workspace && aligned16(workspace) && workspace_bytes >= need),
                  "workspace too small: %zu bytes needed, %zu given", need, workspace_bytes);
    float *part = static_cast<float *>(workspace);
    if (q_weight_grad) a.part[0] = part;
    if (k_weight_grad) a.part[1] = part + blocks[0] * D;
    const int     b = dtype == PTA_F32 ? 4 : 2;
    const QRShape s = qr_shape(a, [&](int V) {
        return (q_weight == nullptr || qr_fits(q, q_stride_t, q_stride_h, V, b)) && (k_weight == nullptr || qr_fits(k, k_stride_t, k_stride_h, V, b)) &&
               qr_fits(q_grad_out, gq_stride_t, gq_stride_h, V, b) && qr_fits(k_grad_out, gk_stride_t, gk_stride_h, V, b);
    });
    const hipStream_t st = as_stream(stream);
    if (dtype == PTA_BF16) qr_backward<PTA_BF16>(a, s, interleaved, st);
    else if (dtype == PTA_F16) qr_backward<PTA_F16>(a, s, interleaved, st);
    else qr_backward<PTA_F32>(a, s, interleaved, st);
    PTA_CHECK_LAUNCH();
    if (sums) {
        QRSums r = {};
        r.part[0] = a.part[0]; r.part[1] = a.part[1];
        r.dw[0] = q_weight_grad; r.dw[1] = k_weight_grad;
        r.dt[0] = q_weight_dtype; r.dt[1] = k_weight_dtype;
        r.rows[0] = static_cast<int>(blocks[0]); r.rows[1] = static_cast<int>(blocks[1]);
        r.D = static_cast<int>(D);
        qr_sums_kernel<<<dim3(static_cast<unsigned>(cdiv(D, 8)), 2), 1024, 0, st>>>(r);
        PTA_CHECK_LAUNCH();
    }
    return PTA_OK;
}

extern "C" int pta_qk_norm_rope_cache_write(const void *q, const void *k, const void *v, int dtype, int64_t num_tokens, int64_t Hq,
                                            int64_t Hkv, int64_t D, int64_t q_stride_t, int64_t q_stride_h, int64_t k_stride_t,
                                            int64_t k_stride_h, int64_t v_stride_t, int64_t v_stride_h, const float *cos, const float *sin,
                                            int64_t num_positions, int64_t rot_dim, const void *positions, int positions_i64,
                                            const void *q_weight, int q_weight_dtype, const void *k_weight, int k_weight_dtype, float eps,
                                            int interleaved, const void *slots, int slots_i64, void *k_cache, void *v_cache, int cache_kind,
                                            int64_t num_pages, int64_t page_size, float *k_scale_inv, float *v_scale_inv, void *q_out,
                                            pta_stream_t stream) {
    clear_error();
    PTA_CHECK_ARG(dtype == PTA_F16 || dtype == PTA_BF16, "queries, keys and values must be bfloat16 or float16 (type %d)", dtype);
    if (int rc = qr_check(dtype, num_tokens, Hq, Hkv, D, rot_dim, num_positions, eps)) return rc;
    PTA_CHECK_ARG(qr_weight_type(q_weight, q_weight_dtype) && qr_weight_type(k_weight, k_weight_dtype), "unknown weight type");
    PTA_CHECK_ARG(cache_kind == PTA_E4M3 || cache_kind == PTA_E5M2 || cache_kind == PTA_CACHE_16BIT, "unknown cache kind %d", cache_kind);
    PTA_CHECK_ARG(D % 16 == 0, "a cache's head_dim must be a multiple of 16 (got %lld)", static_cast<long long>(D));
    PTA_CHECK_ARG(num_pages >= 0 && page_size > 0 && Hkv > 0 && page_size <= INT_MAX && num_pages <= INT_MAX / page_size &&
                      num_pages * page_size <= INT_MAX / Hkv,
                  "the cache has 2^31 rows (pages * page_size * heads) or more");
    if (num_tokens == 0) return PTA_OK;
    PTA_CHECK_ARG((Hq == 0 || (q && q_out)) && k && v && slots && positions && (num_positions == 0 || (cos && sin)), "null pointer");
    PTA_CHECK_ARG(aligned16(q_out), "the output must be 16-byte aligned");
    if (num_pages > 0) {
        PTA_CHECK_ARG(k_cache && v_cache, "null cache");
        PTA_CHECK_ARG(aligned16(k_cache) && aligned16(v_cache), "cache pools must be 16-byte aligned");
        PTA_CHECK_ARG(cache_kind == PTA_CACHE_16BIT || (k_scale_inv && v_scale_inv), "an fp8 cache needs its scales");
    }
    QRArgs a = {};
    qr_fill(a, num_tokens, Hq, Hkv, D, cos, sin, num_positions, rot_dim, positions, positions_i64, q_weight, q_weight_dtype, k_weight,
            k_weight_dtype, eps);
    a.x[0] = q; a.x[1] = k; a.x[2] = v;
    a.xt[0] = q_stride_t; a.xt[1] = k_stride_t; a.xt[2] = v_stride_t;
    a.xh[0] = q_stride_h; a.xh[1] = k_stride_h; a.xh[2] = v_stride_h;
    a.y[0] = q_out;
    a.cache[0] = static_cast<uint8_t *>(k_cache); a.cache[1] = static_cast<uint8_t *>(v_cache);
    a.scale[0] = k_scale_inv; a.scale[1] = v_scale_inv;
    a.slots = slots; a.slots_i64 = slots_i64;
    a.page = static_cast<uint32_t>(page_size); a.nslots = static_cast<uint32_t>(num_pages * page_size);
    const QRShape s = qr_shape(a, [&](int V) {
        return qr_fits(q, q_stride_t, q_stride_h, V, 2) && qr_fits(k, k_stride_t, k_stride_h, V, 2) && qr_fits(v, v_stride_t, v_stride_h, V, 2);
    });
    const hipStream_t st = as_stream(stream);
#define PTA_QRW(KIND)                                                                              \
    do {                                                                                           \
        if (dtype == PTA_BF16) qr_forward<KIND, PTA_BF16>(a, s, interleaved, st);                               \
        else qr_forward<KIND, PTA_F16>(a, s, interleaved, st);                                                  \
    } while (0)
    if (cache_kind == PTA_E4M3) PTA_QRW(PTA_E4M3);
    else if (cache_kind == PTA_E5M2) PTA_QRW(PTA_E5M2);
    else PTA_QRW(PTA_CACHE_16BIT);
#undef PTA_QRW
    PTA_CHECK_LAUNCH();
    return PTA_OK;
}
