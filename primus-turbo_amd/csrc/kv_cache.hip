// Paged key / value cache: new tokens' keys and values written into their
// cache slots (quantized to fp8 with one scale for each token and head, or
// copied), and slots read back.
//
// Layout of one pool (keys or values): [num_pages, Hkv, page_size, D], fp8 or
// 16 bit, and for fp8 scale_inv [num_pages, Hkv, page_size] fp32.  The tokens
// of one page and head are contiguous, which is what the attention reads.  A
// slot is page * page_size + offset.
//
// A row is the D values of one token and head.  The quantization is the
// ROWWISE one (quant_misc.hip): scale = max / fmaxf(amax, 1e-12), q =
// fp8(clamp(x * scale)), scale_inv = 1 / scale; amax drops NaN.
//
// Both kernels are HBM-bound: a row is read once and written once by D / 8
// lanes (16 bytes of 16-bit data each), amax over the lanes by DPP; keys and
// values go in one launch (blockIdx.y).  8192 tokens of 8 heads of 128, bf16 to
// e4m3, are written in 11.5 us (4.4 TB/s), 131072 read back in 157 (5.2 TB/s; a
// large copy reaches 4.9); a few tokens take 3 us of launch.
#include <climits>

#include "common.h"

namespace pta {
namespace {

constexpr int KV_NT = 256;

// Rows of a thread in the read: with one, 131072 tokens of 8 heads of 128 took 217
// us, with eight 158 (their loads are in flight together, and a workgroup uses more
// of the scales' lines that it touches).  Eight once they give every CU four
// workgroups: below, 1021 tokens of 4 heads of 64 want the chip's width.
constexpr int KV_READ_ROWS = 8;

struct KVArgs {
    const void    *x[2];        // keys, values of the tokens (write) or null
    void          *y[2];        // outputs of the read
    int64_t        st[2], sh[2]; // element strides of x: token, head
    uint8_t       *cache[2];
    float         *scale[2];
    const void    *slots;
    int            slots_i64;
    uint32_t       tokens, heads, D, page;
    uint32_t       nslots; // num_pages * page_size
};

// max over groups of LPR lanes (8, 16 or 32)
template <int LPR> __device__ __forceinline__ float max_lpr(float v) {
    v = max8(v);
    if constexpr (LPR >= 16) v = fmaxf(v, dpp_f<PTA_DPP_ROW_MIRROR>(v));
    if constexpr (LPR >= 32) v = max_xor16(v);
    return v;
}

// Row of a pool for (slot, head), or -1 for a slot outside it.
__device__ __forceinline__ int64_t kv_row(const KVArgs &a, uint32_t t, uint32_t h) {
    const int64_t s = a.slots_i64 ? reinterpret_cast<const int64_t *>(a.slots)[t]
                                  : static_cast<int64_t>(reinterpret_cast<const int32_t *>(a.slots)[t]);
    if (s < 0 || s >= a.nslots) return -1;
    const uint32_t p = static_cast<uint32_t>(s) / a.page, o = static_cast<uint32_t>(s) - p * a.page;
    return (static_cast<int64_t>(p) * a.heads + h) * a.page + o;
}

__device__ __forceinline__ uint32_t pack_16(int dt, float a, float b) {
    return dt == PTA_BF16 ? f32_to_bf16_bits(a) | (static_cast<uint32_t>(f32_to_bf16_bits(b)) << 16)
                          : f32_to_f16_bits(a) | (static_cast<uint32_t>(f32_to_f16_bits(b)) << 16);
}

// VEC: pointers and strides of x allow 16-byte loads.
template <int IN_DT, int KIND, int LPR, bool VEC>
__global__ __launch_bounds__(KV_NT) void kv_write_kernel(KVArgs a) {
    const int      which = blockIdx.y;
    const uint32_t l     = threadIdx.x % LPR;
    const uint32_t row   = blockIdx.x * (KV_NT / LPR) + threadIdx.x / LPR;
    const uint32_t t     = row / a.heads, h = row - t * a.heads;
    const bool     in    = t < a.tokens && l * 8 < a.D;
    const int64_t  dst   = t < a.tokens ? kv_row(a, t, h) : -1;
    const int64_t  src   = t * a.st[which] + h * a.sh[which] + l * 8;
    if constexpr (KIND == PTA_CACHE_16BIT) {
        if (!in || dst < 0) return;
        uint4 w;
        if constexpr (VEC) {
            w = *reinterpret_cast<const uint4 *>(reinterpret_cast<const uint16_t *>(a.x[which]) + src);
        } else {
            const uint16_t *p    = reinterpret_cast<const uint16_t *>(a.x[which]) + src;
            uint32_t        e[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) e[i] = p[2 * i] | (static_cast<uint32_t>(p[2 * i + 1]) << 16);
            w = make_uint4(e[0], e[1], e[2], e[3]);
        }
        *reinterpret_cast<uint4 *>(a.cache[which] + (dst * a.D + l * 8) * 2) = w;
    } else {
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (in && dst >= 0) {
            if constexpr (VEC) {
                load8<IN_DT>(a.x[which], src, v);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = load_scalar<IN_DT>(a.x[which], src + i);
            }
        }
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(__builtin_canonicalizef(v[i])));
        m = max_lpr<LPR>(m);
        const float sc = scale_from_amax<KIND>(m, 1e-12f);
        if (!in || dst < 0) return;
        *reinterpret_cast<uint2 *>(a.cache[which] + dst * a.D + l * 8) =
            make_uint2(quant4<KIND>(&v[0], sc), quant4<KIND>(&v[4], sc));
        if (l == 0) a.scale[which][dst] = 1.0f / sc;
    }
}

// R rows of a thread, loaded together.
template <int KIND, int OUT_DT, int LPR, int R> __global__ __launch_bounds__(KV_NT) void kv_read_kernel(KVArgs a) {
    constexpr bool FP8   = KIND != PTA_CACHE_16BIT;
    constexpr int  ROWS  = KV_NT / LPR;
    const int      which = blockIdx.y;
    const uint32_t l = threadIdx.x % LPR, row0 = blockIdx.x * (ROWS * R) + threadIdx.x / LPR, rows = a.tokens * a.heads;
    if (l * 8 >= a.D) return;
    int64_t src[R];
    uint4   w[R];
    float   s[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const uint32_t row = min(row0 + r * ROWS, rows - 1), t = row / a.heads;
        src[r] = kv_row(a, t, row - t * a.heads);
    }
    if (a.nslots > 0) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t at = src[r] < 0 ? 0 : src[r];
            if constexpr (FP8) {
                const uint2 x = *reinterpret_cast<const uint2 *>(a.cache[which] + at * a.D + l * 8);
                w[r]          = make_uint4(x.x, x.y, 0, 0);
                s[r]          = a.scale[which][at];
            } else {
                w[r] = *reinterpret_cast<const uint4 *>(a.cache[which] + (at * a.D + l * 8) * 2);
            }
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const uint32_t row = row0 + r * ROWS;
        if (row >= rows) return;
        const int64_t dst = static_cast<int64_t>(row) * a.D + l * 8;
        if constexpr (!FP8) {
            if (src[r] < 0) w[r] = make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4 *>(reinterpret_cast<uint16_t *>(a.y[which]) + dst) = w[r];
        } else {
            float     v[8];
            const int ws[2] = {static_cast<int>(w[r].x), static_cast<int>(w[r].y)};
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                if constexpr (KIND == PTA_E4M3) {
                    v[4 * j] = __builtin_amdgcn_cvt_f32_fp8(ws[j], 0); v[4 * j + 1] = __builtin_amdgcn_cvt_f32_fp8(ws[j], 1);
                    v[4 * j + 2] = __builtin_amdgcn_cvt_f32_fp8(ws[j], 2); v[4 * j + 3] = __builtin_amdgcn_cvt_f32_fp8(ws[j], 3);
                } else {
                    v[4 * j] = __builtin_amdgcn_cvt_f32_bf8(ws[j], 0); v[4 * j + 1] = __builtin_amdgcn_cvt_f32_bf8(ws[j], 1);
                    v[4 * j + 2] = __builtin_amdgcn_cvt_f32_bf8(ws[j], 2); v[4 * j + 3] = __builtin_amdgcn_cvt_f32_bf8(ws[j], 3);
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = src[r] < 0 ? 0.0f : v[j] * s[r];
            if constexpr (OUT_DT == PTA_F32) {
                float4 *y = reinterpret_cast<float4 *>(reinterpret_cast<float *>(a.y[which]) + dst);
                y[0]      = make_float4(v[0], v[1], v[2], v[3]);
                y[1]      = make_float4(v[4], v[5], v[6], v[7]);
            } else {
                uint32_t o[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) o[j] = pack_16(OUT_DT, v[2 * j], v[2 * j + 1]);
                *reinterpret_cast<uint4 *>(reinterpret_cast<uint16_t *>(a.y[which]) + dst) = make_uint4(o[0], o[1], o[2], o[3]);
            }
        }
    }
}

int kv_lpr(int64_t D) { return D <= 64 ? 8 : D <= 128 ? 16 : 32; }

int kv_check(const void *k_cache, const void *v_cache, int kind, int64_t num_pages, int64_t page_size, int64_t Hkv,
             int64_t D, const void *k_scale, const void *v_scale, const void *slots, int64_t n) {
    PTA_CHECK_ARG(kind == PTA_E4M3 || kind == PTA_E5M2 || kind == PTA_CACHE_16BIT, "unknown cache kind %d", kind);
    PTA_CHECK_ARG(n >= 0 && num_pages >= 0 && page_size > 0 && Hkv > 0, "bad cache sizes");
    PTA_CHECK_ARG(D >= 16 && D <= 256 && D % 16 == 0, "head_dim must be a multiple of 16 in [16, 256] (got %lld)",
                  static_cast<long long>(D));
    PTA_CHECK_ARG(page_size <= INT_MAX && Hkv <= INT_MAX && num_pages <= INT_MAX / page_size &&
                      num_pages * page_size <= INT_MAX / Hkv,
                  "the cache has 2^31 rows (pages * page_size * heads) or more");
    PTA_CHECK_ARG(n <= INT_MAX / Hkv - KV_NT, "too many token rows for one call");
    if (n == 0) return PTA_OK;
    PTA_CHECK_ARG(slots != nullptr, "null slots");
    if (num_pages > 0) {
        PTA_CHECK_ARG(k_cache && v_cache, "null cache");
        PTA_CHECK_ARG(aligned16(k_cache) && aligned16(v_cache), "cache pools must be 16-byte aligned");
        PTA_CHECK_ARG(kind == PTA_CACHE_16BIT || (k_scale && v_scale), "an fp8 cache needs its scales");
    }
    return PTA_OK;
}

} // namespace
} // namespace pta

using namespace pta;

extern "C" int pta_kv_cache_write(const void *k, const void *v, int in_dtype, int64_t num_tokens, int64_t Hkv, int64_t D,
                                  int64_t k_stride_t, int64_t k_stride_h, int64_t v_stride_t, int64_t v_stride_h,
                                  const void *slots, int slots_i64, void *k_cache, void *v_cache, int cache_kind,
                                  int64_t num_pages, int64_t page_size, float *k_scale_inv, float *v_scale_inv,
                                  pta_stream_t stream) {
    clear_error();
    PTA_CHECK_ARG(in_dtype == PTA_F32 || in_dtype == PTA_F16 || in_dtype == PTA_BF16, "unknown input dtype %d", in_dtype);
    PTA_CHECK_ARG(cache_kind != PTA_CACHE_16BIT || in_dtype != PTA_F32, "a 16-bit cache takes 16-bit keys and values");
    if (int rc = kv_check(k_cache, v_cache, cache_kind, num_pages, page_size, Hkv, D, k_scale_inv, v_scale_inv, slots,
                          num_tokens))
        return rc;
    if (num_tokens == 0 || num_pages == 0) return PTA_OK;
    PTA_CHECK_ARG(k && v, "null keys or values");
    KVArgs a = {};
    a.x[0] = k; a.x[1] = v;
    a.st[0] = k_stride_t; a.st[1] = v_stride_t;
    a.sh[0] = k_stride_h; a.sh[1] = v_stride_h;
    a.cache[0] = static_cast<uint8_t *>(k_cache); a.cache[1] = static_cast<uint8_t *>(v_cache);
    a.scale[0] = k_scale_inv; a.scale[1] = v_scale_inv;
    a.slots = slots; a.slots_i64 = slots_i64;
    a.tokens = static_cast<uint32_t>(num_tokens); a.heads = static_cast<uint32_t>(Hkv);
    a.D = static_cast<uint32_t>(D); a.page = static_cast<uint32_t>(page_size);
    a.nslots = static_cast<uint32_t>(num_pages * page_size);
    const int64_t ev = in_dtype == PTA_F32 ? 4 : 8; // elements of 16 bytes
    const bool vec = aligned16(k) && aligned16(v) && k_stride_t % ev == 0 && k_stride_h % ev == 0 &&
                     v_stride_t % ev == 0 && v_stride_h % ev == 0;
    const int         lpr = kv_lpr(D);
    const dim3        grid(static_cast<unsigned>(cdiv(num_tokens * Hkv, KV_NT / lpr)), 2);
    const hipStream_t st = as_stream(stream);
#define PTA_KVW(DT, KIND, LPR)                                                                     \
    do {                                                                                           \
        if (vec) kv_write_kernel<DT, KIND, LPR, true><<<grid, KV_NT, 0, st>>>(a);                  \
        else kv_write_kernel<DT, KIND, LPR, false><<<grid, KV_NT, 0, st>>>(a);                     \
    } while (0)
#define PTA_KVW_L(DT, KIND)                                                                        \
    do {                                                                                           \
        if (lpr == 8) PTA_KVW(DT, KIND, 8);                                                        \
        else if (lpr == 16) PTA_KVW(DT, KIND, 16);                                                 \
        else PTA_KVW(DT, KIND, 32);                                                                \
    } while (0)
#define PTA_KVW_K(DT)                                                                              \
    do {                                                                                           \
        if (cache_kind == PTA_E4M3) PTA_KVW_L(DT, PTA_E4M3);                                       \
        else PTA_KVW_L(DT, PTA_E5M2);                                                              \
    } while (0)
    if (cache_kind == PTA_CACHE_16BIT) PTA_KVW_L(PTA_BF16, PTA_CACHE_16BIT); // moves bits: one type serves both
    else if (in_dtype == PTA_BF16) PTA_KVW_K(PTA_BF16);
    else if (in_dtype == PTA_F16) PTA_KVW_K(PTA_F16);
    else PTA_KVW_K(PTA_F32);
#undef PTA_KVW_K
#undef PTA_KVW_L
#undef PTA_KVW
    PTA_CHECK_LAUNCH();
    return PTA_OK;
}

extern "C" int pta_kv_cache_read(const void *k_cache, const void *v_cache, int cache_kind, int64_t num_pages,
                                 int64_t page_size, int64_t Hkv, int64_t D, const float *k_scale_inv,
                                 const float *v_scale_inv, const void *slots, int slots_i64, int64_t num_tokens,
                                 void *k_out, void *v_out, int out_dtype, pta_stream_t stream) {
    clear_error();
    PTA_CHECK_ARG(out_dtype == PTA_F32 || out_dtype == PTA_F16 || out_dtype == PTA_BF16, "unknown output dtype %d", out_dtype);
    PTA_CHECK_ARG(cache_kind != PTA_CACHE_16BIT || out_dtype != PTA_F32, "a 16-bit cache is read back as it is");
    if (int rc = kv_check(k_cache, v_cache, cache_kind, num_pages, page_size, Hkv, D, k_scale_inv, v_scale_inv, slots,
                          num_tokens))
        return rc;
    if (num_tokens == 0) return PTA_OK;
    PTA_CHECK_ARG(k_out && v_out, "null output");
    PTA_CHECK_ARG(aligned16(k_out) && aligned16(v_out), "outputs must be 16-byte aligned");
    KVArgs a = {};
    a.y[0] = k_out; a.y[1] = v_out;
    a.cache[0] = static_cast<uint8_t *>(const_cast<void *>(k_cache));
    a.cache[1] = static_cast<uint8_t *>(const_cast<void *>(v_cache));
    a.scale[0] = const_cast<float *>(k_scale_inv); a.scale[1] = const_cast<float *>(v_scale_inv);
    a.slots = slots; a.slots_i64 = slots_i64;
    a.tokens = static_cast<uint32_t>(num_tokens); a.heads = static_cast<uint32_t>(Hkv);
    a.D = static_cast<uint32_t>(D); a.page = static_cast<uint32_t>(page_size);
    a.nslots = static_cast<uint32_t>(num_pages * page_size);
    const int         lpr = kv_lpr(D);
    const int64_t     blocks = cdiv(num_tokens * Hkv, KV_NT / lpr); // of one row a thread
    const bool        many   = blocks * 2 >= KV_READ_ROWS * 4 * device_cu_count();
    const dim3        grid(static_cast<unsigned>(many ? cdiv(blocks, KV_READ_ROWS) : blocks), 2);
    const hipStream_t st = as_stream(stream);
#define PTA_KVR_R(KIND, DT, LPR)                                                                   \
    do {                                                                                           \
        if (many) kv_read_kernel<KIND, DT, LPR, KV_READ_ROWS><<<grid, KV_NT, 0, st>>>(a);          \
        else kv_read_kernel<KIND, DT, LPR, 1><<<grid, KV_NT, 0, st>>>(a);                          \
    } while (0)
#define PTA_KVR(KIND, DT)                                                                          \
    do {                                                                                           \
        if (lpr == 8) PTA_KVR_R(KIND, DT, 8);                                                      \
        else if (lpr == 16) PTA_KVR_R(KIND, DT, 16);                                               \
        else PTA_KVR_R(KIND, DT, 32);                                                              \
    } while (0)
#define PTA_KVR_O(KIND)                                                                            \
    do {                                                                                           \
        if (out_dtype == PTA_BF16) PTA_KVR(KIND, PTA_BF16);                                        \
        else if (out_dtype == PTA_F16) PTA_KVR(KIND, PTA_F16);                                     \
        else PTA_KVR(KIND, PTA_F32);                                                               \
    } while (0)
    if (cache_kind == PTA_CACHE_16BIT) PTA_KVR(PTA_CACHE_16BIT, PTA_BF16);
    else if (cache_kind == PTA_E4M3) PTA_KVR_O(PTA_E4M3);
    else PTA_KVR_O(PTA_E5M2);
#undef PTA_KVR_O
#undef PTA_KVR
#undef PTA_KVR_R
    PTA_CHECK_LAUNCH();
    return PTA_OK;
}
