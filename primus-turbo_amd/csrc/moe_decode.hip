// Experts of a decoding step: the C entry (moe_decode.h).
#include "moe_decode.h"

namespace pta {
namespace {

struct MoePlan {
    int64_t groups, TG, S;
    bool    by_entry, packed;
    int64_t rows, all; // of act: a group's, the call's
    size_t  bytes(int64_t I) const { return static_cast<size_t>(all * I * 2); }
};

MoePlan moe_plan(int64_t T, int64_t E, int64_t k) {
    MoePlan p;
    p.groups   = cdiv(T, MOE_TG);
    p.TG       = T < MOE_TG ? T : MOE_TG;
    p.by_entry = p.TG * k <= E;
    p.S        = p.by_entry ? p.TG * k : E;
    // Room for every token in every slot needs no counting, but grows with T E: calls of
    // several groups have a row for each entry (4096 tokens, top 8 of 256, I = 2048: 134 MB
    // for 4.29 GB)
    p.packed = p.groups > 1;
    p.rows   = p.packed ? p.TG * k : p.S * p.TG;
    p.all    = p.packed ? T * k : p.rows;
    return p;
}

template <int XT, int KIND, bool ROW> void moe_launch_down(const MoeArgs &a, unsigned groups, hipStream_t st) {
    if (a.TG <= 16) moe_down_kernel<XT, KIND, ROW, 1, 1, 4><<<dim3(static_cast<unsigned>(cdiv(a.H, 16)), groups), MOE_NT, 0, st>>>(a);
    else moe_down_kernel<XT, KIND, ROW, 2, 2, 4><<<dim3(static_cast<unsigned>(cdiv(a.H, 32)), groups), MOE_NT, 0, st>>>(a);
}

template <int XT, int KIND> void moe_launch_k(const MoeArgs &a, unsigned groups, hipStream_t st) {
    const dim3 up(static_cast<unsigned>(cdiv(a.I, 32)), static_cast<unsigned>(a.S), groups);
    if (a.TG <= 16) moe_up_kernel<XT, KIND, false><<<up, MOE_NT, 0, st>>>(a);
    else moe_up_kernel<XT, KIND, true><<<up, MOE_NT, 0, st>>>(a);
    if constexpr (KIND != PTA_CACHE_16BIT) {
        if (a.scale == MOE_ROW) return moe_launch_down<XT, KIND, true>(a, groups, st);
    }
    moe_launch_down<XT, KIND, false>(a, groups, st);
}

template <int XT> void moe_launch(const MoeArgs &a, int kind, unsigned groups, hipStream_t st) {
    if (kind == PTA_E4M3) moe_launch_k<XT, PTA_E4M3>(a, groups, st);
    else if (kind == PTA_E5M2) moe_launch_k<XT, PTA_E5M2>(a, groups, st);
    else moe_launch_k<XT, PTA_CACHE_16BIT>(a, groups, st);
}

} // namespace
} // namespace pta

using namespace pta;

extern "C" size_t pta_moe_decode_workspace_size(int64_t num_tokens, int64_t num_experts, int64_t topk, int64_t I) {
    if (num_tokens <= 0 || num_experts <= 0 || topk <= 0 || I <= 0) return 0;
    return moe_plan(num_tokens, num_experts, topk).bytes(I);
}

extern "C" int pta_moe_decode(const void *x, int x_dtype, int64_t num_tokens, int64_t H, int64_t x_stride,
                              const void *w_gate_up, const void *w_down, int weight_kind, const float *gate_up_scale_inv,
                              const float *down_scale_inv, int granularity, int64_t num_experts, int64_t I,
                              const void *topk_idx, int idx_i64, const float *topk_probs, int64_t topk, void *y,
                              void *workspace, size_t workspace_bytes, pta_stream_t stream) {
    clear_error();
    PTA_CHECK_ARG(x_dtype == PTA_BF16 || x_dtype == PTA_F16, "tokens must be bfloat16 or float16 (type %d)", x_dtype);
    PTA_CHECK_ARG(weight_kind == PTA_E4M3 || weight_kind == PTA_E5M2 || weight_kind == PTA_CACHE_16BIT,
                  "unknown weight kind %d", weight_kind);
    PTA_CHECK_ARG(weight_kind == PTA_CACHE_16BIT ? granularity == 0
                                                 : granularity == PTA_TENSORWISE || granularity == PTA_ROWWISE ||
                                                       granularity == PTA_BLOCKWISE,
                  "granularity %d does not fit the weights (fp8: TENSORWISE, ROWWISE or BLOCKWISE; 16 bit: 0)", granularity);
    PTA_CHECK_ARG(num_tokens >= 0 && num_tokens <= INT_MAX / 64, "bad token count");
    PTA_CHECK_ARG(num_experts > 0 && num_experts <= MOE_MAX_E, "num_experts must be in [1, %d] (got %lld)", MOE_MAX_E,
                  static_cast<long long>(num_experts));
    PTA_CHECK_ARG(topk > 0 && topk <= MOE_MAX_K, "topk must be in [1, %d] (got %lld)", MOE_MAX_K, static_cast<long long>(topk));
    PTA_CHECK_ARG(H > 0 && I > 0 && H % 16 == 0 && I % 16 == 0 && H <= INT_MAX / 4 && I <= INT_MAX / 4,
                  "hidden and intermediate sizes must be multiples of 16 (got %lld, %lld)", static_cast<long long>(H),
                  static_cast<long long>(I));
    if (num_tokens == 0) return PTA_OK;
    PTA_CHECK_ARG(x && w_gate_up && w_down && topk_idx && topk_probs && y, "null pointer");
    PTA_CHECK_ARG(weight_kind == PTA_CACHE_16BIT || (gate_up_scale_inv && down_scale_inv), "fp8 weights need their scales");
    PTA_CHECK_ARG(aligned16(x) && aligned16(y) && aligned16(w_gate_up) && aligned16(w_down) && x_stride % 8 == 0,
                  "tokens, weights and output must be 16-byte aligned, token rows a multiple of 8 elements apart");
    const MoePlan p = moe_plan(num_tokens, num_experts, topk);
    PTA_CHECK_ARG(p.groups <= 65535, "too many tokens for one call");
    PTA_CHECK_ARG(workspace && aligned16(workspace) && workspace_bytes >= p.bytes(I), "workspace too small: %zu bytes needed, %zu given",
                  p.bytes(I), workspace_bytes);
    MoeArgs a = {};
    a.x = static_cast<const uint16_t *>(x); a.x_st = x_stride;
    a.w1 = static_cast<const uint8_t *>(w_gate_up); a.w2 = static_cast<const uint8_t *>(w_down);
    a.s1 = gate_up_scale_inv; a.s2 = down_scale_inv;
    a.idx = topk_idx; a.idx_i64 = idx_i64; a.probs = topk_probs;
    a.act = static_cast<uint16_t *>(workspace); a.y = static_cast<uint16_t *>(y);
    a.T = static_cast<int>(num_tokens); a.E = static_cast<int>(num_experts); a.k = static_cast<int>(topk);
    a.I = static_cast<int>(I); a.H = static_cast<int>(H); a.S = static_cast<int>(p.S); a.TG = static_cast<int>(p.TG);
    a.by_entry = p.by_entry ? 1 : 0;
    a.rows = static_cast<int>(p.rows); a.packed = p.packed ? 1 : 0;
    a.scale    = granularity; // PTA_TENSORWISE / ROWWISE / BLOCKWISE are MoeScale's values
    const unsigned    groups = static_cast<unsigned>(p.groups);
    const hipStream_t st     = as_stream(stream);
    if (x_dtype == PTA_BF16) moe_launch<PTA_BF16>(a, weight_kind, groups, st);
    else moe_launch<PTA_F16>(a, weight_kind, groups, st);
    PTA_CHECK_LAUNCH();
    return PTA_OK;
}
