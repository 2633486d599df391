// Attention of new tokens over a paged cache: the C entry, the choice between
// the kernels and how far row tiles are split (paged_attention.h).
#include <algorithm>

#include "page_select.h"
#include "paged_attention.h"

namespace pta {
namespace {

// One kernel's share of a call
struct AttnPart {
    int     rows; // of a row tile; 0: not launched
    int     rows_min, rows_max;
    int64_t slots, goal;  // wide
    int64_t split, part_step; // narrow
    bool    part_seq;
    size_t  desc_bytes, ml_bytes, o_bytes;
    size_t  bytes() const { return desc_bytes + ml_bytes + o_bytes; }
};

struct AttnPlan {
    AttnPart part[2]; // narrow, wide
    size_t   bytes() const { return part[0].bytes() + part[1].bytes(); }
};

size_t round256(int64_t n) { return static_cast<size_t>(cdiv(n, 256) * 256); }

// Rows of a sequence up to which the narrow kernel takes it where both run (4 chunks
// of up to 256 tokens under a window of 1024, 32 / 8 heads of 128: 42 us with 16 and 32,
// 47 with 64; 16 of up to 512, 16 heads of 64: 81 to 82 with each; a few tokens of each
// of many long sequences were not among them: 64 of 1 to 3 tokens over 8192, 64 / 8
// heads, where 24 rows go to the wide kernel, take 194), and up
// to which it takes a call's only rows (8 tokens of 32 / 8 heads of 128 over 8192, 32
// rows: 28.7 us, wide 27.3; over 1000: 15.6 and 16.5; 16 tokens, 64 rows: 51.8 and 32.7).
constexpr int ATT_NARROW_MOST = 16, ATT_NARROW_ALONE = 32;
static_assert(ATT_NARROW_MOST <= ATT_NARROW_ROWS, "parts by sequence hold one row tile");

// Workgroups at most that fill the tokens of no sequence.  Where there are none they
// cost nothing that shows: 1 token over 1000 16.0 us without and 15.9 with, 64 tokens
// over 16384 260.6 and 260.7, 16 chunks of up to 512 81.7 and 81.5.
constexpr int ATT_PADS = 64;

// Every sequence gets the same number of chunks: two workgroups a CU from all of
// them, four chunks where sequences may differ in length (64 of up to 16384 tokens:
// 260 us, 281 with one or two), no more than key tiles.
// `even`: all are about as long.
AttnPart attn_narrow_part(int64_t Tq, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t keys, bool mix, bool even) {
    AttnPart      p    = {};
    const int64_t fill = cdiv(2 * device_cu_count(), B * Hkv);
    p.rows     = ATT_NARROW_ROWS;
    p.rows_max = mix ? ATT_NARROW_MOST : INT_MAX;
    p.split    = std::max<int64_t>(1, std::min(std::max<int64_t>(fill, B > 1 && !even ? 4 : 1), cdiv(keys, ATT_NARROW_KEYS)));
    if (p.split > 1) {
        // a mixed call's tokens are mostly the wide form's: parts for the rows that a
        // sequence can have here, unless the tokens are fewer
        p.part_seq  = mix && B * Hkv * ATT_NARROW_ROWS < Tq * Hq;
        p.part_step = p.part_seq ? B * Hkv * ATT_NARROW_ROWS : Tq * Hq;
        p.ml_bytes  = round256(p.split * p.part_step * 8);
        p.o_bytes   = round256(p.split * p.part_step * D * 4);
    }
    return p;
}

// Row tiles are found on the device (their number goes by the lengths); they are
// split where they do not give every CU two (16 chunks of up to 512 tokens over 4096,
// 16 heads of 64: 93 us split for one a CU, 82 for two, 81 for three; 4 of 256 over a
// window of 1024, 32 / 8 heads of 128: 42, 42 and 51, more parts to join).
AttnPart attn_wide_part(int64_t Tq, int64_t B, int64_t Hkv, int64_t G, int64_t D, int64_t keys, bool mix) {
    AttnPart p = {};
    p.rows     = ATT_WIDE_ROWS;
    p.rows_min = mix ? ATT_NARROW_MOST : 0;
    p.rows_max = INT_MAX;
    // row tiles of a head, sum of ceil(n G / rows), over the sequences that come here
    const int64_t full = Tq * G / ATT_WIDE_ROWS, most = full + std::min(B, Tq * G / (p.rows_min + 1));
    const int64_t goal = cdiv(2 * device_cu_count(), Hkv);
    // row tiles alone fill the chip, or no tile has keys for two chunks
    p.goal  = full >= goal || keys <= ATT_WIDE_KEYS ? 0 : goal;
    p.slots = most + p.goal;
    if (p.goal > 0) {
        const int64_t parts = std::min(p.slots, 2 * p.goal); // chunks of split row tiles
        p.desc_bytes = round256(p.slots * 16);
        p.ml_bytes   = round256(parts * Hkv * ATT_WIDE_ROWS * 8);
        p.o_bytes    = round256(parts * Hkv * ATT_WIDE_ROWS * D * 4);
    }
    return p;
}

// All of it goes by sizes that the host has: tokens, sequences, heads and the
// page table's extent.  Lengths stay on the device, so where sequences of few and
// of many rows may be together both forms run, each on its own, in one launch
// (chunks of up to 512 tokens over 4096, 16 heads of 64: 82 us, 103 as two launches;
// of 256 over a window of 1024, 32 / 8 heads of 128: 42 and 46).  The wide form alone
// would make single tokens beside one chunk three times as slow (64 sequences of
// 16384 tokens: 743 us, narrow 261).
AttnPlan attn_plan(int64_t Tq, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_pages, int64_t page, bool even = false) {
    AttnPlan      p = {};
    const int64_t G = Hq / Hkv, keys = max_pages * page;
    // single tokens, or a few rows; no more tokens than sequences may also be one chunk
    // beside empty ones, which is right here, row tile by row tile, but slow
    const bool    few = Tq <= B || Tq * G <= ATT_NARROW_ALONE;
    const bool    mix = !few && B > 1 && G <= ATT_NARROW_MOST; // more rows to a token: none is the narrow form's
    if (few || mix) p.part[0] = attn_narrow_part(Tq, B, Hq, Hkv, D, keys, mix, even);
    if (!few) p.part[1] = attn_wide_part(Tq, B, Hkv, G, D, keys, mix);
    return p;
}

} // namespace
} // namespace pta

using namespace pta;

extern "C" size_t pta_paged_attention_workspace_size(int64_t num_tokens, int64_t num_seqs, int64_t Hq, int64_t Hkv,
                                                     int64_t D, int64_t max_pages, int64_t page_size) {
    if (num_tokens <= 0 || num_seqs <= 0 || Hq <= 0 || Hkv <= 0 || D <= 0 || max_pages < 0 || page_size <= 0) return 0;
    return attn_plan(num_tokens, num_seqs, Hq, Hkv, D, max_pages, page_size).bytes();
}

// Checks the arguments that every form takes, and fills the kernels'.
// table_stride_h: of a page table with a row for each cache head, whose sequences are single
// tokens (so that the narrow form alone runs) of about the same length; 0: one row for all
static int attn_arguments(AttnArgs &a, const void *q, int q_dtype, int64_t num_tokens, int64_t Hq, int64_t D, int64_t q_stride_t, int64_t q_stride_h,
                          const void *k_cache, const void *v_cache, int cache_kind, int64_t num_pages, int64_t page_size, int64_t Hkv,
                          const float *k_scale_inv, const float *v_scale_inv, const int32_t *page_table, int64_t table_stride,
                          int64_t table_stride_h, int64_t max_pages, const int32_t *cu_seqlens_q, const int32_t *seq_lens, int64_t num_seqs,
                          float softmax_scale, int64_t window_size, int64_t num_sinks, void *out, float *lse) {
    PTA_CHECK_ARG(q_dtype == PTA_BF16 || q_dtype == PTA_F16, "queries must be bfloat16 or float16 (type %d)", q_dtype);
    PTA_CHECK_ARG(cache_kind == PTA_E4M3 || cache_kind == PTA_E5M2 || cache_kind == PTA_CACHE_16BIT,
                  "unknown cache kind %d", cache_kind);
    PTA_CHECK_ARG(num_tokens >= 0 && num_seqs >= 0 && num_pages >= 0 && page_size > 0 && max_pages >= 0, "bad sizes");
    PTA_CHECK_ARG(Hkv > 0 && Hq > 0 && Hq % Hkv == 0, "query heads (%lld) must be a multiple of cache heads (%lld)",
                  static_cast<long long>(Hq), static_cast<long long>(Hkv));
    PTA_CHECK_ARG(D >= 16 && D <= 256 && D % 16 == 0, "head_dim must be a multiple of 16 in [16, 256] (got %lld)",
                  static_cast<long long>(D));
    PTA_CHECK_ARG(page_size <= INT_MAX && num_pages <= INT_MAX / page_size && num_pages * page_size <= INT_MAX / Hkv,
                  "the cache has 2^31 rows (pages * page_size * heads) or more");
    PTA_CHECK_ARG(max_pages <= (INT_MAX - 1024) / page_size, "page_table spans 2^31 tokens or more");
    PTA_CHECK_ARG(num_tokens <= (INT_MAX - 1024) / Hq && num_seqs < (1 << 24), "too many tokens or sequences");
    PTA_CHECK_ARG(window_size >= 0 && num_sinks >= 0 && window_size <= INT_MAX / 2 && num_sinks <= INT_MAX / 2,
                  "window_size and num_sinks must not be negative");
    PTA_CHECK_ARG(softmax_scale == softmax_scale && softmax_scale - softmax_scale == 0.0f, "softmax_scale must be finite");
    if (num_tokens == 0) return PTA_OK;
    PTA_CHECK_ARG(num_seqs > 0, "tokens without a sequence");
    PTA_CHECK_ARG(q && out && cu_seqlens_q && seq_lens, "null pointer");
    PTA_CHECK_ARG(max_pages == 0 || page_table, "null page_table");
    PTA_CHECK_ARG(aligned16(q) && aligned16(out) && q_stride_t % 8 == 0 && q_stride_h % 8 == 0,
                  "queries and output must be 16-byte aligned, with strides of multiples of 8 elements");
    if (num_pages > 0) {
        PTA_CHECK_ARG(k_cache && v_cache, "null cache");
        PTA_CHECK_ARG(aligned16(k_cache) && aligned16(v_cache), "cache pools must be 16-byte aligned");
        PTA_CHECK_ARG(cache_kind == PTA_CACHE_16BIT || (k_scale_inv && v_scale_inv), "an fp8 cache needs its scales");
    }
    a = {};
    a.q = static_cast<const uint16_t *>(q);
    a.q_st = q_stride_t; a.q_sh = q_stride_h;
    a.kc = static_cast<const uint8_t *>(k_cache); a.vc = static_cast<const uint8_t *>(v_cache);
    a.ks = k_scale_inv; a.vs = v_scale_inv;
    a.table = page_table; a.table_st = table_stride; a.table_sh = table_stride_h;
    a.cu = cu_seqlens_q; a.lens = seq_lens;
    a.out = static_cast<uint16_t *>(out); a.lse = lse;
    a.B = static_cast<int>(num_seqs); a.Tq = static_cast<int>(num_tokens);
    a.Hq = static_cast<int>(Hq); a.Hkv = static_cast<int>(Hkv); a.G = static_cast<int>(Hq / Hkv); a.D = static_cast<int>(D);
    a.num_pages = static_cast<int>(num_pages); a.page = static_cast<int>(page_size); a.max_pages = static_cast<int>(max_pages);
    // j / page for 0 <= j < 2^31: ceil(2^(32 + s) / page) with s = floor(log2(page)), exact there
    while (page_size >> (a.page_shift + 1)) ++a.page_shift;
    if (page_size & (page_size - 1)) a.page_mul = static_cast<uint32_t>(((1ull << (32 + a.page_shift)) + page_size - 1) / page_size);
    a.window = static_cast<int>(window_size); a.sinks = static_cast<int>(num_sinks);
    a.scale_log2 = softmax_scale * 1.4426950408889634f;
    if (num_pages == 0) { // keys without a row read row 0 of something and drop it
        a.kc = a.vc = static_cast<const uint8_t *>(q);
        a.ks = a.vs = static_cast<const float *>(q);
    }
    return PTA_OK;
}

static int attn_call(const void *q, int q_dtype, int64_t num_tokens, int64_t Hq, int64_t D, int64_t q_stride_t, int64_t q_stride_h,
                     const void *k_cache, const void *v_cache, int cache_kind, int64_t num_pages, int64_t page_size, int64_t Hkv,
                     const float *k_scale_inv, const float *v_scale_inv, const int32_t *page_table, int64_t table_stride,
                     int64_t table_stride_h, int64_t max_pages, const int32_t *cu_seqlens_q, const int32_t *seq_lens, int64_t num_seqs,
                     float softmax_scale, int64_t window_size, int64_t num_sinks, void *out, float *lse, void *workspace,
                     size_t workspace_bytes, pta_stream_t stream) {
    AttnArgs a;
    if (int rc = attn_arguments(a, q, q_dtype, num_tokens, Hq, D, q_stride_t, q_stride_h, k_cache, v_cache, cache_kind, num_pages, page_size,
                                Hkv, k_scale_inv, v_scale_inv, page_table, table_stride, table_stride_h, max_pages, cu_seqlens_q, seq_lens,
                                num_seqs, softmax_scale, window_size, num_sinks, out, lse))
        return rc;
    if (num_tokens == 0) return PTA_OK;
    const AttnPlan p = attn_plan(num_tokens, num_seqs, Hq, Hkv, D, max_pages, page_size, table_stride_h != 0);
    PTA_CHECK_ARG(p.bytes() == 0 || (workspace && aligned16(workspace) && workspace_bytes >= p.bytes()),
                  "workspace too small: %zu bytes needed, %zu given", p.bytes(), workspace_bytes);
    PTA_CHECK_ARG((std::max<int64_t>(p.part[0].split, ATT_JOIN_PARTS) * num_seqs + ATT_JOIN_PARTS * p.part[1].slots) * Hkv <= INT_MAX / 4, "too many row tiles for one call");
    AttnCall c = {};
    c.has_narrow = p.part[0].rows > 0;
    c.has_wide   = p.part[1].rows > 0;
    // 64 elements of 4 values a workgroup, at the sequences' mean of rows
    c.narrow_join_parts = static_cast<int>(std::min<int64_t>(ATT_JOIN_PARTS, cdiv(num_tokens * (Hq / Hkv) * (D / 4), 64 * num_seqs)));
    // the host does not know how many tokens no sequence owns: 8 pieces of a thread if all
    // of them, behind the workgroups that have work
    c.pads = static_cast<int>(std::min<int64_t>(ATT_PADS, cdiv(num_tokens * Hq * (D / 8), 8 * 256)));
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    for (int i = 0; i < 2; ++i) {
        const AttnPart &part = p.part[i];
        AttnArgs       &x    = i == 0 ? c.narrow : c.wide;
        x            = a;
        x.slots      = static_cast<int>(part.slots);
        x.split_goal = static_cast<int>(part.goal);
        x.split      = static_cast<int>(part.split);
        x.part_seq   = part.part_seq;
        x.part_step  = static_cast<int>(part.part_step);
        x.rows_min   = part.rows_min;
        x.rows_max   = part.rows_max;
        if (part.bytes() == 0) continue;
        x.desc    = reinterpret_cast<int4 *>(ws);
        x.part_ml = reinterpret_cast<float2 *>(ws + part.desc_bytes);
        x.part_o  = reinterpret_cast<float *>(ws + part.desc_bytes + part.ml_bytes);
        ws += part.bytes();
    }
    const hipStream_t st = as_stream(stream);
    if (q_dtype == PTA_BF16) attn_launch<PTA_BF16>(c, cache_kind, st);
    else attn_launch<PTA_F16>(c, cache_kind, st);
    PTA_CHECK_LAUNCH();
    return PTA_OK;
}

extern "C" int pta_paged_attention(const void *q, int q_dtype, int64_t num_tokens, int64_t Hq, int64_t D,
                                   int64_t q_stride_t, int64_t q_stride_h, const void *k_cache, const void *v_cache,
                                   int cache_kind, int64_t num_pages, int64_t page_size, int64_t Hkv,
                                   const float *k_scale_inv, const float *v_scale_inv, const int32_t *page_table,
                                   int64_t table_stride, int64_t max_pages, const int32_t *cu_seqlens_q,
                                   const int32_t *seq_lens, int64_t num_seqs, float softmax_scale, int64_t window_size,
                                   int64_t num_sinks, void *out, float *lse, void *workspace, size_t workspace_bytes,
                                   pta_stream_t stream) {
    clear_error();
    return attn_call(q, q_dtype, num_tokens, Hq, D, q_stride_t, q_stride_h, k_cache, v_cache, cache_kind, num_pages, page_size, Hkv,
                     k_scale_inv, v_scale_inv, page_table, table_stride, 0, max_pages, cu_seqlens_q, seq_lens, num_seqs, softmax_scale,
                     window_size, num_sinks, out, lse, workspace, workspace_bytes, stream);
}

// The workspace of attention through selected pages: what was chosen (pages for each token,
// or lists for tiles of tokens), how many keys of its pages each token sees, 0, 1, 2, ... for
// its tokens as sequences, then what the choice and, over the same bytes (it begins when the
// choice has ended), the attention need.
//
// Tokens go by tiles of 16 rows where a sequence has two or more of them on average: their
// pages overlap, and a tile's page is read and converted once for all its rows (1024 tokens
// over 16384, 32 / 8 heads of 128, 16 of 256 pages, of which four tokens take 37: attention
// 128 us, token by token 320; 64 of 2048 pages, with the ranges 680 us, token by token 1217).
// Tables of more than PS_TILE_PAGES pages go token by token: the choice that makes lists has a
// token's scores in one wave's registers, and the one of several waves a token makes none.
namespace {
struct SparsePlan {
    int64_t  K, tile, tiles, cap; // tile: tokens of a tile, 0: none
    size_t   sel, masks, counts, pos, lens, cu, rest;
    AttnPart part; // of tiles
    size_t   bytes() const { return sel + masks + counts + pos + lens + cu + rest; }
};
SparsePlan sparse_plan(int64_t T, int64_t num_seqs, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_pages, int64_t page, int64_t take) {
    SparsePlan p = {};
    p.K    = std::min(take, max_pages);
    p.lens = round256(T * 4);
    p.cu   = round256((T + 1) * 4);
    const int64_t G = Hq / Hkv;
    if (G <= ATT_NARROW_ROWS / 2 && T >= 2 * num_seqs && max_pages > 0 && max_pages <= pta::PS_TILE_PAGES &&
        ATT_NARROW_ROWS * p.K <= (INT_MAX - 1024) / page) { // a list's keys are counted in 32 bits
        p.tile   = ATT_NARROW_ROWS / G;
        p.tiles  = cdiv(T, p.tile);
        // a tile's sequences are at most one run of its tokens each, and a run has a page of its row once
        p.cap    = std::min(p.tile * p.K, std::min(p.tile, num_seqs) * max_pages);
        p.sel    = round256(p.tiles * Hkv * p.cap * 8);
        p.masks  = round256(p.tiles * Hkv * p.cap * 2);
        p.counts = round256(p.tiles * Hkv * 4);
        p.pos    = round256(T * 4);
        p.part   = attn_narrow_part(T, p.tiles, Hq, Hkv, D, p.K * page, false, true);
        p.rest   = std::max(pta::ps_workspace(T, Hkv, max_pages, p.tile), p.part.bytes());
    } else {
        p.sel  = round256(T * Hkv * p.K * 4);
        p.rest = std::max(pta::ps_workspace(T, Hkv, max_pages, 1), attn_plan(T, T, Hq, Hkv, D, p.K, page, true).bytes());
    }
    return p;
}
} // namespace

extern "C" size_t pta_sparse_paged_attention_workspace_size(int64_t num_tokens, int64_t num_seqs, int64_t Hq, int64_t Hkv, int64_t D,
                                                            int64_t max_pages, int64_t page_size, int64_t num_selected) {
    if (num_tokens <= 0 || num_seqs <= 0 || Hkv <= 0 || Hq < Hkv || D <= 0 || max_pages < 0 || page_size <= 0 || num_selected <= 0) return 0;
    return sparse_plan(num_tokens, num_seqs, Hq, Hkv, D, max_pages, page_size, num_selected).bytes();
}

extern "C" int pta_sparse_paged_attention(const void *q, int q_dtype, int64_t num_tokens, int64_t Hq, int64_t D, int64_t q_stride_t,
                                          int64_t q_stride_h, const void *k_cache, const void *v_cache, int cache_kind, int64_t num_pages,
                                          int64_t page_size, int64_t Hkv, const float *k_scale_inv, const float *v_scale_inv,
                                          const void *key_ranges, const int32_t *page_table, int64_t table_stride, int64_t max_pages,
                                          const int32_t *cu_seqlens_q, const int32_t *seq_lens, int64_t num_seqs, int64_t num_selected,
                                          int64_t num_first, int64_t num_last, float softmax_scale, void *out, float *lse,
                                          void *workspace, size_t workspace_bytes, pta_stream_t stream) {
    clear_error();
    if (int rc = ps_check(num_tokens, num_seqs, Hq, Hkv, D, num_pages, page_size, max_pages, num_selected, num_first, num_last)) return rc;
    PTA_CHECK_ARG(softmax_scale > 0.0f && softmax_scale - softmax_scale == 0.0f, "softmax_scale must be positive and finite");
    if (num_tokens == 0) return PTA_OK;
    PTA_CHECK_ARG(num_seqs > 0, "tokens without a sequence");
    const SparsePlan p = sparse_plan(num_tokens, num_seqs, Hq, Hkv, D, max_pages, page_size, num_selected);
    PTA_CHECK_ARG(workspace && aligned16(workspace) && workspace_bytes >= p.bytes(), "workspace too small: %zu bytes needed, %zu given",
                  p.bytes(), workspace_bytes);
    uint8_t *w    = static_cast<uint8_t *>(workspace);
    uint8_t *sel  = w;
    uint8_t *masks = w += p.sel, *counts = w += p.masks, *pos = w += p.counts;
    int32_t *lens = reinterpret_cast<int32_t *>(w += p.pos), *cu = reinterpret_cast<int32_t *>(w += p.lens);
    uint8_t *rest = w += p.cu;
    PSTiles  tiles = {};
    tiles.tokens = static_cast<int>(p.tile);
    tiles.cap    = static_cast<int>(p.cap);
    tiles.list   = reinterpret_cast<int2 *>(sel);
    tiles.masks  = reinterpret_cast<uint16_t *>(masks);
    tiles.counts = reinterpret_cast<int32_t *>(counts);
    tiles.pos    = reinterpret_cast<int32_t *>(pos);
    // all arguments are checked before the first launch
    const int32_t *table = p.tile > 0 ? page_table : reinterpret_cast<const int32_t *>(sel);
    AttnArgs       a;
    if (int rc = attn_arguments(a, q, q_dtype, num_tokens, Hq, D, q_stride_t, q_stride_h, k_cache, v_cache, cache_kind, num_pages, page_size,
                                Hkv, k_scale_inv, v_scale_inv, table, Hkv * p.K, std::max<int64_t>(p.K, 1), p.K, cu, lens, num_tokens,
                                softmax_scale, 0, 0, out, lse))
        return rc;
    const hipStream_t st = as_stream(stream);
    if (int rc = ps_select(q, q_dtype, num_tokens, Hq, D, q_stride_t, q_stride_h, key_ranges, num_pages, page_size, Hkv, page_table,
                           table_stride, max_pages, cu_seqlens_q, seq_lens, num_seqs, num_selected, num_first, num_last,
                           reinterpret_cast<int32_t *>(sel), p.tile > 0 ? &tiles : nullptr, lens, cu, rest, st))
        return rc;
    if (p.tile == 0)
        return attn_call(q, q_dtype, num_tokens, Hq, D, q_stride_t, q_stride_h, k_cache, v_cache, cache_kind, num_pages, page_size, Hkv,
                         k_scale_inv, v_scale_inv, table, Hkv * p.K, std::max<int64_t>(p.K, 1), p.K, cu, lens, num_tokens, softmax_scale, 0, 0,
                         out, lse, rest, p.rest, stream);
    a.tiles     = tiles;
    a.B         = static_cast<int>(p.tiles);
    a.rows_max  = INT_MAX;
    a.split     = static_cast<int>(p.part.split);
    a.part_step = static_cast<int>(p.part.part_step);
    a.part_ml   = reinterpret_cast<float2 *>(rest);
    a.part_o    = reinterpret_cast<float *>(rest + p.part.ml_bytes);
    if (q_dtype == PTA_BF16) attn_launch_tiles<PTA_BF16>(a, cache_kind, st);
    else attn_launch_tiles<PTA_F16>(a, cache_kind, st);
    PTA_CHECK_LAUNCH();
    return PTA_OK;
}
