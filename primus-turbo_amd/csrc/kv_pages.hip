// Pages of a paged key / value cache as wholes: copied, and their books kept on the
// device: sequences that go on from others share full pages, get copies of the
// partly filled last one and fresh pages for what comes, the pages of sequences that
// nobody goes on from are free, and pages in use can be moved to the front.
//
// A page is up to five runs of bytes: keys, values, their scales and the keys'
// ranges, in each of the layers.  Copies are bound by memory: a workgroup moves 16 KB
// of one run at a time, 4 x 16 bytes a thread in flight (4 KB where there is little to
// copy): 5.1 TB/s, what a large copy reaches.
#include <algorithm>
#include <climits>

#include "common.h"

namespace pta {
namespace {

constexpr int KP_NT = 256, KP_RUNS = 5;
// 16-byte pieces of a thread: four where that gives every CU two workgroups (1000 pages of 8 KB in
// 16 layers: 102 us, 102 with two, 218 with eight), else one (8 pages of 136 KB: 3.1 us, 9.7 with
// four).  More bytes than the last cache holds go past it (102 us, 108 through it; 48 pages of
// 139 KB in 8 layers, which the next attention reads: 10.5 and 7.3).
constexpr int    KP_DEPTH = 4;
constexpr double KP_CACHED = 256e6;
constexpr int64_t kp_chunk(int depth) { return static_cast<int64_t>(KP_NT) * depth * 16; } // bytes of a workgroup

struct KPPool {
    uint8_t *p[KP_RUNS];
    int64_t  bytes[KP_RUNS];  // of a page
    int64_t  layer[KP_RUNS];  // to the next layer
    int      first[KP_RUNS];  // number of its first chunk
    int      wide[KP_RUNS];   // 16-byte pieces, else 4-byte ones
    int      runs, chunks, layers;
    int64_t  pages;
};

// Chunk c (of layer and run) of page `to` becomes that of page `from`
template <int DEPTH, bool PAST> __device__ __forceinline__ void kp_copy(const KPPool &a, int64_t from, int64_t to, int layer, int c) {
    // by comparisons: an index that the compiler does not know would put the arguments into memory
    uint8_t *p = a.p[0];
    int64_t  bytes = a.bytes[0], per_layer = a.layer[0];
    int      first = 0, wide = a.wide[0];
#pragma unroll
    for (int i = 1; i < KP_RUNS; ++i)
        if (i < a.runs && c >= a.first[i]) {
            p = a.p[i];
            bytes = a.bytes[i]; per_layer = a.layer[i];
            first = a.first[i]; wide = a.wide[i];
        }
    const int64_t at = (c - first) * kp_chunk(DEPTH), n = min(bytes - at, kp_chunk(DEPTH));
    p += layer * per_layer + at;
    const uint8_t *src = p + from * bytes;
    uint8_t       *dst = p + to * bytes;
    if (wide) {
        typedef uint32_t piece __attribute__((ext_vector_type(4)));
        piece v[DEPTH];
#pragma unroll
        for (int i = 0; i < DEPTH; ++i) {
            const int64_t o = (i * KP_NT + static_cast<int>(threadIdx.x)) * 16;
            if (o < n) v[i] = PAST ? __builtin_nontemporal_load(reinterpret_cast<const piece *>(src + o)) : *reinterpret_cast<const piece *>(src + o);
        }
#pragma unroll
        for (int i = 0; i < DEPTH; ++i) {
            const int64_t o = (i * KP_NT + static_cast<int>(threadIdx.x)) * 16;
            if (o >= n) continue;
            if constexpr (PAST) __builtin_nontemporal_store(v[i], reinterpret_cast<piece *>(dst + o));
            else *reinterpret_cast<piece *>(dst + o) = v[i];
        }
    } else {
        for (int64_t o = threadIdx.x * 4; o < n; o += KP_NT * 4)
            *reinterpret_cast<uint32_t *>(dst + o) = *reinterpret_cast<const uint32_t *>(src + o);
    }
}

__device__ __forceinline__ int64_t kp_index(const void *p, int i64, int64_t i) {
    return i64 ? reinterpret_cast<const int64_t *>(p)[i] : static_cast<int64_t>(reinterpret_cast<const int32_t *>(p)[i]);
}

template <int DEPTH, bool PAST> __global__ __launch_bounds__(KP_NT) void kp_copy_kernel(KPPool a, const void *src, const void *dst, int i64, int64_t total) {
    const int per = a.chunks * a.layers;
    for (int64_t w = blockIdx.x; w < total; w += gridDim.x) {
        const int64_t pair = w / per;
        const int     rest = static_cast<int>(w - pair * per), layer = rest / a.chunks;
        const int64_t s = kp_index(src, i64, pair), d = kp_index(dst, i64, pair);
        if (s < 0 || s >= a.pages || d < 0 || d >= a.pages || s == d) continue;
        kp_copy<DEPTH, PAST>(a, s, d, layer, rest - layer * a.chunks);
    }
}

// ---- the books -------------------------------------------------------------------
struct KFArgs {
    const int32_t *table;
    int64_t        table_st;
    const int32_t *lens;
    const void    *parents; // null: every sequence goes on from itself
    int            parents_i64;
    int            B, N, M, page, P;
    int64_t        reserve;
    int            compact;
    int32_t       *new_table, *new_lens; // [N, M], [N]
    // workspace
    int32_t *owner;      // [P] who has the page: N nobody, -1 everybody (it is full), else the sequence whose last page it is
    int32_t *free_pages; // [P] in rising order, as many as are taken
    int32_t *moved;      // [P] where pages at or past `bound` go (compact)
    int2    *seq;        // [N] place of its first fresh page among the free ones, -1: it came too late; 1 if that is a copy
    int2    *pairs;      // copies: from, to
    int32_t *count;      // pairs; bound
};

struct KFSeq {
    int parent, full, part, has, want; // full pages, 1 for a partly filled one, their sum, pages afterwards
    int last;                          // page that is partly filled, -1: none of the pool's
};

__device__ __forceinline__ KFSeq kf_seq(const KFArgs &a, int i) {
    KFSeq         s = {-1, 0, 0, 0, 0, -1};
    const int64_t p = a.parents ? kp_index(a.parents, a.parents_i64, i) : i;
    if (p < 0 || p >= a.B) return s;
    s.parent        = static_cast<int>(p);
    if (a.lens[p] < 0) return s; // pages had run out for it
    const int64_t most = static_cast<int64_t>(a.M) * a.page;
    const int64_t len  = min(static_cast<int64_t>(a.lens[p]), most);
    s.full = static_cast<int>(len / a.page);
    s.part = len - static_cast<int64_t>(s.full) * a.page > 0;
    s.has  = s.full + s.part;
    s.want = static_cast<int>(min((len + a.reserve + a.page - 1) / a.page, static_cast<int64_t>(a.M)));
    if (s.part) {
        const int u = a.table[s.parent * a.table_st + s.full];
        s.last      = u >= 0 && u < a.P ? u : -1;
    }
    return s;
}

__global__ __launch_bounds__(KP_NT) void kf_init_kernel(KFArgs a) {
    for (int u = blockIdx.x * KP_NT + threadIdx.x; u < a.P; u += gridDim.x * KP_NT) a.owner[u] = a.N;
}

__global__ __launch_bounds__(KP_NT) void kf_mark_kernel(KFArgs a) {
    const int   i = blockIdx.x;
    const KFSeq s = kf_seq(a, i);
    for (int j = threadIdx.x; j < s.has; j += KP_NT) {
        const int u = a.table[s.parent * a.table_st + j];
        if (u >= 0 && u < a.P) atomicMin(&a.owner[u], j < s.full ? -1 : i);
    }
}

constexpr int KF_NT = 1024;

// exclusive sums over the workgroup's threads, and the totals
struct KFSums {
    int x, y, z;
};
__device__ __forceinline__ KFSums kf_scan(KFSums v, int4 *tmp, KFSums &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    KFSums    s = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int x = __shfl_up(s.x, o), y = __shfl_up(s.y, o), z = __shfl_up(s.z, o);
        if (lane >= o) {
            s.x += x;
            s.y += y;
            s.z += z;
        }
    }
    __syncthreads();
    if (lane == 63) tmp[wave] = make_int4(s.x, s.y, s.z, 0);
    __syncthreads();
    KFSums before = {0, 0, 0};
    total         = {0, 0, 0};
#pragma unroll
    for (int w = 0; w < KF_NT / 64; ++w) {
        const int4 t = tmp[w];
        const int  m = w < wave ? -1 : 0;
        before.x += t.x & m;
        before.y += t.y & m;
        before.z += t.z & m;
        total.x += t.x;
        total.y += t.y;
        total.z += t.z;
    }
    return {before.x + s.x - v.x, before.y + s.y - v.y, before.z + s.z - v.z};
}

// One workgroup: a thread has a run of pages, and of sequences.  Where LDS holds the pages'
// owners and the table's entries are few, they are found here, else by the two kernels
// above (64 sequences of 66 pages over 4300: 8.5 us, the three kernels 13).  Past that the runs
// are strided reads of memory by one workgroup: calls of 64 sequences over 12289 pages 26 us (over
// 12288 in LDS 19), over 65536 73, over 200000 225; compacting 35 (25), 128 and 364.
constexpr int     KF_LDS_PAGES = 12 * 1024;
constexpr int64_t KF_LDS_ENTRIES = 128 * KF_NT;

template <bool LDS> __global__ __launch_bounds__(KF_NT) void kf_plan_kernel(KFArgs a) {
    __shared__ int4 tmp[KF_NT / 64];
    __shared__ int  own[LDS ? KF_LDS_PAGES : 1];
    __shared__ int  row[LDS ? KF_NT : 1], full[LDS ? KF_NT : 1], has[LDS ? KF_NT : 1];
    int            *owner = LDS ? own : a.owner;
    const int tid = threadIdx.x;
    const int pr = (a.P + KF_NT - 1) / KF_NT, p0 = min(tid * pr, a.P), p1 = min(p0 + pr, a.P);
    const int nr = LDS ? 1 : (a.N + KF_NT - 1) / KF_NT, n0 = min(tid * nr, a.N), n1 = min(n0 + nr, a.N);
    // the thread's first sequence, mostly its only one, is looked up once
    const KFSeq mine = n0 < n1 ? kf_seq(a, n0) : KFSeq{-1, 0, 0, 0, 0, -1};
    if constexpr (LDS) { // a sequence a thread
        row[tid]  = max(mine.parent, 0);
        full[tid] = mine.full;
        has[tid]  = mine.has;
        for (int u = tid; u < a.P; u += KF_NT) own[u] = a.N;
        __syncthreads();
        const int entries = a.N * a.M;
#pragma unroll 4
        for (int x = tid; x < entries; x += KF_NT) {
            const int i = x / a.M, j = x - i * a.M;
            const int u = j < has[i] ? a.table[row[i] * a.table_st + j] : -1;
            if (u >= 0 && u < a.P) atomicMin(&own[u], j < full[i] ? -1 : i);
        }
        __syncthreads();
    }
    auto seq = [&](int i) __attribute__((always_inline)) { return i == n0 ? mine : kf_seq(a, i); };
    // whether the sequence's last page is another's too
    auto copied = [&](int i, const KFSeq &s) __attribute__((always_inline)) { return s.last >= 0 && owner[s.last] != i ? 1 : 0; };
    KFSums v = {0, 0, 0}, need, total; // pages in use, fresh ones, copies among these
    for (int u = p0; u < p1; ++u) v.x += owner[u] < a.N;
    for (int i = n0; i < n1; ++i) {
        const KFSeq s = seq(i);
        const int   c = copied(i, s);
        v.y += s.want - s.has + c;
        v.z += c;
    }
    KFSums    at    = kf_scan(v, tmp, need);
    const int nfree = a.P - need.x;
    // pages at or past `bound` move to the first free ones
    const int bound = a.compact ? need.x + min(need.y, nfree) : a.P;
    v               = {0, 0, 0}; // free pages, pages that move
    for (int u = p0; u < p1; ++u) {
        if (owner[u] >= a.N) ++v.x;
        else if (u >= bound) ++v.y;
    }
    const KFSums rank = kf_scan(v, tmp, total);
    const int    moves = total.y, taken = moves + min(need.y, nfree);
    for (int u = p0, f = rank.x; u < p1 && f < taken; ++u)
        if (owner[u] >= a.N) a.free_pages[f++] = u;
    __syncthreads(); // the free pages are in place
    if (moves > 0)
        for (int u = max(p0, bound), m = rank.y; u < p1; ++u)
            if (owner[u] < a.N) {
                const int to = a.free_pages[m];
                a.moved[u]   = to;
                a.pairs[m++] = make_int2(u, to);
            }
    for (int i = n0; i < n1; ++i) {
        const KFSeq s = seq(i);
        const int   c = copied(i, s), f = s.want - s.has + c;
        // sequences take their pages in order; those that come too late get none
        const bool none = f > 0 && at.y + f > nfree;
        a.seq[i]        = make_int2(none ? -1 : moves + at.y, c);
        if (c) a.pairs[moves + at.z] = none ? make_int2(-1, -1) : make_int2(s.last, a.free_pages[moves + at.y]);
        at.y += f;
        at.z += c;
    }
    if (tid == 0) {
        a.count[0] = moves + need.z;
        a.count[1] = bound;
    }
}

// The first N workgroups write the sequences' rows, the others copy pages
template <int DEPTH, bool PAST> __global__ __launch_bounds__(KP_NT) void kf_apply_kernel(KFArgs a, KPPool pool) {
    const int i = blockIdx.x;
    if (i < a.N) {
        const KFSeq s = kf_seq(a, i);
        const int2  plan = a.seq[i];
        const int   bound = a.count[1], kept = s.has - plan.y;
        for (int j = threadIdx.x; j < a.M; j += KP_NT) {
            int u = -1;
            if (plan.x >= 0 && j < s.want) {
                if (j < kept) {
                    u = a.table[s.parent * a.table_st + j];
                    if (u >= bound && u < a.P) u = a.moved[u];
                } else {
                    u = a.free_pages[plan.x + j - kept];
                }
            }
            a.new_table[static_cast<int64_t>(i) * a.M + j] = u;
        }
        if (threadIdx.x == 0) a.new_lens[i] = plan.x < 0 ? -1 : s.parent < 0 ? 0 : a.lens[s.parent];
        return;
    }
    const int     per   = pool.chunks * pool.layers;
    const int64_t total = static_cast<int64_t>(a.count[0]) * per;
    for (int64_t w = i - a.N; w < total; w += gridDim.x - a.N) {
        const int64_t pair = w / per;
        const int     rest = static_cast<int>(w - pair * per), layer = rest / pool.chunks;
        const int2    p = a.pairs[pair];
        if (p.x >= 0) kp_copy<DEPTH, PAST>(pool, p.x, p.y, layer, rest - layer * pool.chunks);
    }
}

// How a copy goes
struct KPForm {
    int  depth; // pieces of a thread
    bool past;  // the caches
};

// `pairs`: of pages to copy at most
int kp_pool(KPPool &a, KPForm &form, int64_t pairs, void *k_cache, void *v_cache, int kind, int64_t layers, int64_t num_pages, int64_t Hkv,
            int64_t page_size, int64_t D, float *k_scale, float *v_scale, void *ranges) {
    PTA_CHECK_ARG(kind == PTA_E4M3 || kind == PTA_E5M2 || kind == PTA_CACHE_16BIT, "unknown cache kind %d", kind);
    PTA_CHECK_ARG(layers >= 0 && num_pages >= 0 && page_size > 0 && Hkv > 0, "bad cache sizes");
    PTA_CHECK_ARG(D >= 16 && D <= 256 && D % 16 == 0, "head_dim must be a multiple of 16 in [16, 256] (got %lld)", static_cast<long long>(D));
    PTA_CHECK_ARG(page_size <= INT_MAX && Hkv <= INT_MAX && num_pages <= INT_MAX / page_size && num_pages * page_size <= INT_MAX / Hkv,
                  "the cache has 2^31 rows (pages * page_size * heads) or more");
    a.layers = static_cast<int>(std::min<int64_t>(layers, INT_MAX));
    a.pages  = num_pages;
    if (layers == 0 || num_pages == 0) return PTA_OK;
    PTA_CHECK_ARG(k_cache && v_cache, "null cache");
    PTA_CHECK_ARG(aligned16(k_cache) && aligned16(v_cache) && aligned16(ranges), "cache pools must be 16-byte aligned");
    PTA_CHECK_ARG(kind == PTA_CACHE_16BIT || (k_scale && v_scale), "an fp8 cache needs its scales");
    const bool    fp8 = kind != PTA_CACHE_16BIT;
    const int64_t data = Hkv * page_size * D * (fp8 ? 1 : 2), scale = Hkv * page_size * 4;
    void   *const p[KP_RUNS] = {k_cache, v_cache, fp8 ? k_scale : nullptr, fp8 ? v_scale : nullptr, ranges};
    const int64_t bytes[KP_RUNS] = {data, data, scale, scale, Hkv * D * 4};
    int64_t       all = 0;
    for (int i = 0; i < KP_RUNS; ++i) all += p[i] == nullptr ? 0 : bytes[i];
    const double moved = static_cast<double>(all) * layers * pairs;
    form.depth = moved < static_cast<double>(kp_chunk(KP_DEPTH)) * 2 * device_cu_count() ? 1 : KP_DEPTH;
    form.past  = form.depth > 1 && 2 * moved > KP_CACHED;
    int64_t chunks = 0;
    for (int i = 0; i < KP_RUNS; ++i) {
        if (p[i] == nullptr) continue;
        const int r = a.runs++;
        a.p[r] = static_cast<uint8_t *>(p[i]);
        a.bytes[r] = bytes[i];
        a.layer[r] = bytes[i] * num_pages;
        a.first[r] = static_cast<int>(chunks);
        a.wide[r]  = aligned16(p[i]) && bytes[i] % 16 == 0;
        chunks += cdiv(bytes[i], kp_chunk(form.depth));
    }
    PTA_CHECK_ARG(layers <= INT_MAX / chunks, "too many layers");
    a.chunks = static_cast<int>(chunks);
    return PTA_OK;
}

// Workgroups of a copy: a CU's share of work many times over, so that they end together
unsigned kp_blocks(int64_t total) { return static_cast<unsigned>(std::min<int64_t>(total, 64ll * device_cu_count())); }

struct KFPlan {
    int64_t pairs;
    size_t  owner, free_pages, moved, seq, count, pair_bytes;
    size_t  bytes() const { return owner + free_pages + moved + seq + count + pair_bytes; }
};
size_t kf_round(int64_t n) { return static_cast<size_t>(cdiv(n, 16) * 16); }
KFPlan kf_plan(int64_t N, int64_t M, int64_t P, int compact) {
    KFPlan p     = {};
    p.pairs      = N + (compact ? std::min(P, N * M) : 0);
    p.owner      = kf_round(P * 4);
    p.free_pages = kf_round(P * 4);
    p.moved      = compact ? kf_round(P * 4) : 0;
    p.seq        = kf_round(N * 8);
    p.count      = 16;
    p.pair_bytes = kf_round(p.pairs * 8);
    return p;
}

} // namespace
} // namespace pta

using namespace pta;

extern "C" int pta_kv_cache_copy(void *k_cache, void *v_cache, int cache_kind, int64_t num_layers, int64_t num_pages, int64_t Hkv,
                                 int64_t page_size, int64_t D, float *k_scale_inv, float *v_scale_inv, void *key_ranges,
                                 const void *src_pages, const void *dst_pages, int pages_i64, int64_t num_pairs, pta_stream_t stream) {
    clear_error();
    KPPool a = {};
    KPForm form = {1, false};
    if (int rc = kp_pool(a, form, num_pairs, k_cache, v_cache, cache_kind, num_layers, num_pages, Hkv, page_size, D, k_scale_inv, v_scale_inv, key_ranges)) return rc;
    PTA_CHECK_ARG(num_pairs >= 0 && num_pairs <= INT_MAX, "bad number of pages");
    if (num_pairs == 0 || num_layers == 0 || num_pages == 0) return PTA_OK;
    PTA_CHECK_ARG(src_pages && dst_pages, "null page list");
    const int64_t total = num_pairs * a.chunks * a.layers;
    const auto    kernel = form.depth == 1 ? kp_copy_kernel<1, false> : form.past ? kp_copy_kernel<KP_DEPTH, true> : kp_copy_kernel<KP_DEPTH, false>;
    kernel<<<kp_blocks(total), KP_NT, 0, as_stream(stream)>>>(a, src_pages, dst_pages, pages_i64, total);
    PTA_CHECK_LAUNCH();
    return PTA_OK;
}

extern "C" size_t pta_kv_cache_fork_workspace_size(int64_t num_new_seqs, int64_t max_pages, int64_t num_pages, int compact) {
    if (num_new_seqs <= 0 || max_pages < 0 || num_pages < 0) return 0;
    return kf_plan(num_new_seqs, max_pages, num_pages, compact).bytes();
}

extern "C" int pta_kv_cache_fork(void *k_cache, void *v_cache, int cache_kind, int64_t num_layers, int64_t num_pages, int64_t Hkv,
                                 int64_t page_size, int64_t D, float *k_scale_inv, float *v_scale_inv, void *key_ranges,
                                 const int32_t *page_table, int64_t table_stride, int64_t max_pages, const int32_t *seq_lens,
                                 int64_t num_seqs, const void *parents, int parents_i64, int64_t num_new_seqs, int64_t reserve, int compact,
                                 int32_t *new_page_table, int32_t *new_seq_lens, void *workspace, size_t workspace_bytes,
                                 pta_stream_t stream) {
    clear_error();
    KPPool pool = {};
    KPForm form = {1, false};
    if (int rc = kp_pool(pool, form, num_new_seqs + (compact ? num_pages : 0), k_cache, v_cache, cache_kind, num_layers, num_pages, Hkv, page_size, D, k_scale_inv, v_scale_inv, key_ranges)) return rc;
    PTA_CHECK_ARG(num_seqs >= 0 && num_new_seqs >= 0 && max_pages >= 0 && reserve >= 0, "bad sizes");
    PTA_CHECK_ARG(num_seqs < (1 << 24) && num_new_seqs < (1 << 24) && max_pages <= (INT_MAX - 1024) / page_size &&
                      max_pages <= INT_MAX / 2 / std::max<int64_t>(1, num_new_seqs) - 1,
                  "page_table has too many entries");
    PTA_CHECK_ARG(parents || num_new_seqs == num_seqs, "without parents there are as many new sequences as old ones");
    if (num_new_seqs == 0) return PTA_OK;
    PTA_CHECK_ARG(new_seq_lens && (max_pages == 0 || new_page_table) && (num_seqs == 0 || (seq_lens && (max_pages == 0 || page_table))),
                  "null pointer");
    const KFPlan p = kf_plan(num_new_seqs, max_pages, num_pages, compact);
    PTA_CHECK_ARG(workspace && aligned16(workspace) && workspace_bytes >= p.bytes(), "workspace too small: %zu bytes needed, %zu given",
                  p.bytes(), workspace_bytes);
    KFArgs a = {};
    a.table = page_table; a.table_st = table_stride; a.lens = seq_lens;
    a.parents = parents; a.parents_i64 = parents_i64;
    a.B = static_cast<int>(num_seqs); a.N = static_cast<int>(num_new_seqs); a.M = static_cast<int>(max_pages);
    a.page = static_cast<int>(page_size); a.P = static_cast<int>(num_pages);
    a.reserve = std::min<int64_t>(reserve, INT_MAX); a.compact = compact != 0;
    a.new_table = new_page_table; a.new_lens = new_seq_lens;
    uint8_t *w = static_cast<uint8_t *>(workspace);
    a.owner      = reinterpret_cast<int32_t *>(w);
    a.free_pages = reinterpret_cast<int32_t *>(w += p.owner);
    a.moved      = reinterpret_cast<int32_t *>(w += p.free_pages);
    a.seq        = reinterpret_cast<int2 *>(w += p.moved);
    a.count      = reinterpret_cast<int32_t *>(w += p.seq);
    a.pairs      = reinterpret_cast<int2 *>(w += p.count);
    const hipStream_t st = as_stream(stream);
    if (num_pages <= KF_LDS_PAGES && num_new_seqs <= KF_NT && num_new_seqs * max_pages <= KF_LDS_ENTRIES) {
        kf_plan_kernel<true><<<1, KF_NT, 0, st>>>(a);
    } else {
        if (num_pages > 0) {
            kf_init_kernel<<<static_cast<unsigned>(std::min<int64_t>(cdiv(num_pages, KP_NT), 4 * device_cu_count())), KP_NT, 0, st>>>(a);
            PTA_CHECK_LAUNCH();
        }
        kf_mark_kernel<<<static_cast<unsigned>(a.N), KP_NT, 0, st>>>(a);
        PTA_CHECK_LAUNCH();
        kf_plan_kernel<false><<<1, KF_NT, 0, st>>>(a);
    }
    PTA_CHECK_LAUNCH();
    const int64_t total = num_pages > 0 ? p.pairs * pool.chunks * pool.layers : 0;
    const auto    apply = form.depth == 1 ? kf_apply_kernel<1, false> : form.past ? kf_apply_kernel<KP_DEPTH, true> : kf_apply_kernel<KP_DEPTH, false>;
    apply<<<static_cast<unsigned>(a.N) + kp_blocks(total), KP_NT, 0, st>>>(a, pool);
    PTA_CHECK_LAUNCH();
    return PTA_OK;
}
