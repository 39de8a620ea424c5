// What the kernels of attention over a paged cache share: where keys lie, which of them a row sees, and a row computed key by key.
#pragma once
#include <cuda_bf16.h>

#include "wf_common.cuh"

namespace wf {

typedef __nv_bfloat16 bf16;

constexpr int ATTN_MAX_DIM = 128;
constexpr int TREE_MAX_DRAFTS = 64;  // a row's ancestors are one 64-bit word
constexpr int64_t ATTN_CALL_BYTES = 1LL << 30;  // of a selection's scores, or of rows' sums over a prefix, that a call may have in its stream's scratch

// What rows attend to: a prompt's past and itself; a sequence's context and new tokens; a list of pages for each token and kv head; where sequences have a prefix in
// common, that prefix (the rows of all of them), and what a sequence has of its own behind it; or both, a sequence at a time.
enum AttentionKind { ATTEND_PROMPT, ATTEND_TREE, ATTEND_LISTS, ATTEND_PREFIX, ATTEND_OWN, ATTEND_WHOLE };

// One layer of the cache, or packed keys and values (page_shift 0, a page a token).
struct CacheView {
    bf16* keys;
    bf16* values;
    int64_t pages;
    int kv_heads, dim;
    int page_shift;  // log2 of the tokens of a page
    // first element of (page, head, row)
    __host__ __device__ __forceinline__ size_t at(int64_t page, int head, int row) const {
        return ((((size_t)page * kv_heads + head) << page_shift) + row) * dim;
    }
};

// Keys of one sequence.  table == nullptr: packed, token t is page first + t.  A page outside the cache is never followed: its keys
// are not seen and the status says so.
struct KeyPlace {
    const int* table;
    int64_t first;
    __device__ __forceinline__ int64_t page_of(const CacheView& c, int t) const { return table ? (int64_t)table[t >> c.page_shift] : first + t; }
};

struct PromptParams {
    CacheView cache;
    const bf16* q;
    bf16* out;
    int64_t q_stride;
    const int* q_offsets;
    const int* tables;
    int64_t table_stride;
    const int* k_lens;
    int64_t tokens;
    int seqs, q_heads, group;
    float scale_log2;  // scale * log2(e): the softmax is taken to base 2
    int* status;
};

struct TreeParams {
    CacheView cache;
    const bf16* q;
    bf16* out;
    int64_t q_stride;
    const int* q_offsets;
    const int* tables;
    int64_t table_stride;
    const int* context;
    const uint64_t* ancestors;
    int64_t tokens, max_context;
    int seqs, q_heads, group, max_drafts;
    uint32_t group_inverse;  // 2^32 / group, rounded up; 0 for a group of one
    float scale_log2;
    int* status;
    // lists: tables is int32 [tokens][kv_heads][table_stride], and for each: tokens of the context in the list, keys in all
    const int2* lens;
    // prefixes: sequences groups[g] .. groups[g + 1] - 1 have prefix[g] tokens in common, whose pages the first one's table names
    const int* groups;
    const int* prefix;
    int64_t max_prefix;
    int n_groups;
    int2* prefix_of;  // [seqs], made by the kernel that reads the prefixes: prefix (-1: cannot be, or has no sums for these rows) and first sequence of the group
    float* state;     // of every row over its prefix: sums [tokens * q_heads][state_dim], then maxima, then sums of weights
    int state_dim;
#ifdef __CUDACC__
    __device__ __forceinline__ float* state_maxima() const { return state + (size_t)tokens * q_heads * state_dim; }
    __device__ __forceinline__ float* state_weights() const { return state_maxima() + (size_t)tokens * q_heads; }
    // row / group, for the rows of a sequence (64 x 128 at most)
    __device__ __forceinline__ int token_of(int row) const { return group_inverse ? (int)__umulhi((uint32_t)row, group_inverse) : row; }
#endif
};

#ifdef __CUDACC__
// The rows and keys of a sequence, as the device arrays have them; values that cannot be are cut down and reported.
struct PromptSeq {
    int row0, rows, keys;
    KeyPlace place;
};
__device__ __forceinline__ PromptSeq prompt_seq(const PromptParams& p, int s) {
    PromptSeq q;
    const int a = p.q_offsets[s], b = p.q_offsets[s + 1];
    const bool bad = a < 0 || b < a || (int64_t)b > p.tokens;
    q.row0 = bad ? 0 : a;
    q.rows = bad ? 0 : b - a;
    q.keys = p.tables ? p.k_lens[s] : q.rows;
    const int64_t most = p.tables ? p.table_stride << p.cache.page_shift : p.cache.pages - q.row0;
    const bool bad_keys = q.keys < 0 || (int64_t)q.keys > most;
    if (bad_keys) q.keys = 0;
    if (bad || bad_keys) report_status(p.status, STATUS_BAD_INDEX);
    q.place.table = p.tables ? p.tables + (size_t)s * p.table_stride : nullptr;
    q.place.first = q.row0;
    return q;
}
// Keys of a sequence behind a prefix that lies in another one's pages.
struct SharedPlace {
    const int* first;
    int prefix;
    const int* table;
    __device__ __forceinline__ int64_t page_of(const CacheView& c, int t) const { return (t < prefix ? first : table)[t >> c.page_shift]; }
};
struct TreeSeq {
    int row0, rows, context;
    int news;    // keys behind the context
    int prefix;  // own keys: tokens before them, which other kernels have seen to; whole sequences: tokens in the pages of another one
    int first;   // whole sequences: that one
    KeyPlace place;
};
__device__ __forceinline__ TreeSeq tree_seq(const TreeParams& p, int s) {
    TreeSeq q;
    const int64_t a = p.q_offsets ? p.q_offsets[s] : (int64_t)s * p.max_drafts, b = p.q_offsets ? p.q_offsets[s + 1] : a + p.max_drafts;
    const bool bad = a < 0 || b < a || b > p.tokens || b - a > p.max_drafts;
    q.row0 = bad ? 0 : (int)a;
    q.rows = bad ? 0 : (int)(b - a);
    q.context = p.context[s];
    const bool bad_keys = q.context < 0 || (int64_t)q.context > p.max_context || (int64_t)q.context + q.rows > (p.table_stride << p.cache.page_shift);
    if (bad_keys) q.context = -1;  // its rows are zeros
    if (bad || bad_keys) report_status(p.status, STATUS_BAD_INDEX);
    q.news = q.rows;
    q.place.table = p.tables + (size_t)s * p.table_stride;
    q.place.first = 0;
    return q;
}
// A token's list for a kv head (s counts both): one row of the group.
__device__ __forceinline__ TreeSeq list_seq(const TreeParams& p, int s) {
    TreeSeq q;
    const int2 lens = p.lens[s];
    const bool bad = lens.x < 0 || lens.y < lens.x || lens.y - lens.x > TREE_MAX_DRAFTS || (int64_t)lens.y > p.table_stride << p.cache.page_shift;
    if (bad) report_status(p.status, STATUS_BAD_INDEX);
    q.row0 = s / p.cache.kv_heads;
    q.rows = 1;
    q.context = bad ? -1 : lens.x;  // its rows are zeros
    q.news = bad ? 0 : lens.y - lens.x;
    q.place.table = p.tables + (size_t)s * p.table_stride;
    q.place.first = 0;
    return q;
}
// The rows of a group of sequences, over the prefix that they share.  prefix: -1 where the group cannot be.
struct GroupSeqs {
    int first, stop, prefix;
};
__device__ __forceinline__ GroupSeqs group_seqs(const TreeParams& p, int g) {
    GroupSeqs q;
    q.first = p.groups[g], q.stop = p.groups[g + 1], q.prefix = p.prefix[g];
    if (q.first < 0 || q.stop < q.first || q.stop > p.seqs || q.prefix < 0 || (int64_t)q.prefix > p.max_prefix || q.prefix & ((1 << p.cache.page_shift) - 1) ||
        (int64_t)q.prefix > p.table_stride << p.cache.page_shift) {
        report_status(p.status, STATUS_BAD_INDEX);
        q.prefix = -1;
        q.first = max(0, min(q.first, p.seqs));
        q.stop = max(q.first, min(q.stop, p.seqs));
    }
    return q;
}
// Whether a sequence's rows lie among those of its group: the others have no sums over the prefix.
__device__ __forceinline__ bool rows_in_group(const TreeParams& p, const GroupSeqs& g, int s) {
    if (!p.q_offsets || g.prefix <= 0) return true;
    const int from = p.q_offsets[g.first], to = p.q_offsets[g.stop], a = p.q_offsets[s], b = p.q_offsets[s + 1];
    return from >= 0 && from <= a && a <= b && b <= to && to <= p.tokens;
}
__device__ __forceinline__ TreeSeq prefix_seq(const TreeParams& p, int g) {
    TreeSeq q;
    const GroupSeqs of = group_seqs(p, g);
    const bool some = of.prefix > 0 && of.stop > of.first;
    int64_t a = 0, b = 0;
    if (some) {
        a = p.q_offsets ? p.q_offsets[of.first] : (int64_t)of.first * p.max_drafts;
        b = p.q_offsets ? p.q_offsets[of.stop] : (int64_t)of.stop * p.max_drafts;
    }
    const bool bad = a < 0 || b < a || b > p.tokens;
    if (bad) report_status(p.status, STATUS_BAD_INDEX);
    q.row0 = bad ? 0 : (int)a;
    q.rows = bad ? 0 : (int)(b - a);
    q.context = max(0, of.prefix);
    q.news = 0;
    q.place.table = p.tables + (size_t)(some ? of.first : 0) * p.table_stride;
    q.place.first = 0;
    return q;
}
// What a sequence has behind its prefix.
__device__ __forceinline__ TreeSeq own_seq(const TreeParams& p, int s) {
    TreeSeq q;
    const int64_t a = p.q_offsets ? p.q_offsets[s] : (int64_t)s * p.max_drafts, b = p.q_offsets ? p.q_offsets[s + 1] : a + p.max_drafts;
    const bool bad = a < 0 || b < a || b > p.tokens || b - a > p.max_drafts;
    q.row0 = bad ? 0 : (int)a;
    q.rows = bad ? 0 : (int)(b - a);
    q.prefix = p.prefix_of[s].x;
    const int64_t context = p.context[s], own = context - q.prefix;
    const bool bad_keys = q.prefix < 0 || own < 0 || own > p.max_context || context + q.rows > (p.table_stride << p.cache.page_shift);
    q.context = bad_keys ? -1 : (int)own;  // its rows are zeros
    if (bad_keys) q.prefix = 0;
    if (bad || bad_keys) report_status(p.status, STATUS_BAD_INDEX);
    q.news = q.rows;
    q.place.table = p.tables + (size_t)s * p.table_stride + (q.prefix >> p.cache.page_shift);
    q.place.first = 0;
    return q;
}
// The prefix of a sequence and whose pages hold it; -1 where its group cannot be, or cannot have its rows.
__device__ __forceinline__ int2 prefix_of_seq(const TreeParams& p, int s) {
    int lo = 0, hi = p.n_groups - 1;  // the last group that begins at s or before it
#pragma unroll 1
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (p.groups[mid] <= s) lo = mid;
        else hi = mid - 1;
    }
    const GroupSeqs of = group_seqs(p, lo);
    return make_int2(s < of.first || s >= of.stop || !rows_in_group(p, of, s) ? -1 : of.prefix, of.first);
}
__device__ __forceinline__ TreeSeq whole_seq(const TreeParams& p, int s) {
    TreeSeq q;
    const int64_t a = p.q_offsets ? p.q_offsets[s] : (int64_t)s * p.max_drafts, b = p.q_offsets ? p.q_offsets[s + 1] : a + p.max_drafts;
    const bool bad = a < 0 || b < a || b > p.tokens || b - a > p.max_drafts;
    q.row0 = bad ? 0 : (int)a;
    q.rows = bad ? 0 : (int)(b - a);
    const int64_t context = p.context[s];
    const int2 prefix = prefix_of_seq(p, s);
    const bool bad_keys = prefix.x < 0 || context < prefix.x || context - prefix.x > p.max_context || context + q.rows > (p.table_stride << p.cache.page_shift);
    q.context = bad_keys ? -1 : (int)context;  // its rows are zeros
    q.prefix = bad_keys ? 0 : prefix.x;
    q.first = bad_keys ? 0 : prefix.y;
    if (bad || bad_keys) report_status(p.status, STATUS_BAD_INDEX);
    q.news = q.rows;
    q.place.table = p.tables + (size_t)s * p.table_stride;
    q.place.first = 0;
    return q;
}
template <int KIND> __device__ __forceinline__ TreeSeq seq_of(const TreeParams& p, int s) {
    if (KIND == ATTEND_LISTS) return list_seq(p, s);
    if (KIND == ATTEND_PREFIX) return prefix_seq(p, s);
    if (KIND == ATTEND_OWN) return own_seq(p, s);
    if (KIND == ATTEND_WHOLE) return whole_seq(p, s);
    return tree_seq(p, s);
}
// Of a sequence, a segment or a cut unit: new keys, keys in all; context < 0: one that cannot be.
template <int KIND, class Seq> __device__ __forceinline__ int news_of(const Seq& q) {
    if constexpr (KIND == ATTEND_LISTS) return q.news;
    return KIND == ATTEND_PREFIX ? 0 : q.rows;
}
template <int KIND, class Seq> __device__ __forceinline__ int keys_of(const Seq& q) { return q.context < 0 ? 0 : q.context + news_of<KIND>(q); }

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}
__device__ __forceinline__ void load4(const bf16* p, float (&f)[4]) {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    f[0] = __uint_as_float(w.x << 16);
    f[1] = __uint_as_float(w.x & 0xFFFF0000u);
    f[2] = __uint_as_float(w.y << 16);
    f[3] = __uint_as_float(w.y & 0xFFFF0000u);
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// The kernels take a weight as 2^fma(s, scale, -(m scale)): for the largest score that is 2 to what rounding m scale has left, at most 2^-24 of it.  From 2^20 on
// that may matter, and rows go key by key.
__device__ __forceinline__ bool scores_too_large(float m, float scale) { return m > -INFINITY && fabsf(m * scale) >= 1048576.f; }

// One row by one warp, key by key: lane l has elements 4 l .. 4 l + 3.  softmax(s) v = sum_t 2^(s_t - m) v_t / sum_t 2^(s_t - m) with the
// running maximum m; keys that are not seen are not read, but all pages are looked at.
template <class Place, class Seen>
__device__ __noinline__ void attend_row(const CacheView& c, const Place& place, const bf16* q, bf16* out, int head, int keys, float scale_log2, int* status,
                                        Seen seen) {
    const int lane = threadIdx.x & 31;
    const bool mine = 4 * lane < c.dim;
    float qf[4] = {}, o[4] = {}, m = -INFINITY, l = 0.f;
    if (mine) load4(q + 4 * lane, qf);
    for (int t = 0; t < keys; t++) {
        const int64_t page = place.page_of(c, t);
        if (page < 0 || page >= c.pages) {
            if (lane == 0) report_status(status, STATUS_BAD_INDEX);
            continue;
        }
        if (!seen(t)) continue;
        const size_t at = c.at(page, head, t & ((1 << c.page_shift) - 1)) + 4 * lane;
        float k[4] = {}, v[4] = {};
        if (mine) {
            load4(c.keys + at, k);
            load4(c.values + at, v);
        }
        const float s = warp_sum(qf[0] * k[0] + qf[1] * k[1] + qf[2] * k[2] + qf[3] * k[3]) * scale_log2;
        const float top = fmaxf(m, s), ref = top == -INFINITY ? 0.f : top;
        const float keep = exp2f(m - ref), p = exp2f(s - ref);
        m = top;
        l = l * keep + p;
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] = o[e] * keep + p * v[e];
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    if (mine) *reinterpret_cast<uint2*>(out + 4 * lane) = make_uint2(pack_bf16(l == 0.f ? 0.f : o[0] * inv, l == 0.f ? 0.f : o[1] * inv), pack_bf16(l == 0.f ? 0.f : o[2] * inv, l == 0.f ? 0.f : o[3] * inv));
}

// What a row of a prompt or of a tree sees.
struct SeesUpTo {
    int last;
    __device__ __forceinline__ bool operator()(int t) const { return t <= last; }
};
struct SeesAncestors {
    int context;
    uint64_t word;
    __device__ __forceinline__ bool operator()(int t) const { return t < context || (t - context < TREE_MAX_DRAFTS && (word >> (t - context) & 1)); }
};
__device__ __forceinline__ uint64_t ancestors_of(const TreeParams& p, int row, int i) {
    return p.ancestors ? p.ancestors[row] : (uint64_t)-1 >> (63 - i);
}
// The new keys that token i of a sequence (row `row` of q) sees, of the `news` that there are.
template <int KIND> __device__ __forceinline__ uint64_t sees_of(const TreeParams& p, int row, int i, int news) {
    if (KIND == ATTEND_PREFIX) return 0;
    if (KIND == ATTEND_LISTS) return news == 0 ? 0 : (p.ancestors ? p.ancestors[row] : (uint64_t)-1) & ((uint64_t)-1 >> (64 - news));
    return ancestors_of(p, row, i) & ((uint64_t)-1 >> (64 - news));
}
// A row key by key: token i of unit or segment w, whose list or table has the number w.seq.
template <int KIND, class Unit>
__device__ __forceinline__ void attend_again(const TreeParams& p, const Unit& w, int i, int head, const bf16* q, bf16* out) {
    const uint64_t sees = sees_of<KIND>(p, w.row0 + i, i, news_of<KIND>(w));
    const int keys = keys_of<KIND>(w);
    if (KIND == ATTEND_OWN || KIND == ATTEND_WHOLE) {
        int2 prefix = make_int2(0, 0);
        if (w.context >= 0) prefix = KIND == ATTEND_OWN ? p.prefix_of[w.seq] : prefix_of_seq(p, w.seq);
        const int before = KIND == ATTEND_OWN ? prefix.x : 0;
        const SharedPlace place = {p.tables + (size_t)prefix.y * p.table_stride, prefix.x, p.tables + (size_t)w.seq * p.table_stride};
        attend_row(p.cache, place, q, out, head, before + keys, p.scale_log2, p.status, SeesAncestors{before + w.context, sees});
    } else {
        KeyPlace place;
        place.table = p.tables + (size_t)w.seq * p.table_stride;
        place.first = 0;
        attend_row(p.cache, place, q, out, head, keys, p.scale_log2, p.status, SeesAncestors{w.context, sees});
    }
}
#endif

CacheView cache_layer(const wf_kv_cache& cache, int layer);
int check_kv_cache(Context* c, const char* what, const wf_kv_cache* cache, int layer, bool packed_too);

// A launch that may begin before the kernel in front of it ends.
template <class... Params, class... Args>
inline int launch_clusters(Context* c, const char* what, void (*kernel)(Params...), dim3 grid, unsigned threads, unsigned cluster, size_t smem, cudaStream_t s, const Args&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
    if (e != cudaSuccess) return cuda_status(c, e, what);
    c->launches++;
    return WF_OK;
}

}  // namespace wf
