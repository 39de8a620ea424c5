// What the kernels of attention over a paged cache share: where keys lie, which of them a row sees, and a row computed key by key.
#pragma once
#include <cuda_bf16.h>

#include "wf_common.cuh"

namespace wf {

typedef __nv_bfloat16 bf16;

constexpr int ATTN_MAX_DIM = 128;
constexpr int TREE_MAX_DRAFTS = 64;  // a row's ancestors are one 64-bit word

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
#ifdef __CUDACC__
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
struct TreeSeq {
    int row0, rows, context;
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
    q.place.table = p.tables + (size_t)s * p.table_stride;
    q.place.first = 0;
    return q;
}

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
template <class Seen>
__device__ __noinline__ void attend_row(const CacheView& c, const KeyPlace& place, const bf16* q, bf16* out, int head, int keys, float scale_log2, int* status,
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
#endif

}  // namespace wf
