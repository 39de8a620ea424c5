// Which pages of a cache a new token reads: bounds of the keys of a page in 8 bits (wf_page_bounds), and the pages whose bounds promise the largest scores (wf_select_pages).
//
//   hi_d = ceil(max_t k[t, d] / 2^e), lo_d = floor(min_t k[t, d] / 2^e)      e the least for which they fit -127 .. 127
//   score of a page = 2^e max over the heads of the group of 2^f sum_d q_d (q_d > 0 ? hi_d : lo_d)     q rounded to -127 .. 127 times 2^f
// No key of the page has a larger product with that q.  The scales are powers of two, so a score is an integer below 2^21 times a power of two: exact, the same in
// whatever order it is summed, and ties are ties.  It is kept as a whole number of the same order: sign, exponent and 20 bits behind the leading one, which no scale can overflow.
#include <algorithm>
#include <atomic>
#include <climits>

#include "wf_attention.cuh"

namespace wf {

constexpr int LEAST_SCALE = -60;  // exponent: products of two scales are normal numbers

// The exponent of the scale for a largest magnitude of these bf16 bits (finite ones): 127 x 2^e >= size.  size = m 2^x, 127 = 1.984375 x 2^6, and of the
// significands of bf16 only the last is above that.
__device__ __forceinline__ int scale_exponent(uint32_t bits) {
    const int x = (int)(bits >> 7) - 127;
    return max(LEAST_SCALE, (bits & 0x7F) == 0x7F ? x - 5 : x - 6);
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // of a normal number

struct BoundsParams {
    CacheView cache;
    size_t layer_elements, layer_entries;  // keys, and (page, head) pairs, of a layer
    int8_t* codes;
    float* scales;
    const int* tables;
    int64_t table_stride;
    const int* first;
    const int* stop;
    int64_t seqs;
    unsigned units;  // pages of a sequence that may be touched, times heads
    int* status;
};

// A warp has one head of one page in one layer, contiguous in memory: a lane has 8 elements of a row, 32 / (dim / 8) rows go with one load, BOUNDS_DEPTH loads are in flight.  Every key of the
// pages is read once and nothing is left to wait for but HBM: 8192 tokens of 32 layers x 8 heads of 128 (537 MB and 9 of bounds) 75 us, as fast as a plain read; 16 decoded tokens, whose pages of
// up to 64 tokens are read again in all of 32 layers (39 MB), 6.3 us where the L2 has them, half of it a launch and the two loads before the first key (the table, the page), and 15 out of HBM: a launch, those
// loads and one round of warps, each of which waits for all of its keys once.
constexpr int BOUNDS_WARPS = 4, BOUNDS_DEPTH = 8;
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {  // NaN where one of them is
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__global__ void __launch_bounds__(BOUNDS_WARPS * 32) page_bounds_kernel(const __grid_constant__ BoundsParams p) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const unsigned unit = blockIdx.x * BOUNDS_WARPS + (threadIdx.x >> 5), heads = (unsigned)p.cache.kv_heads;
    if (unit >= p.units) return;
    const int lane = threadIdx.x & 31, pieces = p.cache.dim / 8, rows_at_once = 32 / pieces, active = rows_at_once * pieces;
    const int index = (int)(unit / heads), head = (int)(unit - index * heads), shift = p.cache.page_shift, page_tokens = 1 << shift;
    const bf16* const keys = p.cache.keys + (size_t)blockIdx.z * p.layer_elements;
    for (int64_t s = blockIdx.y; s < p.seqs; s += gridDim.y) {
        const int first = p.first[s], stop = p.stop[s];
        const bool bad = first < 0 || stop < first || (int64_t)stop > p.table_stride << shift ||
                         (first < stop && ((stop - 1) >> shift) - (first >> shift) >= (int)(p.units / heads));  // more than the call has room for
        if (bad) {
            if (lane == 0) report_status(p.status, STATUS_BAD_INDEX);
            continue;
        }
        const int j = (first >> shift) + index;
        const int64_t begin = (int64_t)j << shift;  // of a range whose call has room for more: behind 2^31, too
        if (first == stop || begin >= stop) continue;
        const int64_t page = p.tables[s * p.table_stride + j];
        if (page < 0 || page >= p.cache.pages) {
            if (lane == 0) report_status(p.status, STATUS_BAD_INDEX);
            continue;
        }
        const uint4* from = reinterpret_cast<const uint4*>(keys + p.cache.at(page, head, 0)) + lane;
        const int all = lane < active ? (int)min((int64_t)page_tokens, stop - begin) * pieces - lane : 0;  // this lane's pieces: 0, active, 2 active .. below it
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; e++) hi[e] = 0xFF80FF80u, lo[e] = 0x7F807F80u;  // -Inf, +Inf
#pragma unroll 1
        for (int i = 0; i < all; i += BOUNDS_DEPTH * active) {
            uint4 v[BOUNDS_DEPTH];
#pragma unroll
            for (int e = 0; e < BOUNDS_DEPTH; e++) v[e] = __ldcs(from + (i + e * active < all ? i + e * active : i));  // a piece again where there is no other
#pragma unroll
            for (int e = 0; e < BOUNDS_DEPTH; e++) {
                hi[0] = max2(hi[0], v[e].x), hi[1] = max2(hi[1], v[e].y), hi[2] = max2(hi[2], v[e].z), hi[3] = max2(hi[3], v[e].w);
                lo[0] = min2(lo[0], v[e].x), lo[1] = min2(lo[1], v[e].y), lo[2] = min2(lo[2], v[e].z), lo[3] = min2(lo[3], v[e].w);
            }
        }
        // over the lanes that have the same elements of other rows; every lane ends with some piece's
        const int piece = lane % pieces;
        uint32_t high[4], low[4], size = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            high[e] = __shfl_sync(0xFFFFFFFFu, hi[e], piece);
            low[e] = __shfl_sync(0xFFFFFFFFu, lo[e], piece);
#pragma unroll 1
            for (int r = 1; r < rows_at_once; r++) {
                high[e] = max2(high[e], __shfl_sync(0xFFFFFFFFu, hi[e], piece + r * pieces));
                low[e] = min2(low[e], __shfl_sync(0xFFFFFFFFu, lo[e], piece + r * pieces));
            }
            const uint32_t a = high[e] & 0x7FFF7FFFu, b = low[e] & 0x7FFF7FFFu;
            size = max(max(size, max(a & 0xFFFF, a >> 16)), max(b & 0xFFFF, b >> 16));
        }
        size = __reduce_max_sync(0xFFFFFFFFu, size);
        const bool fine = size < 0x7F80;  // neither Inf nor NaN
        const int exponent = scale_exponent(size);
        const float by = power_of_two(-(fine ? exponent : 0));
        uint32_t up[2] = {0, 0}, down[2] = {0, 0};
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int a = __float2int_ru(__uint_as_float(e & 1 ? high[e / 2] & 0xFFFF0000u : high[e / 2] << 16) * by);
            const int b = __float2int_rd(__uint_as_float(e & 1 ? low[e / 2] & 0xFFFF0000u : low[e / 2] << 16) * by);
            up[e / 4] |= (uint32_t)(a & 0xFF) << 8 * (e & 3);
            down[e / 4] |= (uint32_t)(b & 0xFF) << 8 * (e & 3);
        }
        const size_t entry = (size_t)blockIdx.z * p.layer_entries + (size_t)page * heads + head;
        int8_t* const to = p.codes + entry * 2 * p.cache.dim + piece * 8;
        if (lane < pieces) {
            *reinterpret_cast<uint2*>(to) = fine ? make_uint2(up[0], up[1]) : make_uint2(0, 0);
            *reinterpret_cast<uint2*>(to + p.cache.dim) = fine ? make_uint2(down[0], down[1]) : make_uint2(0, 0);
        }
        if (lane == 0) p.scales[entry] = fine ? power_of_two(exponent) : INFINITY;
    }
}

// ---------------------------------------------------------------- selection
struct SelectParams {
    const bf16* q;
    int64_t q_stride;
    const int8_t* codes;  // of the layer
    const float* scales;
    const int* q_offsets;
    const int* tables;
    int64_t table_stride;
    const int* context;
    int* pages_out;
    int2* lens_out;
    int64_t tokens, max_context, pages;
    int kv_heads, dim, group, page_shift, max_drafts, width, first, recent, tree;
    int room;            // pages whose scores a token and kv head may have
    uint32_t* scores;    // [tokens][kv_heads][room], where a kernel of its own makes them
    int score_pages;     // of a CTA there
    unsigned lists;      // sequences times max_drafts times heads
    uint32_t group_inverse;  // 2^32 / group, rounded up; 0 for a group of one
    int* status;
    __device__ __forceinline__ int token_of(int head) const { return group_inverse ? (int)__umulhi((uint32_t)head, group_inverse) : head; }  // head / group, below 64 x 128
};
constexpr int SELECT_MAX_GROUP = 128, SELECT_BINS = 256, SELECT_FEW = 256;  // SELECT_FEW: no more than a CTA has threads

__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// What a sequence's new tokens choose from.  rows: its new tokens; context < 0: a sequence that cannot be.
struct SelectSeq {
    int64_t row0;
    int rows, context;
    int last, tail, first, between;  // pages in all, from where on all are taken, how many at the start are, how many lie between
    int take;                        // how many of those between a list has room for (0 or more: the host sees to it that the ends fit)
    __device__ __forceinline__ bool scored() const { return take > 0 && take < between; }  // else a list has all of them, or none
};
__device__ __forceinline__ SelectSeq select_seq(const SelectParams& p, int s, bool report) {
    SelectSeq q;
    const int64_t a = p.q_offsets ? p.q_offsets[s] : (int64_t)s * p.max_drafts, b = p.q_offsets ? p.q_offsets[s + 1] : a + p.max_drafts;
    const bool no_rows = a < 0 || b < a || b > p.tokens || b - a > p.max_drafts;
    q.row0 = no_rows ? 0 : a;
    q.rows = no_rows ? 0 : (int)(b - a);
    q.context = p.context[s];
    const bool bad = q.context < 0 || (int64_t)q.context > p.max_context || (int64_t)q.context + q.rows > p.table_stride << p.page_shift;
    if ((no_rows || bad) && report) report_status(p.status, STATUS_BAD_INDEX);
    if (bad) q.context = -1;
    q.last = bad ? 0 : (q.context + q.rows + (1 << p.page_shift) - 1) >> p.page_shift;
    q.tail = bad ? 0 : max(0, q.context - p.recent) >> p.page_shift;
    q.first = min(p.first, q.tail);
    q.between = q.tail - q.first;
    q.take = min(q.between, p.width - q.first - (q.last - q.tail));
    return q;
}

// A head of q (4 elements a lane, zeros behind the last) in 8 bits: a word of those that are positive, one of those that are negative; the exponent of its scale, LEAST_SCALE to 122.
__device__ __forceinline__ int quantized(uint2 w, uint32_t& plus, uint32_t& minus) {
    const uint32_t x = w.x & 0x7FFF7FFFu, y = w.y & 0x7FFF7FFFu;
    const uint32_t size = __reduce_max_sync(0xFFFFFFFFu, max(max(x & 0xFFFF, x >> 16), max(y & 0xFFFF, y >> 16)));
    const bool fine = size < 0x7F80;  // a head with an Inf or a NaN has no preferences
    const int exponent = fine ? scale_exponent(size) : 0;
    const float by = power_of_two(-exponent);
    int v[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const uint32_t half = e & 2 ? w.y : w.x;
        v[e] = __float2int_rn(__uint_as_float(e & 1 ? half & 0xFFFF0000u : half << 16) * by);
    }
    const uint32_t bytes = fine ? __byte_perm(__byte_perm(v[0], v[1], 0x0040), __byte_perm(v[2], v[3], 0x0040), 0x5410) : 0;
    uint32_t negative;  // every byte's sign, eight times
    asm("prmt.b32 %0, %1, 0, 0xBA98;" : "=r"(negative) : "r"(bytes));
    plus = bytes & ~negative;
    minus = bytes & negative;
    return exponent;
}
// Puts a head's codes where the lanes of an MMA take them from: column `column` of [columns / 8][CHUNKS][32] vectors.
template <int CHUNKS> __device__ __forceinline__ void place_codes(uint4* codes, int column, int dim, uint32_t plus, uint32_t minus) {
    const int lane = threadIdx.x & 31;
    if (4 * lane >= dim) return;
    auto word = [](int k) { return k / 64 * 128 + (k & 63) / 16 * 4 + (k & 15) / 4; };  // of byte k of a page's codes
    uint32_t* const to = reinterpret_cast<uint32_t*>(codes) + column / 8 * (CHUNKS * 128) + (column & 7) * 16;
    to[word(4 * lane)] = plus;
    to[word(dim + 4 * lane)] = minus;
}
// A score of a head is a whole number below 2^21 times its scale, 2^-60 to 2^122; less 2^SCORE_BASE that is a number that a float holds exactly.
constexpr int SCORE_BASE = 16;
__device__ __forceinline__ float score_scale(int exponent) { return power_of_two(exponent - SCORE_BASE); }

// Sixteen pages, first + t * 16 .. of the table: lane g * 4 + quad has 16 codes of pages g and g + 8 in every chunk.  Which of them are called which k of the product does not matter, so
// long as q has the same.
template <int CHUNKS> struct PageTile {
    uint4 codes[2][CHUNKS];
    int scale[2];  // what a page's scale adds to a score; FIRST: the page comes before others, NOWHERE: it is not in the cache
    static constexpr int NOWHERE = INT_MIN + 1, FIRST = INT_MIN;
    // the pages' numbers; behind the last place page 0, whose score goes nowhere
    static __device__ __forceinline__ int2 find(const int* table, const SelectSeq& q, int t) {
        const int n = t * 16 + ((threadIdx.x & 31) >> 2);
        return make_int2(n < q.between ? table[q.first + n] : 0, n + 8 < q.between ? table[q.first + n + 8] : 0);
    }
    __device__ __forceinline__ void load(const SelectParams& p, int head, int2 pages) {
        const int quad = threadIdx.x & 3, bytes = 2 * p.dim;
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int page = e ? pages.y : pages.x;
            const bool real = page >= 0 && page < p.pages;
            const size_t entry = (size_t)(real ? page : 0) * p.kv_heads + head;
#pragma unroll
            for (int k = 0; k < CHUNKS; k++)
                codes[e][k] = 64 * k + 16 * quad < bytes ? *reinterpret_cast<const uint4*>(p.codes + entry * bytes + 64 * k + 16 * quad) : make_uint4(0, 0, 0, 0);
            const int exponent = (int)(__float_as_uint(p.scales[entry]) >> 23 & 0xFF);
            scale[e] = !real ? NOWHERE : exponent == 0xFF ? FIRST : (exponent - 127 - LEAST_SCALE + SCORE_BASE - LEAST_SCALE) << 20;
            if (!real) report_status(p.status, STATUS_BAD_INDEX);
        }
    }
    // eight columns: sums of pages g (0, 1) and g + 8 (2, 3) with columns 2 quad, 2 quad + 1
    __device__ __forceinline__ void multiply(const uint4* q, int (&sum)[4]) const {
        sum[0] = sum[1] = sum[2] = sum[3] = 0;
#pragma unroll
        for (int k = 0; k < CHUNKS; k++) {
            const uint4 b = q[k * 32 + (threadIdx.x & 31)];
            mma_s8(sum, codes[0][k].x, codes[1][k].x, codes[0][k].y, codes[1][k].y, b.x, b.y);
            mma_s8(sum, codes[0][k].z, codes[1][k].z, codes[0][k].w, codes[1][k].w, b.z, b.w);
        }
    }
    // The largest score over the heads, of page g + 8 e, with that page's scale, as an unsigned number of the same order: the exponent (127 less LEAST_SCALE twice and more, so that no scale
    // changes a sign) above 20 bits of significand, which such a number has.
    static __device__ __forceinline__ uint32_t key(float best, int scale) {
        const int size = (int)((__float_as_uint(best) & 0x7FFFFFFFu) >> 3) + scale;
        const uint32_t key = 0x80000000u + (uint32_t)(best == 0.f ? 0 : best < 0.f ? -size : size);
        return scale <= NOWHERE ? (scale == FIRST ? 0xFFFFFFFFu : 0u) : key;
    }
};

// Scores of all new tokens of a sequence, a CTA a kv head and p.score_pages pages, a warp 16 pages at a time: the codes of a page are read once for all of them.  Columns of the product are
// the heads of a token, padded to PADDED (0: to a multiple of eight above it), token by token; as many tokens at a time as SCORE_COLUMNS have room for.
// Bound by instructions: a tile of 16 pages by 8 columns has 4 to 8 products of the tensor cores and several times as many instructions on what comes out.  21 tokens of 24 / 8 heads of 96 over 8189 pages: 13 MB of
// codes (2 us), 12 to 17 us, of which 3 bring the 63 heads that a CTA has to 8 bits; in the kernel below, without tiles of several tokens, 97.
constexpr int SCORE_WARPS = 8, SCORE_PAGES = SCORE_WARPS * 16, SCORE_COLUMNS = 128, SCORE_HEADS = 4;  // heads asked for at a time
template <int CHUNKS, int PADDED> __global__ void __launch_bounds__(SCORE_WARPS * 32, 2) score_pages_kernel(const __grid_constant__ SelectParams p) {
    constexpr int TILES = PADDED == 0 ? 1 : 2;  // of eight columns at a time
    __shared__ uint4 q_codes[SCORE_COLUMNS / 8 * CHUNKS * 32];
    __shared__ float q_scale[SCORE_COLUMNS];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, quad = lane & 3;
    const int s = blockIdx.y / p.kv_heads, head = blockIdx.y - s * p.kv_heads, padded = PADDED ? PADDED : (p.group + 7) & ~7;
    const SelectSeq q = select_seq(p, s, false);
    const int begin = blockIdx.x * p.score_pages, end = min(begin + p.score_pages, q.between);
    // the kernel behind this one does not look at the scores where all pages are taken, or none
    if (q.rows == 0 || begin >= end || !q.scored()) return;
    const int* const table = p.tables + (size_t)s * p.table_stride;
    const int tokens_at_once = SCORE_COLUMNS / padded;
    const size_t apart = (size_t)p.kv_heads * p.room;  // scores of a token
    for (int token0 = 0; token0 < q.rows; token0 += tokens_at_once) {
        const int tokens = min(tokens_at_once, q.rows - token0), heads = tokens * p.group, column_tiles = (tokens * padded + 7) / 8;
        int t = begin / 16 + warp;
        const int last = (end - 1) / 16;
        // two tiles ahead of the one that is multiplied: the numbers of one's pages, the codes of the next one
        PageTile<CHUNKS> tile;
        int2 pages = PageTile<CHUNKS>::find(table, q, t);
        tile.load(p, head, pages);
        pages = PageTile<CHUNKS>::find(table, q, t + SCORE_WARPS);
        __syncthreads();
        for (int n = threadIdx.x; n < SCORE_COLUMNS / 8 * CHUNKS * 32; n += SCORE_WARPS * 32) q_codes[n] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        for (int n0 = warp; n0 < heads; n0 += SCORE_WARPS * SCORE_HEADS) {
            uint2 w[SCORE_HEADS];
#pragma unroll
            for (int e = 0; e < SCORE_HEADS; e++) {
                const int n = n0 + e * SCORE_WARPS, i = p.token_of(n), h = n - i * p.group;
                w[e] = make_uint2(0, 0);
                if (n < heads && 4 * lane < p.dim)
                    w[e] = *reinterpret_cast<const uint2*>(p.q + (q.row0 + token0 + i) * p.q_stride + (size_t)(head * p.group + h) * p.dim + 4 * lane);
            }
#pragma unroll
            for (int e = 0; e < SCORE_HEADS; e++) {
                const int n = n0 + e * SCORE_WARPS, i = p.token_of(n), h = n - i * p.group;
                if (n >= heads) break;
                uint32_t plus, minus;
                const int scale = quantized(w[e], plus, minus);
                place_codes<CHUNKS>(q_codes, i * padded + h, p.dim, plus, minus);
                if (lane == 0) q_scale[i * padded + h] = score_scale(scale);
            }
        }
        __syncthreads();
#pragma unroll 1
        for (; t <= last; t += SCORE_WARPS) {
            PageTile<CHUNKS> next;
            next.load(p, head, pages);
            pages = PageTile<CHUNKS>::find(table, q, t + 2 * SCORE_WARPS);
            float best[2] = {-INFINITY, -INFINITY};
            uint32_t* to = p.scores + ((size_t)(q.row0 + token0) * p.kv_heads + head) * p.room + t * 16 + g;  // page g, of the token that the columns have come to
            const bool inside[2] = {t * 16 + g < q.between, t * 16 + g + 8 < q.between};
            int left = tokens, h0 = 0;  // tokens from there on, heads of the first one that are done (PADDED 0)
            // (PADDED 2, 4, 8) whether this lane's columns are heads, which of the tokens of eight columns it stores (none: TREE_MAX_DRAFTS), of which page
            const bool one = (2 * quad & (PADDED - 1)) < p.group, two = (2 * quad & (PADDED - 1)) + 1 < p.group;
            const int mine = PADDED == 8 && quad > 1 ? TREE_MAX_DRAFTS : PADDED == 4 ? quad >> 1 : PADDED == 2 ? quad : 0;
            const bool mine_inside = quad & 1 ? inside[1] : inside[0];
            if (PADDED > 1) to += PADDED == 2 ? quad * apart : PADDED == 4 ? (quad >> 1) * apart + 8 * (quad & 1) : 8 * (quad & 1);
#pragma unroll 1
            for (int n0 = 0; n0 < column_tiles; n0 += TILES) {  // (there are codes, if only zeros, for SCORE_COLUMNS)
                int sum[TILES][4];
#pragma unroll
                for (int e = 0; e < TILES; e++) tile.multiply(q_codes + (n0 + e) * CHUNKS * 32, sum[e]);
#pragma unroll
                for (int i = 0; i < TILES; i++) {
                    const float2 scales = *reinterpret_cast<const float2*>(q_scale + (n0 + i) * 8 + 2 * quad);
                    float v[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) v[e] = (float)sum[i][e] * (e & 1 ? scales.y : scales.x);
                    if constexpr (PADDED == 1) {
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (2 * quad + (e & 1) < left && inside[e >> 1]) to[(2 * quad + (e & 1)) * apart + 8 * (e >> 1)] = tile.key(v[e], tile.scale[e >> 1]);
                        to += 8 * apart, left -= 8;
                    } else if constexpr (PADDED > 1) {
                        // the largest over the columns of a token that this lane has and its neighbours have; 8 / PADDED tokens
                        float top[2];
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            top[e] = fmaxf(two ? v[2 * e + 1] : -INFINITY, one ? v[2 * e] : -INFINITY);
                            if (PADDED >= 4) top[e] = fmaxf(top[e], __shfl_xor_sync(0xFFFFFFFFu, top[e], 1));
                            if (PADDED >= 8) top[e] = fmaxf(top[e], __shfl_xor_sync(0xFFFFFFFFu, top[e], 2));
                        }
                        if (PADDED == 2) {
#pragma unroll
                            for (int e = 0; e < 2; e++)
                                if (quad < left && inside[e]) to[8 * e] = tile.key(top[e], tile.scale[e]);
                        } else if (mine < left && mine_inside) {  // of two lanes that know both, one has page g and the other page g + 8
                            *to = tile.key(quad & 1 ? top[1] : top[0], quad & 1 ? tile.scale[1] : tile.scale[0]);
                        }
                        to += 8 / PADDED * apart, left -= 8 / PADDED;
                    } else {
                        const int h = h0 + 2 * quad;
#pragma unroll
                        for (int e = 0; e < 2; e++) best[e] = fmaxf(best[e], h + 1 < p.group ? fmaxf(v[2 * e], v[2 * e + 1]) : h < p.group ? v[2 * e] : -INFINITY);
                        if ((h0 += 8) < padded) continue;
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            best[e] = fmaxf(best[e], __shfl_xor_sync(0xFFFFFFFFu, best[e], 1));
                            best[e] = fmaxf(best[e], __shfl_xor_sync(0xFFFFFFFFu, best[e], 2));
                            if (quad == 0 && left > 0 && inside[e]) to[8 * e] = tile.key(best[e], tile.scale[e]);
                            best[e] = -INFINITY;
                        }
                        to += apart, left--, h0 = 0;
                    }
                }
            }
            tile = next;
        }
    }
}

// Scores that the kernel before this one left (ld_once says why not by a plain load).
__device__ __forceinline__ uint4 load_scores(const uint32_t* from) {
    uint4 v;
    asm volatile("ld.global.cs.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(from));
    return v;
}

// What a list has in any case, by `lanes` threads of which this is number `lane`: the places that the scores do not decide, the lengths.
__device__ __forceinline__ void write_ends(const SelectParams& p, const SelectSeq& q, int64_t line, int i, const int* table, int* list, int lane, int lanes) {
    const int first = q.first, take = q.take, count = first + q.last - q.tail + take;
    for (int n = lane; n < p.width - take; n += lanes) {
        const int at = n < first ? n : n + take, page = at < first ? at : q.tail + at - first - take;
        list[at] = at < count ? table[page] : -1;
    }
    if (lane == 0) {
        const int held = q.context < 0 ? 0 : q.context - ((q.between - take) << p.page_shift);
        p.lens_out[line] = make_int2(held, q.context < 0 ? 0 : held + (p.tree ? q.rows : i + 1));
    }
}

// The pages of a new token and kv head by a warp, where their scores lie in memory and are few, or none is left out: a lane keeps RUN of them.  The largest are those from T on, the largest number for which there are
// enough of them, found bit by bit; no barrier and no shared memory.  (4152 lists of some 70 pages, their scores included: 17 us; by CTAs of eight warps, sixteen rounds of them, 36.)
constexpr int FEW_WARPS = 4;
template <int RUN> __global__ void __launch_bounds__(FEW_WARPS * 32) select_few_kernel(const __grid_constant__ SelectParams p) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const unsigned unit = blockIdx.x * FEW_WARPS + (threadIdx.x >> 5), per_seq = (unsigned)p.max_drafts * p.kv_heads, s = unit / per_seq, of_seq = unit - s * per_seq;
    if (unit >= p.lists) return;
    const int lane = threadIdx.x & 31, i = (int)(of_seq / p.kv_heads), head = (int)(of_seq - i * p.kv_heads);
    const SelectSeq q = select_seq(p, (int)s, lane == 0 && of_seq == 0);
    if (i >= q.rows) return;
    const int64_t line = (q.row0 + i) * p.kv_heads + head;
    const int* const table = p.tables + (size_t)s * p.table_stride;
    int* const list = p.pages_out + (size_t)line * p.width;
    const int take = q.take;
    const int from = lane * RUN, valid = max(0, min(RUN, q.between - from));
    uint32_t d[RUN];
    if (q.scored()) {
        const uint32_t* const scores = p.scores + (size_t)line * p.room;
#pragma unroll
        for (int e = 0; e < RUN; e += 4) {
            const uint4 v = e < valid ? load_scores(scores + from + e) : make_uint4(0, 0, 0, 0);
            d[e] = v.x, d[e + 1] = v.y, d[e + 2] = v.z, d[e + 3] = v.w;
        }
    }
    write_ends(p, q, line, i, table, list, lane, 32);
    if (!q.scored()) {
        for (int n = lane; n < take; n += 32) list[q.first + n] = table[q.first + n];
        return;
    }
    uint32_t low = 0xFFFFFFFFu, high = 0;
#pragma unroll
    for (int e = 0; e < RUN; e++)
        if (e < valid) low = min(low, d[e]), high = max(high, d[e]);
    low = __reduce_min_sync(0xFFFFFFFFu, low);
    high = __reduce_max_sync(0xFFFFFFFFu, high);
#pragma unroll
    for (int e = 0; e < RUN; e++) d[e] = e < valid ? d[e] - low : 0;  // (what is above 0 is a page's)
    uint32_t border = 0;
    for (int bit = 31 - __clz(high - low); bit >= 0; bit--) {
        const uint32_t next = border | 1u << bit;
        int enough = 0;
#pragma unroll
        for (int e = 0; e < RUN; e++) enough += d[e] >= next;
        enough = __reduce_add_sync(0xFFFFFFFFu, enough);
        if (enough >= take) border = next;
        if (enough == take) break;
    }
    // Those above the border, and of those on it the first ones: how many of each there are up to this lane, in one word.
    uint32_t both = 0;
#pragma unroll
    for (int e = 0; e < RUN; e++) both += d[e] > border ? 1u : e < valid && d[e] == border ? 1u << 16 : 0;
    uint32_t up_to = both;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, up_to, o);
        if (lane >= o) up_to += v;
    }
    const int need = take - (int)(__shfl_sync(0xFFFFFFFFu, up_to, 31) & 0xFFFF);
    int above = (int)((up_to - both) & 0xFFFF), like = (int)((up_to - both) >> 16);
#pragma unroll
    for (int e = 0; e < RUN; e++) {
        const bool on = e < valid && d[e] == border;
        if (d[e] > border || (on && like < need)) list[q.first + above + min(like, need)] = table[q.first + from + e];
        above += d[e] > border;
        like += on;
    }
}

// A cluster has one new token and kv head.  Its CTAs score a part of the pages each, 16 pages by the heads of the group a warp at a time (mma.sync on the codes: [q+ | q-] . [hi | lo],
// the positive elements of q in the one half and the negative ones in the other), and leave the scores in the first CTA's shared memory, which takes the largest.  SCORED: the scores lie in
// memory.  CHUNKS of 64 codes of a page (hi and lo together).  RUN: scores of a thread, which it keeps in registers; 0: as many as there are, read again each time.
// Bound by latencies: launch, context, table, codes, and some six barriers of the selection.  One token of 8 kv heads over 497 pages 6.4 us, of 48 sequences with up to 250 pages 9.7 (13 MB, 1.4 TB/s).
// The largest are found by two or three histograms of eight bits instead of a sort: what is left in a bin of the second, at most 256 scores, is ranked by comparing all with all.
template <int CHUNKS, int WARPS, int RUN, bool SCORED> __global__ void __launch_bounds__(WARPS * 32, WARPS <= 8 && RUN != 2 ? 2 : WARPS <= 8 ? 3 : SCORED ? 2 : 1) select_pages_kernel(const __grid_constant__ SelectParams p) {
    constexpr int THREADS = WARPS * 32;
    constexpr bool AHEAD = RUN != 2;  // (few pages: a warp has one or two tiles of them, and registers are worth more)
    constexpr bool IN_MEMORY = SCORED && RUN > 0;  // registers take the scores from there
    static_assert(!SCORED || RUN != 2, "few scores in memory: select_few_kernel");
    extern __shared__ uint4 dynamic[];  // scores [room], as unsigned numbers of the same order; codes of the heads; exponents of their scales
    uint32_t* const keys = reinterpret_cast<uint32_t*>(dynamic);
    uint4* const q_codes = dynamic + p.room / 4;
    float* const q_scale = reinterpret_cast<float*>(q_codes + (p.group + 7) / 8 * CHUNKS * 32);
    __shared__ uint32_t bins[SELECT_BINS], warp_low[WARPS], warp_high[WARPS], found[3];
    __shared__ unsigned long long totals[WARPS];
    __shared__ uint32_t few[SELECT_FEW], few_count;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    uint32_t rank, ranks;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
    cluster_arrive();  // the first CTA is there before anything is sent to it
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, quad = lane & 3;
    const unsigned unit = blockIdx.x / ranks, per_seq = (unsigned)p.max_drafts * p.kv_heads, s = unit / per_seq, of_seq = unit - s * per_seq;
    const int i = (int)(of_seq / p.kv_heads), head = (int)(of_seq - i * p.kv_heads);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const SelectSeq q = select_seq(p, (int)s, tid == 0 && rank == 0 && of_seq == 0);
    if (i >= q.rows) {  // all of the cluster
        cluster_wait();
        return;
    }
    const int64_t row = q.row0 + i;
    const int* const table = p.tables + (size_t)s * p.table_stride;
    const int first = q.first, between = q.between, take = q.take;
    int* const list = p.pages_out + ((size_t)row * p.kv_heads + head) * p.width;
    if (rank == ranks - 1) write_ends(p, q, row * p.kv_heads + head, i, table, list, tid, THREADS);
    if (!q.scored()) {
        if (rank == 0)
            for (int n = tid; n < take; n += THREADS) list[first + n] = table[first + n];
        cluster_wait();
        return;
    }

    const uint32_t* const scores = SCORED ? p.scores + ((size_t)row * p.kv_heads + head) * p.room : nullptr;
    if (SCORED) {
        cluster_wait();
        if (!IN_MEMORY) {
            for (int n = 4 * tid; n < between; n += 4 * THREADS) *reinterpret_cast<uint4*>(keys + n) = load_scores(scores + n);
            __syncthreads();
        }
    } else {
        // This warp's first pages are on their way while the heads of the group are brought to 8 bits, a warp a head.
        const int tiles = (between + 15) / 16, mine0 = (int)((int64_t)tiles * rank / ranks), mine1 = (int)((int64_t)tiles * (rank + 1) / ranks);
        PageTile<CHUNKS> tile;
        int2 pages = PageTile<CHUNKS>::find(table, q, min(mine0 + warp, tiles - 1));
        tile.load(p, head, pages);
        if (AHEAD) pages = PageTile<CHUNKS>::find(table, q, mine0 + warp + WARPS);
        const int column_tiles = (p.group + 7) / 8;
        for (int n = tid; n < column_tiles * CHUNKS * 32; n += THREADS) q_codes[n] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        for (int h = warp; h < p.group; h += WARPS) {
            const bf16* from = p.q + row * p.q_stride + (size_t)(head * p.group + h) * p.dim + 4 * lane;
            uint32_t plus, minus;
            const int scale = quantized(4 * lane < p.dim ? *reinterpret_cast<const uint2*>(from) : make_uint2(0, 0), plus, minus);
            place_codes<CHUNKS>(q_codes, h, p.dim, plus, minus);
            if (lane == 0) q_scale[h] = score_scale(scale);
        }
        __syncthreads();
        if (ranks > 1) cluster_wait();

        const uint32_t to = map_to_rank((uint32_t)__cvta_generic_to_shared(keys), 0);
#pragma unroll 1
        for (int t = mine0 + warp; t < mine1; t += WARPS) {
            PageTile<CHUNKS> next;
            if (AHEAD) {
                next.load(p, head, pages);
                pages = PageTile<CHUNKS>::find(table, q, t + 2 * WARPS);
            }
            float best[2] = {-INFINITY, -INFINITY};
            for (int n = 0; n < column_tiles; n++) {
                int sum[4];
                tile.multiply(q_codes + n * CHUNKS * 32, sum);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int h = n * 8 + 2 * quad + (e & 1);
                    if (h < p.group) best[e >> 1] = fmaxf(best[e >> 1], (float)sum[e] * q_scale[h]);
                }
            }
#pragma unroll
            for (int e = 0; e < 2; e++) {
                best[e] = fmaxf(best[e], __shfl_xor_sync(0xFFFFFFFFu, best[e], 1));
                best[e] = fmaxf(best[e], __shfl_xor_sync(0xFFFFFFFFu, best[e], 2));
                const int n = t * 16 + g + 8 * e;
                if (quad == 0 && n < between) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to + 4 * (uint32_t)n), "r"(tile.key(best[e], tile.scale[e])) : "memory");
            }
            if (AHEAD) tile = next;
            else if (t + WARPS < mine1) tile.load(p, head, PageTile<CHUNKS>::find(table, q, t + WARPS));
        }
        if (ranks > 1) {
            cluster_arrive();
            cluster_wait();
            if (rank) return;  // nothing is sent to the others
        } else {
            cluster_wait();  // that of the start
            __syncthreads();
        }
    }

    // A thread has a run of pages: `run` of them from `from` on (of odd length where they lie in shared memory, for the sake of the banks).
    const int run = RUN ? RUN : ((between + THREADS - 1) / THREADS) | 1, from = min(tid * run, between), valid = min(run, between - from);
    uint32_t kept[RUN ? RUN : 1];
    if constexpr (RUN > 0) {
#pragma unroll
        for (int e = 0; e < RUN; e += RUN < 4 ? 2 : 4) {
            if constexpr (RUN < 4) {
                const uint2 v = e < valid ? *reinterpret_cast<const uint2*>(keys + from + e) : make_uint2(0, 0);
                kept[e] = v.x, kept[e + 1] = v.y;
            } else {
                const uint4 v = e < valid ? IN_MEMORY ? load_scores(scores + from + e) : *reinterpret_cast<const uint4*>(keys + from + e) : make_uint4(0, 0, 0, 0);
                kept[e] = v.x, kept[e + 1] = v.y, kept[e + 2] = v.z, kept[e + 3] = v.w;
            }
        }
    }
    // f(score) for each of them
    auto each = [&](auto f) {
        if constexpr (RUN > 0) {
#pragma unroll
            for (int e = 0; e < RUN; e++)
                if (e < valid) f(e, kept[e]);
        } else {
            for (int e = 0; e < valid; e++) f(e, keys[from + e]);
        }
    };
    uint32_t low = 0xFFFFFFFFu, high = 0;
    each([&](int, uint32_t key) { low = min(low, key), high = max(high, key); });

    // The largest `take` of them: the key of the last one, by eight bits at a time of what is above the smallest key, and how many of that key.
    low = __reduce_min_sync(0xFFFFFFFFu, low);
    high = __reduce_max_sync(0xFFFFFFFFu, high);
    if (lane == 0) warp_low[warp] = low, warp_high[warp] = high;
    if (tid < SELECT_BINS) bins[tid] = 0;
    if (tid == 0) few_count = 0;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; w++) low = min(low, warp_low[w]), high = max(high, warp_high[w]);
    int bits = 32 - __clz(high - low);           // of the differences that are still open
    uint32_t prefix = 0, need = (uint32_t)take;  // what is decided of the difference; how many are still to be taken of those that begin so
    while (bits > 0) {
        const int less = max(0, bits - 8);
        each([&](int, uint32_t key) {
            const uint32_t d = key - low;
            if (bits == 32 || d >> bits == prefix >> bits) atomicAdd(&bins[d >> less & (SELECT_BINS - 1)], 1u);
        });
        __syncthreads();
        if (warp == 0) {  // the bin of the last one, from above: a lane has eight bins
            uint32_t mine[8], sum = 0;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                uint32_t& bin = bins[SELECT_BINS - 1 - (lane * 8 + e)];
                sum += mine[e] = bin;
                bin = 0;
            }
            uint32_t before = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, before, o);
                if (lane >= o) before += v;
            }
            before -= sum;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                if (before < need && before + mine[e] >= need) found[0] = (uint32_t)(SELECT_BINS - 1 - (lane * 8 + e)), found[1] = need - before, found[2] = mine[e];
                before += mine[e];
            }
        }
        __syncthreads();
        prefix |= found[0] << less;
        need = found[1];
        bits = less;
        if (found[2] == need) break;  // all that begin so
        if (found[2] <= SELECT_FEW && bits > 0) {  // few begin so: the key of the last one is that of which fewer than `need` are larger and `need` or more are not smaller
            each([&](int, uint32_t key) {
                const uint32_t d = key - low;
                if (d >> bits == prefix >> bits) few[atomicAdd(&few_count, 1u)] = d;
            });
            __syncthreads();
            const uint32_t candidates = few_count, d = tid < candidates ? few[tid] : 0;
            uint32_t larger = 0, same = 0;
            if (tid < candidates)
                for (uint32_t j = 0; j < candidates; j++) larger += few[j] > d, same += few[j] == d;
            if (tid < candidates && larger < need && larger + same >= need) found[0] = d, found[1] = need - larger;  // (all that have it write the same)
            __syncthreads();
            prefix = found[0], need = found[1], bits = 0;
            break;
        }
        __syncthreads();
    }
    // Those that begin above the prefix, and of those that begin like it the first `need`.
    const uint32_t border = prefix >> bits;
    uint32_t mine = 0, alike = 0;  // of the run: above the border, on it
    each([&](int, uint32_t key) {
        const uint32_t d = (key - low) >> bits;
        mine += d > border;
        alike += d == border;
    });
    const unsigned long long both = (unsigned long long)alike << 32 | mine;
    unsigned long long sum = both;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long v = __shfl_up_sync(0xFFFFFFFFu, sum, o);
        if (lane >= o) sum += v;
    }
    if (lane == 31) totals[warp] = sum;
    __syncthreads();
    sum -= both;
    for (int w = 0; w < warp; w++) sum += totals[w];
    uint32_t above = (uint32_t)sum, like = (uint32_t)(sum >> 32);
    each([&](int e, uint32_t key) {
        const uint32_t d = (key - low) >> bits;
        if (d > border || (d == border && like < need)) {
            const uint32_t at = above + min(like, need);
            if (RUN > 0) keys[at] = (uint32_t)(from + e);  // the scores that lay there are in registers
            else list[first + at] = table[first + from + e];
        }
        above += d > border;
        like += d == border;
    });
    if (RUN > 0) {
        __syncthreads();
        for (int n = tid; n < take; n += THREADS) list[first + n] = table[first + keys[n]];
    }
}

}  // namespace wf

using namespace wf;

#define SELECT_ENTER(ctxh)                                                 \
    Context* c = get_context(ctxh);                                        \
    if (!c) return WF_ERR_INVALID_HANDLE;                                  \
    ScopedLock _lk(c);                                                     \
    if (!_lk.ok) return WF_ERR_BUSY;                                       \
    WF_CUDA(c, cudaSetDevice(c->device));                                  \
    cudaStream_t s = resolve_stream(c, stream)

template <int CHUNKS, int WARPS, int RUN, bool SCORED> static int launch_selection(Context* c, const SelectParams& p, int64_t units, unsigned cluster, cudaStream_t s) {
    static std::atomic<uint64_t> ready{0};  // devices whose attribute is set
    constexpr size_t HEADS = SCORED ? 0 : CHUNKS * 32 * sizeof(uint4) + 8 * sizeof(int);  // bytes for eight heads
    const size_t smem = (size_t)p.room * 4 + (p.group + 7) / 8 * HEADS;
    if (!(ready.load() >> (c->device & 63) & 1)) {
        WF_CUDA(c, cudaFuncSetAttribute(select_pages_kernel<CHUNKS, WARPS, RUN, SCORED>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(WF_SELECT_MAX_PAGES * 4 + SELECT_MAX_GROUP / 8 * HEADS)));
        ready.fetch_or(1ull << (c->device & 63));
    }
    return launch_clusters(c, "select_pages", select_pages_kernel<CHUNKS, WARPS, RUN, SCORED>, dim3((unsigned)(units * cluster)), WARPS * 32, cluster, smem, s, p);
}
template <int CHUNKS> static int launch_selections(Context* c, SelectParams p, int seqs, cudaStream_t s) {
    p.lists = (unsigned)((int64_t)seqs * p.max_drafts * p.kv_heads);
    const int64_t units = p.lists, bytes = p.tokens * p.kv_heads * p.room * 4;
    const dim3 few((unsigned)((units + FEW_WARPS - 1) / FEW_WARPS));
    // Lists that have room for all pages of the longest context: nothing is scored.  (24 tokens x 16 heads over 7 to 16 pages 3.3 us, by CTAs 4.9.)
    if (p.room <= 512 && (std::min(p.max_context + p.max_drafts, p.table_stride << p.page_shift) + (1 << p.page_shift) - 1) >> p.page_shift <= p.width)
        return launch_clusters(c, "select_pages", select_few_kernel<4>, few, FEW_WARPS * 32, 1, 0, s, p);
    // Several new tokens of a sequence read the same codes.  In one kernel each token's cluster reads them, in two a CTA scores pages for all of them: that begins later, and by the more, the more heads each
    // of its CTAs brings to 8 bits.  Microseconds by one / by two, tokens x sequences with pages of 16: 32 / 8 heads (20 to 84 heads of a CTA), 64 pages, 5 x 4, 5 x 16, 21 x 4, 21 x 16 (160 to 2688 lists)
    // 7.0 / 8.5, 12.3 / 9.5, 12.3 / 11.7, 35.6 / 15.2; 500 pages 13.2 / 11.5, 23.6 / 16.9, 24.4 / 20.8, 77 / 29; 16 / 2 heads (168), 21 x 4, 21 x 16, 21 x 48: 7.1 / 17.8, 12.6 / 17.8, 28.4 / 18.6.  More pages: 32 / 8
    // heads, 1000, 2 x 1, 5 x 1, 21 x 1: 9.8 / 10.7, 13.4 / 12.1, 18.3 / 15.3; 4000: 20.7 / 16.1, 22.3 / 15.7, 60 / 22.6; 16 / 2 heads, 21 x 1, 21 x 4 of 4000: 22.2 / 28.3, 60 / 32.
    const int64_t heads = (int64_t)p.max_drafts * p.group, lists = p.tokens * p.kv_heads;
    const bool scored = p.room <= 512 ? lists >= 200 + 11 * heads / 2 : lists * p.room >= 20480 + 1024 * heads;
    if (p.max_drafts > 1 && scored && bytes <= ATTN_CALL_BYTES && (int64_t)seqs * p.kv_heads <= 65535) {
        GemvScratch& scratch = c->gemv_scratch[s];
        if (bytes > scratch.attn_bytes) {
            const int rc = refuse_allocation_while_recording(c, s, "the scores of select_pages");
            if (rc != WF_OK) return rc;
            scratch.d_attn.reset();
            scratch.attn_bytes = 0;
            WF_CUDA(c, make_shared_device(c, scratch.d_attn, (size_t)bytes));
            scratch.attn_bytes = bytes;
        }
        p.scores = reinterpret_cast<uint32_t*>(scratch.d_attn.get());
        const int64_t lines = (int64_t)seqs * p.kv_heads, pieces = (p.room + SCORE_PAGES - 1) / SCORE_PAGES;
        // two CTAs on every SM at once: what a CTA does before its first page, the queries, is done by as few as that
        const int64_t each = (lines * pieces + 2 * c->sm_count - 1) / (2 * c->sm_count);  // pieces of a CTA
        p.score_pages = (int)(each * SCORE_PAGES);
        const dim3 grid((unsigned)((pieces + each - 1) / each), (unsigned)lines);
        auto score = [&](auto kernel) { return launch_clusters(c, "select_pages", kernel, grid, SCORE_WARPS * 32, 1, 0, s, p); };
        const int rc = p.group == 1   ? score(score_pages_kernel<CHUNKS, 1>)
                       : p.group == 2 ? score(score_pages_kernel<CHUNKS, 2>)
                       : p.group <= 4 ? score(score_pages_kernel<CHUNKS, 4>)
                       : p.group <= 8 ? score(score_pages_kernel<CHUNKS, 8>)
                                      : score(score_pages_kernel<CHUNKS, 0>);
        if (rc != WF_OK) return rc;
        if (p.room <= 128) return launch_clusters(c, "select_pages", select_few_kernel<4>, few, FEW_WARPS * 32, 1, 0, s, p);
        if (p.room <= 512) return launch_clusters(c, "select_pages", select_few_kernel<16>, few, FEW_WARPS * 32, 1, 0, s, p);
        if (p.room <= 2048) return launch_selection<CHUNKS, 8, 8, true>(c, p, units, 1, s);
        return p.room <= 8192 ? launch_selection<CHUNKS, 16, 16, true>(c, p, units, 1, s) : launch_selection<CHUNKS, 16, 0, true>(c, p, units, 1, s);
    }
    // As many CTAs a token and head as leave every CTA an SM and eight tiles of pages: one token of 8 heads at 250, 500, 1000, 8125 pages in clusters of 1 / 2 / 4 / 8: 7.2 / 7.0 / 6.7 / 6.7,
    // 10.0 / 7.9 / 6.7 / 6.3, 14.0 / 11.3 / 9.6 / 9.0, 52 / 33 / 22 / 17 us; of 48 x 8 heads at 250 9.7 / 14.6 / 20 / 36.
    unsigned cluster = 1;
    while (cluster < 8 && units * cluster * 2 <= c->sm_count && p.room >= 128 * (int)cluster) cluster *= 2;
    if (p.room <= 512) return launch_selection<CHUNKS, 8, 2, false>(c, p, units, cluster, s);
    if (p.room <= 2048) return launch_selection<CHUNKS, 8, 8, false>(c, p, units, cluster, s);
    return p.room <= 8192 ? launch_selection<CHUNKS, 16, 16, false>(c, p, units, cluster, s) : launch_selection<CHUNKS, 16, 0, false>(c, p, units, cluster, s);
}

extern "C" {

int wf_page_bounds(int64_t ctx, const wf_kv_cache* cache, int64_t codes_dev, int64_t scales_dev, int64_t tables_dev, int64_t table_stride, int64_t first_dev, int64_t stop_dev,
                   int64_t seqs, int64_t max_tokens, int64_t stream) {
    SELECT_ENTER(ctx);
    const char* what = "page_bounds";
    const int rc = check_kv_cache(c, what, cache, 0, false);
    if (rc != WF_OK) return rc;
    if (!codes_dev || !scales_dev || codes_dev & 15 || scales_dev & 3)
        return set_error(c, WF_ERR_INVALID_ARGUMENT, "%s: codes is a 16-byte aligned device array, scales a 4-byte aligned one", what);
    if (seqs < 0 || seqs > (1LL << 31) - 1 || table_stride < 1 || table_stride > (1LL << 31) / cache->page_tokens - 1 || max_tokens < 0 ||
        max_tokens > (1LL << 31) - 1024)
        return set_error(c, WF_ERR_SHAPE, "%s: seqs=%lld table_stride=%lld max_tokens=%lld", what, (long long)seqs, (long long)table_stride, (long long)max_tokens);
    if (seqs == 0 || max_tokens == 0) return WF_OK;
    if (!tables_dev || !first_dev || !stop_dev || (tables_dev | first_dev | stop_dev) & 3)
        return set_error(c, WF_ERR_INVALID_ARGUMENT, "%s: tables, first and stop are 4-byte aligned device arrays", what);
    BoundsParams p{};
    p.cache = cache_layer(*cache, 0);
    p.layer_entries = (size_t)cache->pages * cache->kv_heads;
    p.layer_elements = p.layer_entries * cache->page_tokens * cache->head_dim;
    p.codes = reinterpret_cast<int8_t*>(codes_dev);
    p.scales = reinterpret_cast<float*>(scales_dev);
    p.tables = reinterpret_cast<const int*>(tables_dev);
    p.table_stride = table_stride;
    p.first = reinterpret_cast<const int*>(first_dev);
    p.stop = reinterpret_cast<const int*>(stop_dev);
    p.seqs = seqs;
    p.status = c->d_status;
    const int64_t touched = std::min(table_stride, (max_tokens + cache->page_tokens - 2) / cache->page_tokens + 1);  // pages of max_tokens tokens, wherever they begin
    const int64_t units = touched * cache->kv_heads;
    if (units > (1LL << 31) - 1) return set_error(c, WF_ERR_TOO_LARGE, "%s: %lld tokens of %d heads", what, (long long)max_tokens, cache->kv_heads);
    p.units = (unsigned)units;
    return launch_clusters(c, what, page_bounds_kernel, dim3((unsigned)((units + BOUNDS_WARPS - 1) / BOUNDS_WARPS), (unsigned)std::min<int64_t>(seqs, 65535), (unsigned)cache->layers),
                         BOUNDS_WARPS * 32, 1, 0, s, p);
}

int wf_select_pages(int64_t ctx, const wf_select_pages_args* a, int64_t stream) {
    SELECT_ENTER(ctx);
    const char* what = "select_pages";
    if (!a) return set_error(c, WF_ERR_INVALID_ARGUMENT, "%s: null arguments", what);
    if (a->tokens == 0 || a->seqs == 0) return WF_OK;
    if (!a->q_dev || !a->codes_dev || !a->scales_dev || (a->q_dev | a->codes_dev) & 15 || a->scales_dev & 3)
        return set_error(c, WF_ERR_INVALID_ARGUMENT, "%s: q and codes must be 16-byte aligned device addresses, scales a 4-byte aligned one", what);
    if (!a->tables_dev || !a->context_dev || (a->tables_dev | a->context_dev | a->q_offsets_dev) & 3)
        return set_error(c, WF_ERR_INVALID_ARGUMENT, "%s: tables, context and q_offsets are 4-byte aligned device arrays", what);
    if (!a->pages_out_dev || !a->lens_out_dev || a->pages_out_dev & 3 || a->lens_out_dev & 7)
        return set_error(c, WF_ERR_INVALID_ARGUMENT, "%s: pages_out is a 4-byte aligned device array, lens_out an 8-byte aligned one", what);
    const int page = a->page_tokens;
    if (page < 16 || page > 1024 || (page & (page - 1))) return set_error(c, WF_ERR_SHAPE, "%s: page_tokens %d is not a power of two from 16 to 1024", what, page);
    if (a->head_dim < 8 || a->head_dim > ATTN_MAX_DIM || a->head_dim % 8)
        return set_error(c, WF_ERR_SHAPE, "%s: head_dim %d is not a multiple of 8 from 8 to %d", what, a->head_dim, ATTN_MAX_DIM);
    if (a->kv_heads < 1 || a->kv_heads > 1024 || a->pages < 1 || a->pages * a->kv_heads > (1LL << 31) - 1024 || a->pages > (1LL << 31) - 1)
        return set_error(c, WF_ERR_SHAPE, "%s: bad cache, pages=%lld kv_heads=%d", what, (long long)a->pages, a->kv_heads);
    if (a->tokens < 0 || a->tokens > (1LL << 31) - 1024 || a->seqs < 0 || a->q_heads < 1 || a->q_heads > 8192 || a->tokens * a->q_heads >= (1LL << 31) || a->q_heads % a->kv_heads)
        return set_error(c, WF_ERR_SHAPE, "%s: bad shape tokens=%lld seqs=%d q_heads=%d kv_heads=%d", what, (long long)a->tokens, a->seqs, a->q_heads, a->kv_heads);
    if (a->q_heads / a->kv_heads > SELECT_MAX_GROUP) return set_error(c, WF_ERR_TOO_LARGE, "%s: more than %d query heads for each kv head", what, SELECT_MAX_GROUP);
    if (a->q_stride < (int64_t)a->q_heads * a->head_dim || a->q_stride % 8) return set_error(c, WF_ERR_SHAPE, "%s: q_stride %lld", what, (long long)a->q_stride);
    if (a->max_drafts < 1 || a->max_drafts > TREE_MAX_DRAFTS) return set_error(c, WF_ERR_TOO_LARGE, "%s: max_drafts %d is not 1 .. %d", what, a->max_drafts, TREE_MAX_DRAFTS);
    if (!a->q_offsets_dev && a->tokens != (int64_t)a->seqs * a->max_drafts)
        return set_error(c, WF_ERR_SHAPE, "%s: %lld tokens are not %d for each of %d sequences", what, (long long)a->tokens, a->max_drafts, a->seqs);
    if (a->table_stride < 1 || a->table_stride > (1LL << 31) / page - 1 || a->max_context < 0 || a->max_context > (1LL << 31) - 1024)
        return set_error(c, WF_ERR_SHAPE, "%s: table_stride %lld, max_context %lld", what, (long long)a->table_stride, (long long)a->max_context);
    if (a->first < 0 || a->recent < 0 || a->recent > 1 << 30 || a->width < 1 || a->width > (1LL << 31) / page - 1)
        return set_error(c, WF_ERR_SHAPE, "%s: first=%d recent=%d width=%d", what, a->first, a->recent, a->width);
    // the last `recent` tokens and the new ones, wherever the first of them lies in its page
    const int64_t ends = (int64_t)a->first + ((int64_t)a->recent + a->max_drafts + page - 2) / page + 1;
    if (a->width < ends) return set_error(c, WF_ERR_SHAPE, "%s: lists of %d pages, %lld are taken in any case", what, a->width, (long long)ends);
    const int64_t most = (std::min(a->max_context, a->table_stride * page) + page - 1) / page;  // pages of a context
    if (most > WF_SELECT_MAX_PAGES) return set_error(c, WF_ERR_TOO_LARGE, "%s: a context of %lld pages, at most %d", what, (long long)most, WF_SELECT_MAX_PAGES);
    const int64_t units = (int64_t)a->seqs * a->max_drafts * a->kv_heads;
    if (units > (1LL << 27)) return set_error(c, WF_ERR_TOO_LARGE, "%s: %d sequences of up to %d tokens, %d heads", what, a->seqs, a->max_drafts, a->kv_heads);
    SelectParams p{};
    p.q = reinterpret_cast<const bf16*>(a->q_dev);
    p.q_stride = a->q_stride;
    p.codes = reinterpret_cast<const int8_t*>(a->codes_dev);
    p.scales = reinterpret_cast<const float*>(a->scales_dev);
    p.q_offsets = reinterpret_cast<const int*>(a->q_offsets_dev);
    p.tables = reinterpret_cast<const int*>(a->tables_dev);
    p.table_stride = a->table_stride;
    p.context = reinterpret_cast<const int*>(a->context_dev);
    p.pages_out = reinterpret_cast<int*>(a->pages_out_dev);
    p.lens_out = reinterpret_cast<int2*>(a->lens_out_dev);
    p.tokens = a->tokens, p.max_context = a->max_context, p.pages = a->pages;
    p.kv_heads = a->kv_heads, p.dim = a->head_dim, p.group = a->q_heads / a->kv_heads;
    p.page_shift = __builtin_ctz((unsigned)page);
    p.max_drafts = a->max_drafts, p.width = a->width, p.first = a->first, p.recent = a->recent, p.tree = a->flags & WF_SELECT_TREE;
    p.group_inverse = p.group == 1 ? 0 : (uint32_t)(((1ull << 32) + p.group - 1) / p.group);
    p.room = (int)((most + 15) / 16 * 16);
    p.status = c->d_status;
    return 2 * a->head_dim <= 128 ? launch_selections<2>(c, p, a->seqs, s) : 2 * a->head_dim <= 192 ? launch_selections<3>(c, p, a->seqs, s) : launch_selections<4>(c, p, a->seqs, s);
}

}  // extern "C"
