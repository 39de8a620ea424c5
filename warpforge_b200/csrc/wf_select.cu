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

int check_kv_cache(Context* c, const char* what, const wf_kv_cache* cache, int layer, bool packed_too);
CacheView cache_layer(const wf_kv_cache& cache, int layer);

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

// A warp has one head of one page in one layer, contiguous in memory: a lane has 8 elements of a row, 32 / (dim / 8) rows go with one load, BOUNDS_DEPTH loads are in flight.
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
        const int j = (first >> shift) + index, begin = j << shift;
        if (first == stop || begin >= stop) continue;
        const int64_t page = p.tables[s * p.table_stride + j];
        if (page < 0 || page >= p.cache.pages) {
            if (lane == 0) report_status(p.status, STATUS_BAD_INDEX);
            continue;
        }
        const uint4* from = reinterpret_cast<const uint4*>(keys + p.cache.at(page, head, 0)) + lane;
        const int all = lane < active ? min(page_tokens, stop - begin) * pieces - lane : 0;  // this lane's pieces: 0, active, 2 active .. below it
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
    int room;  // pages whose scores a CTA can hold
    int* status;
};
constexpr int SELECT_WARPS = 16, SELECT_THREADS = SELECT_WARPS * 32;
constexpr int SELECT_MAX_GROUP = 128, SELECT_BINS = 256;

__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// A cluster has one new token and kv head.  Its CTAs score a part of the pages each, 16 pages by the heads of the group a warp at a time (mma.sync on the codes: [q+ | q-] . [hi | lo],
// the positive elements of q in the one half and the negative ones in the other), and leave the scores in the first CTA's shared memory, which takes the largest.
// CHUNKS of 64 codes of a page (hi and lo together).
template <int CHUNKS> __global__ void __launch_bounds__(SELECT_THREADS) select_pages_kernel(const __grid_constant__ SelectParams p) {
    extern __shared__ uint32_t keys[];  // [room] scores, as unsigned numbers of the same order
    __shared__ uint4 q_codes[SELECT_MAX_GROUP / 8][CHUNKS][32];  // as the lanes of an MMA take them
    __shared__ int q_scale[SELECT_MAX_GROUP];  // exponents as they are added to a score
    __shared__ uint32_t bins[SELECT_BINS], warp_sums[SELECT_WARPS], warp_low[SELECT_WARPS], warp_high[SELECT_WARPS], found[3];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    uint32_t rank, ranks;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
    cluster_arrive();  // the first CTA is there before anything is sent to it
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, quad = lane & 3;
    const unsigned unit = blockIdx.x / ranks, per_seq = (unsigned)p.max_drafts * p.kv_heads, s = unit / per_seq, of_seq = unit - s * per_seq;
    const int i = (int)(of_seq / p.kv_heads), head = (int)(of_seq - i * p.kv_heads);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int64_t a = p.q_offsets ? p.q_offsets[s] : (int64_t)s * p.max_drafts, b = p.q_offsets ? p.q_offsets[s + 1] : a + p.max_drafts;
    const bool no_rows = a < 0 || b < a || b > p.tokens || b - a > p.max_drafts;
    if (no_rows && tid == 0 && rank == 0) report_status(p.status, STATUS_BAD_INDEX);
    if (no_rows || i >= (int)(b - a)) {  // all of the cluster
        cluster_wait();
        return;
    }
    const int rows = (int)(b - a), context = p.context[s], shift = p.page_shift, page_tokens = 1 << shift;
    const int64_t row = a + i;
    const bool bad = context < 0 || (int64_t)context > p.max_context || (int64_t)context + rows > p.table_stride << shift;
    if (bad && tid == 0 && rank == 0) report_status(p.status, STATUS_BAD_INDEX);
    const int* const table = p.tables + (size_t)s * p.table_stride;
    const int last = bad ? 0 : (context + rows + page_tokens - 1) >> shift;             // pages of the sequence
    const int tail = bad ? 0 : max(0, context - p.recent) >> shift;                     // from here on all are taken
    const int first = min(p.first, tail), between = tail - first, ends = first + last - tail;
    const int take = min(between, p.width - ends), count = ends + take;                 // the host sees to it that the ends fit
    int* const list = p.pages_out + ((size_t)row * p.kv_heads + head) * p.width;
    if (rank == ranks - 1) {
        for (int n = tid; n < p.width - take; n += SELECT_THREADS) {  // the places that the scores do not decide
            const int at = n < first ? n : n + take, page = at < first ? at : tail + at - first - take;
            list[at] = at < count ? table[page] : -1;
        }
        if (tid == 0) {
            const int held = bad ? 0 : context - (between - take) * page_tokens;
            p.lens_out[row * p.kv_heads + head] = make_int2(held, bad ? 0 : held + (p.tree ? rows : i + 1));
        }
    }
    if (take == between) {  // all of them
        if (rank == 0)
            for (int n = tid; n < take; n += SELECT_THREADS) list[first + n] = table[first + n];
        cluster_wait();
        return;
    }

    // The heads of the group in 8 bits, a warp a head.
    const int column_tiles = (p.group + 7) / 8;
    for (int n = tid; n < column_tiles * CHUNKS * 32; n += SELECT_THREADS) (&q_codes[0][0][0])[n] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    for (int h = warp; h < p.group; h += SELECT_WARPS) {
        const bf16* q = p.q + row * p.q_stride + (size_t)(head * p.group + h) * p.dim + 4 * lane;
        const bool mine = 4 * lane < p.dim;
        const uint2 w = mine ? *reinterpret_cast<const uint2*>(q) : make_uint2(0, 0);
        const uint32_t x = w.x & 0x7FFF7FFFu, y = w.y & 0x7FFF7FFFu;
        const uint32_t size = __reduce_max_sync(0xFFFFFFFFu, max(max(x & 0xFFFF, x >> 16), max(y & 0xFFFF, y >> 16)));
        const bool fine = size < 0x7F80;  // a head with an Inf or a NaN has no preferences
        const int exponent = fine ? scale_exponent(size) : 0;
        const float by = power_of_two(-exponent);
        uint32_t plus = 0, minus = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const uint32_t half = e & 2 ? w.y : w.x;
            const int v = fine ? __float2int_rn(__uint_as_float(e & 1 ? half & 0xFFFF0000u : half << 16) * by) : 0;
            plus |= (uint32_t)(max(v, 0) & 0xFF) << 8 * e;
            minus |= (uint32_t)(min(v, 0) & 0xFF) << 8 * e;
        }
        if (mine) {
            const int k0 = 4 * lane, k1 = p.dim + 4 * lane;  // bytes of a page's codes
            auto at = [&](int k) { return reinterpret_cast<uint32_t*>(&q_codes[h / 8][k / 64][(h & 7) * 4 + (k & 63) / 16]) + (k & 15) / 4; };
            *at(k0) = plus;
            *at(k1) = minus;
        }
        if (lane == 0) q_scale[h] = (exponent - LEAST_SCALE) << 20;
    }
    __syncthreads();
    if (ranks > 1) cluster_wait();

    // Scores.  Lane g * 4 + quad has 16 codes of pages g and g + 8 of a tile in every chunk; which of them are called which k of the product does not matter, so long as q has the same.
    const uint32_t to = map_to_rank((uint32_t)__cvta_generic_to_shared(keys), 0);
    const int tiles = (between + 15) / 16, mine0 = (int)((int64_t)tiles * rank / ranks), mine1 = (int)((int64_t)tiles * (rank + 1) / ranks);
    const int codes = 2 * p.dim;
    for (int t = mine0 + warp; t < mine1; t += SELECT_WARPS) {
        int64_t entry[2];
        bool real[2], inside[2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int n = t * 16 + g + 8 * e;
            inside[e] = n < between;
            const int64_t page = inside[e] ? table[first + n] : 0;
            real[e] = page >= 0 && page < p.pages;
            if (!real[e] && quad == 0) report_status(p.status, STATUS_BAD_INDEX);
            entry[e] = (real[e] ? page : 0) * p.kv_heads + head;
        }
        uint4 c[2][CHUNKS];
        uint32_t scale[2];  // exponent as in a float
#pragma unroll
        for (int e = 0; e < 2; e++) {
#pragma unroll
            for (int k = 0; k < CHUNKS; k++) {
                const bool some = 64 * k + 16 * quad < codes;
                c[e][k] = some ? *reinterpret_cast<const uint4*>(p.codes + entry[e] * codes + 64 * k + 16 * quad) : make_uint4(0, 0, 0, 0);
            }
            scale[e] = __float_as_uint(p.scales[entry[e]]) >> 23 & 0xFF;
        }
        int best[2] = {INT_MIN, INT_MIN};
        for (int n = 0; n < column_tiles; n++) {
            int sum[4] = {0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < CHUNKS; k++) {
                const uint4 q = q_codes[n][k][lane];
                mma_s8(sum, c[0][k].x, c[1][k].x, c[0][k].y, c[1][k].y, q.x, q.y);
                mma_s8(sum, c[0][k].z, c[1][k].z, c[0][k].w, c[1][k].w, q.z, q.w);
            }
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int h = n * 8 + 2 * quad + (e & 1);
                // a float's exponent and the 20 bits of significand that such a number has, and the scale's exponent on top
                const int size = sum[e] ? (__float_as_int((float)abs(sum[e])) >> 3) + q_scale[h] : 0;
                if (h < p.group) best[e >> 1] = max(best[e >> 1], sum[e] < 0 ? -size : size);
            }
        }
#pragma unroll
        for (int e = 0; e < 2; e++) {
            best[e] = max(best[e], __shfl_xor_sync(0xFFFFFFFFu, best[e], 1));
            best[e] = max(best[e], __shfl_xor_sync(0xFFFFFFFFu, best[e], 2));
            const int more = ((int)scale[e] - 127 - LEAST_SCALE) << 20;  // the page's scale (a size begins at 127 << 20: no sign changes)
            const int score = best[e] > 0 ? best[e] + more : best[e] < 0 ? best[e] - more : 0;
            const uint32_t key = !real[e] ? 0 : scale[e] == 0xFF ? 0xFFFFFFFFu : (uint32_t)score ^ 0x80000000u;
            if (quad == 0 && inside[e]) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to + 4 * (uint32_t)(t * 16 + g + 8 * e)), "r"(key) : "memory");
        }
    }
    if (ranks > 1) {
        cluster_arrive();
        cluster_wait();
        if (rank) return;  // nothing is sent to the others
    } else {
        cluster_wait();  // that of the start
        __syncthreads();
    }

    // The largest `take` of them: the key of the last one, by eight bits at a time of what is above the smallest key, and how many of that key.
    uint32_t low = 0xFFFFFFFFu, high = 0;
    for (int n = tid; n < between; n += SELECT_THREADS) low = min(low, keys[n]), high = max(high, keys[n]);
    low = __reduce_min_sync(0xFFFFFFFFu, low);
    high = __reduce_max_sync(0xFFFFFFFFu, high);
    if (lane == 0) warp_low[warp] = low, warp_high[warp] = high;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < SELECT_WARPS; w++) low = min(low, warp_low[w]), high = max(high, warp_high[w]);
    int bits = 32 - __clz(high - low);      // of the differences that are still open
    uint32_t prefix = 0, need = (uint32_t)take;  // what is decided of the difference; how many are still to be taken of those that begin so
    while (bits > 0) {
        const int less = max(0, bits - 8);
        if (tid < SELECT_BINS) bins[tid] = 0;
        __syncthreads();
        for (int n = tid; n < between; n += SELECT_THREADS) {
            const uint32_t d = keys[n] - low;
            if (bits == 32 || d >> bits == prefix >> bits) atomicAdd(&bins[d >> less & (SELECT_BINS - 1)], 1u);
        }
        __syncthreads();
        if (warp == 0) {  // the bin of the last one, from above: a lane has eight bins
            uint32_t mine[8], sum = 0;
#pragma unroll
            for (int e = 0; e < 8; e++) sum += mine[e] = bins[SELECT_BINS - 1 - (lane * 8 + e)];
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
        __syncthreads();
    }
    // Those that begin above the prefix, and of those that begin like it the first `need`.  A thread has a run of pages, of odd length for the sake of the banks.
    const int run = ((between + SELECT_THREADS - 1) / SELECT_THREADS) | 1, from = min(tid * run, between), end = min(from + run, between);
    const uint32_t border = prefix >> bits;
    uint32_t mine = 0, alike = 0;  // of the run: above the border, on it
    for (int n = from; n < end; n++) {
        const uint32_t d = (keys[n] - low) >> bits;
        mine += d > border;
        alike += d == border;
    }
    unsigned long long both = (unsigned long long)alike << 32 | mine, sum = both;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long v = __shfl_up_sync(0xFFFFFFFFu, sum, o);
        if (lane >= o) sum += v;
    }
    __shared__ unsigned long long totals[SELECT_WARPS];
    if (lane == 31) totals[warp] = sum;
    __syncthreads();
    sum -= both;
    for (int w = 0; w < warp; w++) sum += totals[w];
    uint32_t above = (uint32_t)sum, like = (uint32_t)(sum >> 32);
    for (int n = from; n < end; n++) {
        const uint32_t d = (keys[n] - low) >> bits;
        const bool taken = d > border || (d == border && like < need);
        if (taken) list[first + above + min(like, need)] = table[first + n];
        above += d > border;
        like += d == border;
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

template <class Params>
static int launch_select(Context* c, const char* what, void (*kernel)(Params), dim3 grid, unsigned threads, unsigned cluster, size_t smem, cudaStream_t s, const Params& p) {
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
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
    if (e != cudaSuccess) return cuda_status(c, e, what);
    c->launches++;
    return WF_OK;
}

template <int CHUNKS> static int launch_selection(Context* c, const SelectParams& p, int64_t units, unsigned cluster, cudaStream_t s) {
    static std::atomic<uint64_t> ready{0};  // devices whose attribute is set
    if (!(ready.load() >> (c->device & 63) & 1)) {
        WF_CUDA(c, cudaFuncSetAttribute(select_pages_kernel<CHUNKS>, cudaFuncAttributeMaxDynamicSharedMemorySize, WF_SELECT_MAX_PAGES * 4));
        ready.fetch_or(1ull << (c->device & 63));
    }
    return launch_select(c, "select_pages", select_pages_kernel<CHUNKS>, dim3((unsigned)(units * cluster)), SELECT_THREADS, cluster, (size_t)p.room * 4, s, p);
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
    return launch_select(c, what, page_bounds_kernel, dim3((unsigned)((units + BOUNDS_WARPS - 1) / BOUNDS_WARPS), (unsigned)std::min<int64_t>(seqs, 65535), (unsigned)cache->layers),
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
    p.room = (int)((most + 15) / 16 * 16);
    p.status = c->d_status;
    unsigned cluster = 1;
    while (cluster < 8 && units * cluster * 2 <= c->sm_count && most >= 256 * (int)cluster) cluster *= 2;
    return 2 * a->head_dim <= 128 ? launch_selection<2>(c, p, units, cluster, s) : launch_selection<4>(c, p, units, cluster, s);
}

}  // extern "C"
