// The pages of a key/value cache: who holds them (host), copies of pages and the move of kept tokens (device).
#include <algorithm>
#include <mutex>
#include <new>
#include <queue>
#include <unordered_set>

#include "wf_attention.cuh"

namespace wf {

CacheView cache_layer(const wf_kv_cache& cache, int layer);
int check_kv_cache(Context* c, const char* what, const wf_kv_cache* cache, int layer, bool packed_too);

// ---------------------------------------------------------------- who holds which page
struct PagePool {
    std::mutex mu;
    std::vector<int64_t> holders;
    std::priority_queue<int32_t, std::vector<int32_t>, std::greater<int32_t>> free_ids;  // lowest first: a cache stays dense at its start
};
static std::mutex g_pools_mu;
static std::unordered_set<PagePool*> g_pools;

// The pool stays locked, and in the registry, while `f` works on it.  Nothing may leave a C entry as an exception.
template <class F> static int with_pool(int64_t handle, F f) {
    try {
        std::lock_guard<std::mutex> lk(g_pools_mu);
        PagePool* p = reinterpret_cast<PagePool*>(handle);
        if (!p || !g_pools.count(p)) return WF_ERR_INVALID_HANDLE;
        std::lock_guard<std::mutex> in(p->mu);
        return f(*p);
    } catch (const std::bad_alloc&) {
        return WF_ERR_CUDA_BASE + (int)cudaErrorMemoryAllocation;
    } catch (...) {
        return WF_ERR_INVALID_ARGUMENT;
    }
}

// ---------------------------------------------------------------- copies
struct CopyParams {
    CacheView cache;
    size_t layer_elements;
    int layers;
    const int2* pairs;
    const int* rows;
    int64_t n;
    int* status;
};
// A unit is one head of one page in one layer, keys or values: contiguous on both sides.  A CTA has a unit at a time, COPY_DEPTH 16-byte pieces a thread in flight,
// and knows where the next one lies before it copies.  Bound by HBM (24 pages of 64 tokens, part full, 8 heads of 128, 32 layers: 204 MB in 39 to 44 us, 0.71 to 0.80 of a
// copy's rate).
constexpr int COPY_THREADS = 128, COPY_DEPTH = 8, COPY_CTAS = 8;  // CTAs of an SM
__global__ void __launch_bounds__(COPY_THREADS, COPY_CTAS) copy_pages_kernel(const __grid_constant__ CopyParams p) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const unsigned heads = (unsigned)p.cache.kv_heads, n = (unsigned)p.n, units = n * heads;  // of a layer's keys or values
    const int page_tokens = 1 << p.cache.page_shift;
    bf16* const base = (blockIdx.y & 1 ? p.cache.values : p.cache.keys) + (size_t)(blockIdx.y >> 1) * p.layer_elements;  // keys of layer 0, values of layer 0, keys of layer 1 ..
    int2 pair;
    int rows;
    auto look = [&](unsigned u) {
        pair = p.pairs[u / heads];
        rows = p.rows ? p.rows[u / heads] : page_tokens;
    };
    unsigned u = blockIdx.x;
    if (u < units) look(u);
    for (; u < units; u += gridDim.x) {
        const bool bad = pair.x < 0 || pair.y < 0 || pair.x >= p.cache.pages || pair.y >= p.cache.pages || rows < 0 || rows > page_tokens;
        if (bad && threadIdx.x == 0) report_status(p.status, STATUS_BAD_INDEX);
        const int head = (int)(u % heads), pieces = bad || pair.x == pair.y ? 0 : rows * p.cache.dim / 8;
        const uint4* from = reinterpret_cast<const uint4*>(base + p.cache.at(pair.x, head, 0));
        uint4* to = reinterpret_cast<uint4*>(base + p.cache.at(pair.y, head, 0));
        if (u + gridDim.x < units) look(u + gridDim.x);
        for (int j0 = threadIdx.x; j0 < pieces; j0 += COPY_DEPTH * COPY_THREADS) {
            uint4 v[COPY_DEPTH];
#pragma unroll
            for (int e = 0; e < COPY_DEPTH; e++)
                if (j0 + e * COPY_THREADS < pieces) v[e] = __ldcs(from + j0 + e * COPY_THREADS);
#pragma unroll
            for (int e = 0; e < COPY_DEPTH; e++)
                if (j0 + e * COPY_THREADS < pieces) __stcs(to + j0 + e * COPY_THREADS, v[e]);
        }
    }
}

struct CompactParams {
    CacheView cache;
    size_t layer_elements;
    int layers;
    const int* tables;
    int64_t table_stride;
    const int* context;
    const int* kept;
    int64_t kept_stride;
    const int* counts;
    int64_t seqs;
    int* status;
};
// A thread has one 16-byte piece of every kept token of a (layer, keys or values, sequence, head) and takes them in order, COMPACT_DEPTH
// at a time: all loads, then all stores.  kept ascends, so kept[i] >= i and token i is stored to a place that only an earlier
// token (or itself) came from: no load of a later batch can find it overwritten, and no two threads touch the same piece.  Bound by the launch and four loads that follow
// from one another (count, kept, table, key): 16 sequences of 16 drafts, 32 layers of 8 heads of 128, 8.5 us.
constexpr int COMPACT_THREADS = 128, COMPACT_DEPTH = 8;
__global__ void __launch_bounds__(COMPACT_THREADS) compact_kernel(const __grid_constant__ CompactParams p) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const unsigned pieces = (unsigned)p.cache.dim / 8, columns = pieces * p.cache.kv_heads, u = blockIdx.x * COMPACT_THREADS + threadIdx.x;
    if (u >= columns) return;
    const int piece = (int)(u % pieces), head = (int)(u / pieces), shift = p.cache.page_shift;
    bf16* const base = (blockIdx.z & 1 ? p.cache.values : p.cache.keys) + (size_t)(blockIdx.z >> 1) * p.layer_elements;
    for (int64_t s = blockIdx.y; s < p.seqs; s += gridDim.y) {
        const int* table = p.tables + s * p.table_stride;
        const int* kept = p.kept + s * p.kept_stride;
        const int64_t start = p.context[s], most = p.table_stride << shift;
        const int count = p.counts[s];
        bool bad = start < 0 || count < 0 || count > p.kept_stride;
        auto place = [&](int64_t t) -> uint4* {
            const int64_t page = table[t >> shift];
            if (page < 0 || page >= p.cache.pages) return nullptr;
            return reinterpret_cast<uint4*>(base + p.cache.at(page, head, (int)(t & ((1 << shift) - 1)))) + piece;
        };
        int before = -1;
        for (int i0 = 0; i0 < count && !bad; i0 += COMPACT_DEPTH) {
            uint4 v[COMPACT_DEPTH];
            uint4* to[COMPACT_DEPTH];
            int next[COMPACT_DEPTH];
#pragma unroll
            for (int e = 0; e < COMPACT_DEPTH; e++) next[e] = i0 + e < count ? kept[i0 + e] : 0;
#pragma unroll
            for (int e = 0; e < COMPACT_DEPTH; e++) {
                to[e] = nullptr;
                if (i0 + e >= count || bad) continue;
                const int j = next[e];
                if (j <= before || start + j >= most) {
                    bad = true;
                    continue;
                }
                before = j;
                if (j == i0 + e) continue;  // where it belongs already
                const uint4* from = place(start + j);
                to[e] = place(start + i0 + e);
                if (!from || !to[e]) {
                    bad = true;
                    to[e] = nullptr;
                    continue;
                }
                v[e] = *from;
            }
#pragma unroll
            for (int e = 0; e < COMPACT_DEPTH; e++)
                if (to[e]) *to[e] = v[e];
        }
        if (bad) report_status(p.status, STATUS_BAD_INDEX);
    }
}

}  // namespace wf

using namespace wf;

template <class Params> static int launch_cache(Context* c, const char* what, void (*kernel)(Params), dim3 grid, unsigned threads, cudaStream_t s, const Params& p) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
    if (e != cudaSuccess) return cuda_status(c, e, what);
    c->launches++;
    return WF_OK;
}

#define CACHE_ENTER(ctxh)                                                  \
    Context* c = get_context(ctxh);                                        \
    if (!c) return WF_ERR_INVALID_HANDLE;                                  \
    ScopedLock _lk(c);                                                     \
    if (!_lk.ok) return WF_ERR_BUSY;                                       \
    WF_CUDA(c, cudaSetDevice(c->device));                                  \
    cudaStream_t s = resolve_stream(c, stream)

extern "C" {

int wf_cache_copy_pages(int64_t ctx, const wf_kv_cache* cache, int64_t pairs_dev, int64_t rows_dev, int64_t n, int64_t stream) {
    CACHE_ENTER(ctx);
    const char* what = "cache_copy_pages";
    const int rc = check_kv_cache(c, what, cache, 0, false);
    if (rc != WF_OK) return rc;
    if (n < 0 || n > (1LL << 31) / cache->kv_heads - 1) return set_error(c, WF_ERR_SHAPE, "%s: %lld pairs", what, (long long)n);
    if (n == 0) return WF_OK;
    if (!pairs_dev || pairs_dev & 7 || rows_dev & 3) return set_error(c, WF_ERR_INVALID_ARGUMENT, "%s: pairs is an 8-byte aligned device array, rows a 4-byte aligned one", what);
    CopyParams p{};
    p.cache = cache_layer(*cache, 0);
    p.layer_elements = (size_t)cache->pages * cache->kv_heads * cache->page_tokens * cache->head_dim;
    p.layers = cache->layers;
    p.pairs = reinterpret_cast<const int2*>(pairs_dev);
    p.rows = reinterpret_cast<const int*>(rows_dev);
    p.n = n;
    p.status = c->d_status;
    const int64_t units = n * cache->kv_heads, wave = (int64_t)c->sm_count * COPY_CTAS;  // CTAs that the device holds
    const int64_t x = std::min<int64_t>(units, std::max<int64_t>(1, wave / (2 * cache->layers)));
    return launch_cache(c, what, copy_pages_kernel, dim3((unsigned)x, 2 * (unsigned)cache->layers), COPY_THREADS, s, p);
}

int wf_cache_compact(int64_t ctx, const wf_kv_cache* cache, int64_t tables_dev, int64_t table_stride, int64_t context_dev, int64_t kept_dev, int64_t kept_stride,
                     int64_t counts_dev, int64_t seqs, int64_t stream) {
    CACHE_ENTER(ctx);
    const char* what = "cache_compact";
    const int rc = check_kv_cache(c, what, cache, 0, false);
    if (rc != WF_OK) return rc;
    if (seqs < 0 || seqs > (1LL << 31) - 1 || kept_stride < 0 || kept_stride > (1LL << 31) - 1 || table_stride < 1 || table_stride > (1LL << 31) / cache->page_tokens - 1)
        return set_error(c, WF_ERR_SHAPE, "%s: seqs=%lld kept_stride=%lld table_stride=%lld", what, (long long)seqs, (long long)kept_stride, (long long)table_stride);
    if (seqs == 0 || kept_stride == 0) return WF_OK;
    if (!tables_dev || !context_dev || !kept_dev || !counts_dev || (tables_dev | context_dev | kept_dev | counts_dev) & 3)
        return set_error(c, WF_ERR_INVALID_ARGUMENT, "%s: tables, context, kept and counts are 4-byte aligned device arrays", what);
    CompactParams p{};
    p.cache = cache_layer(*cache, 0);
    p.layer_elements = (size_t)cache->pages * cache->kv_heads * cache->page_tokens * cache->head_dim;
    p.layers = cache->layers;
    p.tables = reinterpret_cast<const int*>(tables_dev);
    p.table_stride = table_stride;
    p.context = reinterpret_cast<const int*>(context_dev);
    p.kept = reinterpret_cast<const int*>(kept_dev);
    p.kept_stride = kept_stride;
    p.counts = reinterpret_cast<const int*>(counts_dev);
    p.seqs = seqs;
    p.status = c->d_status;
    const unsigned columns = (unsigned)cache->kv_heads * (unsigned)(cache->head_dim / 8);  // 16-byte pieces of a token
    return launch_cache(c, what, compact_kernel, dim3((columns + COMPACT_THREADS - 1) / COMPACT_THREADS, (unsigned)std::min<int64_t>(seqs, 65535), 2 * (unsigned)cache->layers), COMPACT_THREADS, s, p);
}

int wf_pages_create(int64_t pages, int64_t* pool) {
    if (!pool) return WF_ERR_INVALID_ARGUMENT;
    *pool = 0;
    if (pages < 0 || pages > (1LL << 31) - 1) return WF_ERR_SHAPE;
    try {
        std::unique_ptr<PagePool> p(new PagePool);
        p->holders.assign((size_t)pages, 0);
        std::vector<int32_t> ids((size_t)pages);
        for (int64_t i = 0; i < pages; i++) ids[(size_t)i] = (int32_t)i;
        p->free_ids = decltype(p->free_ids)(std::greater<int32_t>(), std::move(ids));
        std::lock_guard<std::mutex> lk(g_pools_mu);
        g_pools.insert(p.get());
        *pool = reinterpret_cast<int64_t>(p.release());
        return WF_OK;
    } catch (...) {
        return WF_ERR_CUDA_BASE + (int)cudaErrorMemoryAllocation;
    }
}

int wf_pages_destroy(int64_t pool) {
    PagePool* p = reinterpret_cast<PagePool*>(pool);
    std::lock_guard<std::mutex> lk(g_pools_mu);
    if (!p || !g_pools.erase(p)) return WF_ERR_INVALID_HANDLE;
    delete p;
    return WF_OK;
}

int wf_pages_take(int64_t pool, int64_t n, int32_t* ids) {
    return with_pool(pool, [&](PagePool& p) {
        if (n < 0 || (n > 0 && !ids)) return WF_ERR_INVALID_ARGUMENT;
        if (n > (int64_t)p.free_ids.size()) return WF_ERR_TOO_LARGE;
        for (int64_t i = 0; i < n; i++) {
            ids[i] = p.free_ids.top();
            p.free_ids.pop();
            p.holders[(size_t)ids[i]] = 1;
        }
        return WF_OK;
    });
}

int wf_pages_share(int64_t pool, int64_t n, const int32_t* ids) {
    return with_pool(pool, [&](PagePool& p) {
        if (n < 0 || (n > 0 && !ids)) return WF_ERR_INVALID_ARGUMENT;
        for (int64_t i = 0; i < n; i++)
            if (ids[i] < 0 || (size_t)ids[i] >= p.holders.size() || p.holders[(size_t)ids[i]] < 1) return WF_ERR_INDEX;
        for (int64_t i = 0; i < n; i++) p.holders[(size_t)ids[i]]++;
        return WF_OK;
    });
}

int wf_pages_release(int64_t pool, int64_t n, const int32_t* ids) {
    return with_pool(pool, [&](PagePool& p) {
        if (n < 0 || (n > 0 && !ids)) return WF_ERR_INVALID_ARGUMENT;
        int64_t done = 0;
        for (; done < n; done++) {
            if (ids[done] < 0 || (size_t)ids[done] >= p.holders.size() || p.holders[(size_t)ids[done]] < 1) break;
            p.holders[(size_t)ids[done]]--;
        }
        if (done < n) {  // nothing is changed
            while (done-- > 0) p.holders[(size_t)ids[done]]++;
            return WF_ERR_INDEX;
        }
        for (int64_t i = 0; i < n; i++)
            if (p.holders[(size_t)ids[i]] == 0) {
                p.holders[(size_t)ids[i]] = -1;  // named twice: freed once
                p.free_ids.push(ids[i]);
            }
        for (int64_t i = 0; i < n; i++)
            if (p.holders[(size_t)ids[i]] < 0) p.holders[(size_t)ids[i]] = 0;
        return WF_OK;
    });
}

int wf_pages_info(int64_t pool, int64_t* pages, int64_t* free_pages) {
    return with_pool(pool, [&](PagePool& p) {
        if (pages) *pages = (int64_t)p.holders.size();
        if (free_pages) *free_pages = (int64_t)p.free_ids.size();
        return WF_OK;
    });
}

int wf_pages_holders(int64_t pool, int32_t id, int64_t* holders) {
    return with_pool(pool, [&](PagePool& p) {
        if (!holders) return WF_ERR_INVALID_ARGUMENT;
        if (id < 0 || (size_t)id >= p.holders.size()) return WF_ERR_INDEX;
        *holders = p.holders[(size_t)id];
        return WF_OK;
    });
}

}  // extern "C"
