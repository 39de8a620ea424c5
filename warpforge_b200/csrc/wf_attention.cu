// Attention over a paged cache: wf_prompt_attention and wf_tree_attention.
//   out = softmax(scale q k^T) v   over the keys that a row sees, with base-2 exponentials: softmax(x) = 2^(x log2 e - m) / sum
#include <algorithm>
#include <atomic>

#include "wf_attention_prompt.cuh"
#include "wf_attention_tree.cuh"

using namespace wf;

static int check_cache(Context* c, const char* what, const wf_kv_cache* cache, int layer, bool packed_too) {
    if (!cache) return set_error(c, WF_ERR_INVALID_ARGUMENT, "%s: null cache", what);
    if (!cache->keys_dev || !cache->values_dev || (cache->keys_dev | cache->values_dev) & 15)
        return set_error(c, WF_ERR_INVALID_ARGUMENT, "%s: keys and values must be 16-byte aligned device addresses", what);
    if (cache->layers < 1 || cache->layers > 32767 || layer < 0 || layer >= cache->layers) return set_error(c, WF_ERR_SHAPE, "%s: layer %d of %d", what, layer, cache->layers);
    if (cache->head_dim < 8 || cache->head_dim > ATTN_MAX_DIM || cache->head_dim % 8)
        return set_error(c, WF_ERR_SHAPE, "%s: head_dim %d is not a multiple of 8 from 8 to %d", what, cache->head_dim, ATTN_MAX_DIM);
    const int p = cache->page_tokens;
    if (!(packed_too && p == 1 && cache->layers == 1) && (p < 16 || p > 1024 || (p & (p - 1))))
        return set_error(c, WF_ERR_SHAPE, "%s: page_tokens %d is not a power of two from 16 to 1024", what, p);
    if (cache->kv_heads < 1 || cache->kv_heads > 1024 || cache->pages < 0 || cache->pages > (1LL << 31) - 1 ||
        cache->pages * cache->kv_heads * p > (1LL << 31) - 1024)
        return set_error(c, WF_ERR_SHAPE, "%s: bad cache, pages=%lld kv_heads=%d", what, (long long)cache->pages, cache->kv_heads);
    return WF_OK;
}
namespace wf {
CacheView cache_layer(const wf_kv_cache& cache, int layer) {
    CacheView v;
    v.pages = cache.pages;
    v.kv_heads = cache.kv_heads;
    v.dim = cache.head_dim;
    v.page_shift = __builtin_ctz((unsigned)cache.page_tokens);
    const size_t skip = (size_t)layer * cache.pages * cache.kv_heads * cache.page_tokens * cache.head_dim;
    v.keys = reinterpret_cast<bf16*>(cache.keys_dev) + skip;
    v.values = reinterpret_cast<bf16*>(cache.values_dev) + skip;
    return v;
}
int check_kv_cache(Context* c, const char* what, const wf_kv_cache* cache, int layer, bool packed_too) { return check_cache(c, what, cache, layer, packed_too); }
}  // namespace wf
static int check_queries(Context* c, const char* what, int64_t q, int64_t out, int64_t q_stride, int64_t tokens, int seqs, int q_heads, const wf_kv_cache* cache) {
    if (!q || !out || (q | out) & 15) return set_error(c, WF_ERR_INVALID_ARGUMENT, "%s: q and out must be 16-byte aligned device addresses", what);
    if (tokens < 0 || tokens > (1LL << 31) - 1024 || seqs < 0 || q_heads < 1 || q_heads > 8192 || tokens * q_heads >= (1LL << 31))
        return set_error(c, WF_ERR_SHAPE, "%s: bad shape tokens=%lld seqs=%d q_heads=%d", what, (long long)tokens, seqs, q_heads);
    if (q_heads % cache->kv_heads) return set_error(c, WF_ERR_SHAPE, "%s: %d query heads over %d kv heads", what, q_heads, cache->kv_heads);
    if (q_heads / cache->kv_heads > 128) return set_error(c, WF_ERR_TOO_LARGE, "%s: more than 128 query heads for each kv head", what);
    if (q_stride < (int64_t)q_heads * cache->head_dim || q_stride % 8) return set_error(c, WF_ERR_SHAPE, "%s: q_stride %lld", what, (long long)q_stride);
    return WF_OK;
}
template <class... Params, class... Args>
static int launch_attention(Context* c, const char* what, void (*kernel)(Params...), dim3 grid, unsigned threads, size_t smem, cudaStream_t s, const Args&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
    if (e != cudaSuccess) return cuda_status(c, e, what);
    c->launches++;
    return WF_OK;
}

// bf16 [z][y][x] with the given distances (elements) between y and z; boxes of 64 elements x by x bz, 128-byte swizzle, zeros outside
static int encode_rows(Context* c, CUtensorMap* map, const void* base, int64_t x, int64_t y, int64_t z, int64_t y_apart, int64_t z_apart, int by, int bz) {
    const cuuint64_t dims[3] = {(cuuint64_t)x, (cuuint64_t)y, (cuuint64_t)z}, strides[2] = {(cuuint64_t)y_apart * 2, (cuuint64_t)z_apart * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)by, (cuuint32_t)bz}, step[3] = {1, 1, 1};
    const EncodeTiledFn encode = encode_tiled_fn();
    if (!encode) return set_error(c, WF_ERR_NO_DEVICE, "the driver has no cuTensorMapEncodeTiled");
    const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_error(c, WF_ERR_CUDA_BASE + (int)cudaErrorInvalidValue, "cuTensorMapEncodeTiled failed: %d", (int)r);
    return WF_OK;
}
static int encode_cache(Context* c, CUtensorMap* map, const bf16* base, const CacheView& v, int box_rows) {
    if (v.page_shift == 0) return encode_rows(c, map, base, v.dim, v.kv_heads, v.pages, v.dim, (int64_t)v.kv_heads * v.dim, 1, box_rows);
    return encode_rows(c, map, base, v.dim, 1, (v.pages * v.kv_heads) << v.page_shift, v.dim, v.dim, 1, box_rows);
}
static bool rows_of_sectors(const bf16* out, int dim) { return reinterpret_cast<uintptr_t>(out) % 32 == 0 && dim % 16 == 0; }
static int dim_chunks(int dim) { return (dim + 63) / 64; }

template <int CHUNKS> static int launch_prompt(Context* c, const PromptParams& p, cudaStream_t s) {
    const char* what = "prompt_attention";
    static std::atomic<uint64_t> ready{0};  // devices whose attribute is set
    if (!(ready.load() >> (c->device & 63) & 1)) {
        WF_CUDA(c, cudaFuncSetAttribute(prompt_tiles_kernel<CHUNKS, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, PromptShape<CHUNKS>::SMEM));
        ready.fetch_or(1ull << (c->device & 63));
    }
    GemvScratch& scratch = c->gemv_scratch[s];
    if (!scratch.d_attn_sched) {
        const int rc = refuse_allocation_while_recording(c, s, "the counters of prompt_attention");
        if (rc != WF_OK) return rc;
        std::shared_ptr<unsigned int> sched;
        WF_CUDA(c, make_shared_device(c, sched, 2 * sizeof(unsigned int)));
        WF_CUDA(c, cudaMemsetAsync(sched.get(), 0, 2 * sizeof(unsigned int), s));
        scratch.d_attn_sched = sched;
    }
    PromptTiles t{};
    t.p = p;
    t.tile_tokens = PA_ROWS / p.group;
    t.box_rows = p.tables ? std::min(PA_KEYS, 1 << p.cache.page_shift) : PA_KEYS;
    t.sched = scratch.d_attn_sched.get();
    t.wide_rows = rows_of_sectors(p.out, p.cache.dim);
    CUtensorMap q, k, v;
    int rc = encode_rows(c, &q, p.q, p.cache.dim, p.q_heads, p.tokens, p.cache.dim, p.q_stride, p.group, t.tile_tokens);
    if (rc == WF_OK) rc = encode_cache(c, &k, p.cache.keys, p.cache, t.box_rows);
    if (rc == WF_OK) rc = encode_cache(c, &v, p.cache.values, p.cache, t.box_rows);
    if (rc != WF_OK) return rc;
    // Items of two tiles of rows; of one, on which both groups of a CTA work, where that many would leave half of the device idle.  Pairs / ones in us: 256, 512, 640, 1024 tokens
    // of 32 / 32 heads of 128 10.9 / 10.0, 14.5 / 12.2, 15.2 / 17.6, 22.6 / 23.7; 300, 600, 1000 of 32 / 8 heads 12.5 / 11.4, 16.5 / 16.9, 21.5 / 23.2.
    const int64_t pairs = (p.tokens + (int64_t)p.seqs * (2 * t.tile_tokens - 1)) / (2 * t.tile_tokens) * p.cache.kv_heads;
    if (pairs > (1LL << 31) - 65536) return set_error(c, WF_ERR_TOO_LARGE, "%s: %lld tokens of %d heads", what, (long long)p.tokens, p.q_heads);
    t.split = 2 * pairs <= c->sm_count;
    const int64_t items = t.split ? (p.tokens + (int64_t)p.seqs * (t.tile_tokens - 1)) / t.tile_tokens * p.cache.kv_heads : pairs;
    return launch_attention(c, what, prompt_tiles_kernel<CHUNKS, false>, (unsigned)std::min<int64_t>(items, c->sm_count), PA_THREADS, (size_t)PromptShape<CHUNKS>::SMEM, s, t, q, k, v);
}

// Where the pieces of cut units go.
static int tree_scratch(Context* c, cudaStream_t s, int64_t floats, TreeCuts* cuts) {
    GemvScratch& scratch = c->gemv_scratch[s];
    const int64_t head = (c->sm_count * (int64_t)sizeof(TreeCut) + 255) & ~255LL, bytes = head + floats * (int64_t)sizeof(float);
    if (bytes > scratch.attn_bytes) {
        const int rc = refuse_allocation_while_recording(c, s, "the pieces of tree_attention");
        if (rc != WF_OK) return rc;
        scratch.d_attn.reset();
        scratch.attn_bytes = 0;
        WF_CUDA(c, make_shared_device(c, scratch.d_attn, (size_t)bytes));
        scratch.attn_bytes = bytes;
    }
    cuts->cuts = reinterpret_cast<TreeCut*>(scratch.d_attn.get());
    cuts->pieces = reinterpret_cast<float*>(scratch.d_attn.get() + head);
    return WF_OK;
}
static int launch_join(Context* c, const TreeParams& p, const TreeCuts& cuts, unsigned ctas, int rows, cudaStream_t s) {
    return launch_attention(c, "tree_attention", tree_join_kernel, dim3(ctas, (unsigned)((rows + JOIN_WARPS - 1) / JOIN_WARPS)), JOIN_WARPS * 32, 0, s, p, cuts);
}
template <int CHUNKS, int MT> static int launch_tree(Context* c, const TreeParams& p, cudaStream_t s) {
    const char* what = "tree_attention";
    typedef TreeShape<CHUNKS, MT> Shape;
    static std::atomic<uint64_t> ready{0};  // devices whose attribute is set
    if (!(ready.load() >> (c->device & 63) & 1)) {
        WF_CUDA(c, cudaFuncSetAttribute(tree_tiles_kernel<CHUNKS, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::SMEM));
        ready.fetch_or(1ull << (c->device & 63));
    }
    const int64_t blocks = ((int64_t)p.max_drafts * p.group + Shape::ROWS - 1) / Shape::ROWS, tiles = (p.max_context + p.max_drafts + TA_KEYS - 1) / TA_KEYS;
    TreeTiles t{};
    t.p = p;
    const int64_t units = p.seqs * blocks * p.cache.kv_heads;
    t.c.may_cut = line_is_cut(units, tiles, c->sm_count, TA_CUT_TILES, TA_CUT_ANYWAY);
    t.c.piece_rows = t.c.tile_rows = t.c.tile_room = Shape::ROWS;
    t.c.dim = Shape::DIM;
    int rc = tree_scratch(c, s, t.c.may_cut ? (int64_t)c->sm_count * 2 * Shape::PIECE : 0, &t.c);
    CUtensorMap k, v;
    if (rc == WF_OK) rc = encode_cache(c, &k, p.cache.keys, p.cache, TA_KEYS);
    if (rc == WF_OK) rc = encode_cache(c, &v, p.cache.values, p.cache, TA_KEYS);
    if (rc != WF_OK) return rc;
    const int64_t most = t.c.may_cut ? std::min<int64_t>(units, c->sm_count) * tiles : units;  // CTAs that can have work
    const unsigned grid = (unsigned)std::min<int64_t>(most, c->sm_count);
    rc = launch_attention(c, what, tree_tiles_kernel<CHUNKS, MT>, grid, TA_THREADS, (size_t)Shape::SMEM, s, t, k, v);
    return rc == WF_OK && t.c.may_cut ? launch_join(c, p, t.c, grid, Shape::ROWS, s) : rc;
}

// The prompt kernel on the rows of trees.
template <int CHUNKS> static int launch_wide_tree(Context* c, const TreeParams& p, cudaStream_t s) {
    static std::atomic<uint64_t> ready{0};  // devices whose attribute is set
    if (!(ready.load() >> (c->device & 63) & 1)) {
        WF_CUDA(c, cudaFuncSetAttribute(prompt_tiles_kernel<CHUNKS, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, PromptShape<CHUNKS>::SMEM));
        ready.fetch_or(1ull << (c->device & 63));
    }
    PromptTiles t{};
    t.tree = p;
    t.p.cache = p.cache;
    t.p.q = p.q, t.p.out = p.out, t.p.q_stride = p.q_stride;
    t.p.tables = p.tables, t.p.table_stride = p.table_stride;
    t.p.q_heads = p.q_heads, t.p.group = p.group;
    t.p.scale_log2 = p.scale_log2;
    t.p.status = p.status;
    t.tile_tokens = PA_ROWS / p.group;
    t.box_rows = std::min(PA_KEYS, 1 << p.cache.page_shift);
    t.wide_rows = rows_of_sectors(p.out, p.cache.dim);
    const int64_t blocks = (p.max_drafts + 2 * t.tile_tokens - 1) / (2 * t.tile_tokens), tiles = (p.max_context + p.max_drafts + PA_KEYS - 1) / PA_KEYS;
    const int64_t units = p.seqs * blocks * p.cache.kv_heads;
    t.c.may_cut = line_is_cut(units, tiles, c->sm_count, PA_CUT_TILES, PA_CUT_ANYWAY);
    t.c.piece_rows = p.max_drafts <= t.tile_tokens ? PA_ROWS : 2 * PA_ROWS;
    t.c.tile_rows = t.tile_tokens * p.group;
    t.c.tile_room = PA_ROWS;
    t.c.dim = CHUNKS * 64;
    int rc = tree_scratch(c, s, t.c.may_cut ? (int64_t)c->sm_count * 2 * t.c.piece_rows * (t.c.dim + 2) : 0, &t.c);
    CUtensorMap q, k, v;
    if (rc == WF_OK) rc = encode_rows(c, &q, p.q, p.cache.dim, p.q_heads, p.tokens, p.cache.dim, p.q_stride, p.group, t.tile_tokens);
    if (rc == WF_OK) rc = encode_cache(c, &k, p.cache.keys, p.cache, t.box_rows);
    if (rc == WF_OK) rc = encode_cache(c, &v, p.cache.values, p.cache, t.box_rows);
    if (rc != WF_OK) return rc;
    const int64_t most = t.c.may_cut ? std::min<int64_t>(units, c->sm_count) * tiles : units;  // CTAs that can have work
    const unsigned grid = (unsigned)std::min<int64_t>(most, c->sm_count);
    rc = launch_attention(c, "tree_attention", prompt_tiles_kernel<CHUNKS, true>, grid, PA_THREADS, (size_t)PromptShape<CHUNKS>::SMEM, s, t, q, k, v);
    return rc == WF_OK && t.c.may_cut ? launch_join(c, p, t.c, grid, std::min(p.max_drafts, 2 * t.tile_tokens) * p.group, s) : rc;
}

#define ATTENTION_ENTER(ctxh)                                              \
    Context* c = get_context(ctxh);                                        \
    if (!c) return WF_ERR_INVALID_HANDLE;                                  \
    ScopedLock _lk(c);                                                     \
    if (!_lk.ok) return WF_ERR_BUSY;                                       \
    WF_CUDA(c, cudaSetDevice(c->device));                                  \
    cudaStream_t s = resolve_stream(c, stream)

extern "C" {

int wf_prompt_attention(int64_t ctx, const wf_prompt_attention_args* a, const wf_kv_cache* cache, int layer, int64_t stream) {
    ATTENTION_ENTER(ctx);
    const char* what = "prompt_attention";
    if (!a || !cache) return set_error(c, WF_ERR_INVALID_ARGUMENT, "%s: null arguments", what);
    if (a->tokens == 0 || a->seqs == 0) return WF_OK;
    int rc = check_cache(c, what, cache, layer, true);
    if (rc == WF_OK) rc = check_queries(c, what, a->q_dev, a->out_dev, a->q_stride, a->tokens, a->seqs, a->q_heads, cache);
    if (rc != WF_OK) return rc;
    const bool packed = cache->page_tokens == 1;
    if (!a->q_offsets_dev || a->q_offsets_dev & 3 || a->tables_dev & 3 || a->k_lens_dev & 3)
        return set_error(c, WF_ERR_INVALID_ARGUMENT, "%s: q_offsets, tables and k_lens are 4-byte aligned device arrays", what);
    if (packed ? a->tables_dev || a->k_lens_dev : !a->tables_dev || !a->k_lens_dev)
        return set_error(c, WF_ERR_INVALID_ARGUMENT, "%s: pages need tables and k_lens, packed keys take neither", what);
    if (!packed && (a->table_stride < 1 || a->table_stride > (1LL << 31) / cache->page_tokens - 1))
        return set_error(c, WF_ERR_SHAPE, "%s: table_stride %lld", what, (long long)a->table_stride);
    if (!(a->scale > 0.f) || a->scale > 1e30f) return set_error(c, WF_ERR_INVALID_ARGUMENT, "%s: scale %g", what, (double)a->scale);
    if (cache->pages < 1) return set_error(c, WF_ERR_SHAPE, "%s: a cache without pages", what);
    PromptParams p{};
    p.cache = cache_layer(*cache, layer);
    p.q = reinterpret_cast<const bf16*>(a->q_dev);
    p.out = reinterpret_cast<bf16*>(a->out_dev);
    p.q_stride = a->q_stride;
    p.q_offsets = reinterpret_cast<const int*>(a->q_offsets_dev);
    p.tables = reinterpret_cast<const int*>(a->tables_dev);
    p.table_stride = a->table_stride;
    p.k_lens = reinterpret_cast<const int*>(a->k_lens_dev);
    p.tokens = a->tokens;
    p.seqs = a->seqs;
    p.q_heads = a->q_heads;
    p.group = a->q_heads / cache->kv_heads;
    p.scale_log2 = a->scale * 1.44269504f;
    p.status = c->d_status;
    return dim_chunks(cache->head_dim) == 1 ? launch_prompt<1>(c, p, s) : launch_prompt<2>(c, p, s);
}

int wf_tree_attention(int64_t ctx, const wf_tree_attention_args* a, const wf_kv_cache* cache, int layer, int64_t stream) {
    ATTENTION_ENTER(ctx);
    const char* what = "tree_attention";
    if (!a || !cache) return set_error(c, WF_ERR_INVALID_ARGUMENT, "%s: null arguments", what);
    if (a->tokens == 0 || a->seqs == 0) return WF_OK;
    int rc = check_cache(c, what, cache, layer, false);
    if (rc == WF_OK) rc = check_queries(c, what, a->q_dev, a->out_dev, a->q_stride, a->tokens, a->seqs, a->q_heads, cache);
    if (rc != WF_OK) return rc;
    if (!a->tables_dev || !a->context_dev || (a->tables_dev | a->context_dev | a->q_offsets_dev) & 3 || a->ancestors_dev & 7)
        return set_error(c, WF_ERR_INVALID_ARGUMENT, "%s: tables and context are 4-byte aligned device arrays, ancestors 8-byte aligned", what);
    if (a->max_drafts < 1 || a->max_drafts > TREE_MAX_DRAFTS) return set_error(c, WF_ERR_TOO_LARGE, "%s: max_drafts %d is not 1 .. %d", what, a->max_drafts, TREE_MAX_DRAFTS);
    if (!a->q_offsets_dev && a->tokens != (int64_t)a->seqs * a->max_drafts)
        return set_error(c, WF_ERR_SHAPE, "%s: %lld tokens are not %d for each of %d sequences", what, (long long)a->tokens, a->max_drafts, a->seqs);
    if (a->table_stride < 1 || a->table_stride > (1LL << 31) / cache->page_tokens - 1 || a->max_context < 0 || a->max_context > (1LL << 31) - 1024)
        return set_error(c, WF_ERR_SHAPE, "%s: table_stride %lld, max_context %lld", what, (long long)a->table_stride, (long long)a->max_context);
    if (!(a->scale > 0.f) || a->scale > 1e30f) return set_error(c, WF_ERR_INVALID_ARGUMENT, "%s: scale %g", what, (double)a->scale);
    if (cache->pages < 1) return set_error(c, WF_ERR_SHAPE, "%s: a cache without pages", what);
    TreeParams p{};
    p.cache = cache_layer(*cache, layer);
    p.q = reinterpret_cast<const bf16*>(a->q_dev);
    p.out = reinterpret_cast<bf16*>(a->out_dev);
    p.q_stride = a->q_stride;
    p.q_offsets = reinterpret_cast<const int*>(a->q_offsets_dev);
    p.tables = reinterpret_cast<const int*>(a->tables_dev);
    p.table_stride = a->table_stride;
    p.context = reinterpret_cast<const int*>(a->context_dev);
    p.ancestors = reinterpret_cast<const uint64_t*>(a->ancestors_dev);
    p.tokens = a->tokens;
    p.max_context = a->max_context;
    p.seqs = a->seqs;
    p.q_heads = a->q_heads;
    p.group = a->q_heads / cache->kv_heads;
    p.max_drafts = a->max_drafts;
    p.group_inverse = p.group == 1 ? 0 : (uint32_t)(((1ull << 32) + p.group - 1) / p.group);
    p.scale_log2 = a->scale * 1.44269504f;
    p.status = c->d_status;
    const int rows = a->max_drafts * p.group, chunks = dim_chunks(cache->head_dim);  // rows of a sequence and kv head
    // Tiles of 128 rows on the 5th-generation tensor cores, or of 16 or 32 on mma.sync.  48 sequences of 1500 tokens, 8 heads of 128, 20 / 24 / 32 rows: 71.5 / 72.3 / 73.2 us
    // against 65.1 / 66.1 / 67.8; 8 of 2000, 4 / 16 / 32 rows: 22.4 / 23.3 / 23.9 against 19.1 / 20.7 / 25.7; one of 600: 12.3 for all three against 9.5 / 10.1 / 13.4.  With more
    // than 32 rows a row's sums no longer fit in the registers of the warps that multiply.
    if (rows > 32) return chunks == 1 ? launch_wide_tree<1>(c, p, s) : launch_wide_tree<2>(c, p, s);
    if (chunks == 1) return rows <= 16 ? launch_tree<1, 1>(c, p, s) : launch_tree<1, 2>(c, p, s);
    return rows <= 16 ? launch_tree<2, 1>(c, p, s) : launch_tree<2, 2>(c, p, s);
}

}  // extern "C"
