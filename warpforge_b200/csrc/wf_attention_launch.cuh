// What the entry points of attention share: checks, tensor maps, scratch, launches.
#pragma once
#include <algorithm>
#include <atomic>

#include "wf_attention_prompt.cuh"
#include "wf_attention_tree.cuh"

namespace wf {

inline int check_queries(Context* c, const char* what, int64_t q, int64_t out, int64_t q_stride, int64_t tokens, int seqs, int q_heads, const wf_kv_cache* cache) {
    if (!q || !out || (q | out) & 15) return set_error(c, WF_ERR_INVALID_ARGUMENT, "%s: q and out must be 16-byte aligned device addresses", what);
    if (tokens < 0 || tokens > (1LL << 31) - 1024 || seqs < 0 || seqs > (1LL << 31) - 1024 || q_heads < 1 || q_heads > 8192 || tokens * q_heads >= (1LL << 31))
        return set_error(c, WF_ERR_SHAPE, "%s: bad shape tokens=%lld seqs=%d q_heads=%d", what, (long long)tokens, seqs, q_heads);
    if (q_heads % cache->kv_heads) return set_error(c, WF_ERR_SHAPE, "%s: %d query heads over %d kv heads", what, q_heads, cache->kv_heads);
    if (q_heads / cache->kv_heads > 128) return set_error(c, WF_ERR_TOO_LARGE, "%s: more than 128 query heads for each kv head", what);
    if (q_stride < (int64_t)q_heads * cache->head_dim || q_stride % 8) return set_error(c, WF_ERR_SHAPE, "%s: q_stride %lld", what, (long long)q_stride);
    return WF_OK;
}
template <class... Params, class... Args>
inline int launch_attention(Context* c, const char* what, void (*kernel)(Params...), dim3 grid, unsigned threads, size_t smem, cudaStream_t s, const Args&... args) {
    return launch_clusters(c, what, kernel, grid, threads, 1, smem, s, args...);
}

// bf16 [z][y][x] with the given distances (elements) between y and z; boxes of 64 elements x by x bz, 128-byte swizzle, zeros outside
inline int encode_rows(Context* c, CUtensorMap* map, const void* base, int64_t x, int64_t y, int64_t z, int64_t y_apart, int64_t z_apart, int by, int bz) {
    const cuuint64_t dims[3] = {(cuuint64_t)x, (cuuint64_t)y, (cuuint64_t)z}, strides[2] = {(cuuint64_t)y_apart * 2, (cuuint64_t)z_apart * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)by, (cuuint32_t)bz}, step[3] = {1, 1, 1};
    const EncodeTiledFn encode = encode_tiled_fn();
    if (!encode) return set_error(c, WF_ERR_NO_DEVICE, "the driver has no cuTensorMapEncodeTiled");
    const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_error(c, WF_ERR_CUDA_BASE + (int)cudaErrorInvalidValue, "cuTensorMapEncodeTiled failed: %d", (int)r);
    return WF_OK;
}
inline int encode_cache(Context* c, CUtensorMap* map, const bf16* base, const CacheView& v, int box_rows) {
    if (v.page_shift == 0) return encode_rows(c, map, base, v.dim, v.kv_heads, v.pages, v.dim, (int64_t)v.kv_heads * v.dim, 1, box_rows);
    return encode_rows(c, map, base, v.dim, 1, (v.pages * v.kv_heads) << v.page_shift, v.dim, v.dim, 1, box_rows);
}
inline bool rows_of_sectors(const bf16* out, int dim) { return reinterpret_cast<uintptr_t>(out) % 32 == 0 && dim % 16 == 0; }
inline int dim_chunks(int dim) { return (dim + 63) / 64; }

// Where the pieces of cut units go; `extra` bytes behind them, whose address *more is.
inline int tree_scratch(Context* c, cudaStream_t s, int64_t ctas, int64_t floats, TreeCuts* cuts, int64_t extra = 0, uint8_t** more = nullptr) {
    GemvScratch& scratch = c->gemv_scratch[s];
    const int64_t head = (ctas * (int64_t)sizeof(TreeCut) + 255) & ~255LL, pieces = head + ((floats * (int64_t)sizeof(float) + 255) & ~255LL), bytes = pieces + extra;
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
    if (more) *more = scratch.d_attn.get() + pieces;
    return WF_OK;
}
template <int KIND, bool PARTS> inline int launch_join(Context* c, const TreeParams& p, const TreeCuts& cuts, unsigned ctas, int rows, cudaStream_t s) {
    return launch_attention(c, "tree_attention", tree_join_kernel<KIND, PARTS>, dim3(ctas, (unsigned)((rows + JOIN_WARPS - 1) / JOIN_WARPS)), JOIN_WARPS * 32, 0, s, p, cuts);
}
// The kernel for few rows, units on a line.  units: sequences (lists) times heads, with up to unit_rows rows and unit_keys keys each.
template <int CHUNKS, int MT, int KIND> inline int launch_tree(Context* c, const TreeParams& p, int64_t units, int unit_rows, int64_t unit_keys, cudaStream_t s) {
    const char* what = "tree_attention";
    typedef TreeShape<CHUNKS, MT> Shape;
    static std::atomic<uint64_t> ready{0};  // devices whose attribute is set
    if (!(ready.load() >> (c->device & 63) & 1)) {
        WF_CUDA(c, cudaFuncSetAttribute(tree_tiles_kernel<CHUNKS, MT, KIND>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::SMEM));
        ready.fetch_or(1ull << (c->device & 63));
    }
    const int64_t tiles = (unit_keys + TA_KEYS - 1) / TA_KEYS;
    units *= (unit_rows + Shape::ROWS - 1) / Shape::ROWS;
    // every list is a tile on the line, and what a unit costs beside it
    if (KIND == ATTEND_LISTS && units * (1 + Shape::UNIT_TILES) >= 1LL << 31) return set_error(c, WF_ERR_TOO_LARGE, "%s: %lld lists, rows %d at a time", what, (long long)units, Shape::ROWS);
    TreeTiles t{};
    t.p = p;
    t.c.may_cut = line_is_cut(units, tiles, c->sm_count, TA_CUT_TILES, TA_CUT_ANYWAY);
    t.c.piece_rows = t.c.tile_rows = t.c.tile_room = Shape::ROWS;
    t.c.dim = Shape::DIM;
    int rc = tree_scratch(c, s, c->sm_count, t.c.may_cut ? (int64_t)c->sm_count * 2 * Shape::PIECE : 0, &t.c);
    CUtensorMap k, v;
    if (rc == WF_OK) rc = encode_cache(c, &k, p.cache.keys, p.cache, TA_KEYS);
    if (rc == WF_OK) rc = encode_cache(c, &v, p.cache.values, p.cache, TA_KEYS);
    if (rc != WF_OK) return rc;
    const int64_t most = t.c.may_cut ? std::min<int64_t>(units, c->sm_count) * tiles : units;  // CTAs that can have work
    const unsigned grid = (unsigned)std::min<int64_t>(most, c->sm_count);
    rc = launch_attention(c, what, tree_tiles_kernel<CHUNKS, MT, KIND>, grid, Shape::THREADS, (size_t)Shape::SMEM, s, t, k, v);
    return rc == WF_OK && t.c.may_cut ? launch_join<KIND, false>(c, p, t.c, grid, Shape::ROWS, s) : rc;
}
// Units by number, each in a CTA or a cluster.  CTAS of an SM.
template <int CHUNKS, int MT, int KIND, int CTAS, bool CLUSTER> inline int launch_numbered(Context* c, const TreeParams& p, int64_t units, int parts, int64_t blocks, cudaStream_t s) {
    typedef TreeShape<CHUNKS, MT, CTAS> Shape;
    auto* const kernel = tree_tiles_kernel<CHUNKS, MT, KIND, CTAS, true, CLUSTER>;
    static std::atomic<uint64_t> ready{0};  // devices whose attribute is set
    if (!(ready.load() >> (c->device & 63) & 1)) {
        WF_CUDA(c, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::SMEM));
        ready.fetch_or(1ull << (c->device & 63));
    }
    TreeTiles t{};
    t.p = p;
    t.c.blocks = (int)blocks;
    t.c.units = (int)units;
    t.c.parts = parts;
    CUtensorMap k, v;
    int rc = encode_cache(c, &k, p.cache.keys, p.cache, TA_KEYS);
    if (rc == WF_OK) rc = encode_cache(c, &v, p.cache.values, p.cache, TA_KEYS);
    if (rc != WF_OK) return rc;
    const unsigned grid = CLUSTER ? (unsigned)(units * parts) : (unsigned)std::min<int64_t>(units, c->sm_count * CTAS);
    return launch_clusters(c, "tree_attention", kernel, dim3(grid), Shape::THREADS, (unsigned)parts, (size_t)Shape::SMEM, s, t, k, v);
}
// Clusters of so many CTAs that the device has at a time.
template <int CHUNKS, int MT, int KIND, int CTAS> inline int clusters_at_once(Context* c, int size) {
    typedef TreeShape<CHUNKS, MT, CTAS> Shape;
    static std::atomic<int> known[64][MAX_CLUSTER + 1];  // and one more; 0: not asked
    std::atomic<int>& held = known[c->device & 63][size];
    if (held.load() == 0) {
        auto* const kernel = tree_tiles_kernel<CHUNKS, MT, KIND, CTAS, true, true>;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)size * 1024);
        cfg.blockDim = dim3(Shape::THREADS);
        cfg.dynamicSmemBytes = Shape::SMEM;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = (unsigned)size;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        int n = 0;
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::SMEM) != cudaSuccess || cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
            n = 0;
            cudaGetLastError();
        }
        held.store(n + 1);
    }
    return held.load() - 1;
}
// How units with few rows go to the SMs.  Up to one an SM, the parts of a unit go to a cluster of large CTAs, as many as let all units be there at once; then to clusters of small CTAs; then
// each to a small CTA of its own.  An SM has three of them (a fourth where that spares a second round of units); where there are more and they are long, large CTAs share a line of them, since of
// units that a CTA takes one after the other two may be long.  Microseconds for lists of 256 / 4096 keys, 32 / 8 heads of 128, on the line and in clusters: 8 units 7.0 / 12.6 and 6.6 / 9.2
// (clusters of 8), 24 7.1 / 16.6 and 6.8 / 14.3 (4), 72 8.4 / 34 and 6.9 / 28.6 (2), 128 9.1 / 53 and 8.0 / 46.6 (4 small), 192 14.1 / 73 and 8.8 / 66 (2 small).  Of 256 / 2048 keys, with four
// small CTAs and with three: 352 units 13.2 / 63 and 12.3 / 61, 480 15.9 / 79 and 20.2 / 102, 576 17.6 / 94 and 21 / 105, 640 24.2 / 130 and 21.4 / 109, 1200 35 / 209 and 31 / 193 (36 / 215 on the line for
// 640 of 256 / 4096 keys).  800 units of 2560, 4096 keys, alike: 177, 267 on the line, 161, 248 in threes; 640 of 200 to 6000: 158 and 177; 800, most of 30 keys, one in eight of 6000: 77 and 185.
// Of 17 to 32 rows an SM would have two small CTAs, and the line is quicker: 80 units of 2048 keys 27.9 against 33, 192 49 against 69.
template <int CHUNKS, int MT, int KIND> inline int launch_units(Context* c, const TreeParams& p, int64_t units, int unit_rows, int64_t unit_keys, cudaStream_t s) {
    const int64_t blocks = (unit_rows + 16 * MT - 1) / (16 * MT), all = units * blocks, tiles = (unit_keys + TA_KEYS - 1) / TA_KEYS;
    if (units < UNIT_ITEMS && unit_keys < UNIT_KEYS) {
        for (int parts = MAX_CLUSTER; parts > 1; parts /= 2)
            if (tiles >= 8 * parts && all <= clusters_at_once<CHUNKS, MT, KIND, 1>(c, parts)) return launch_numbered<CHUNKS, MT, KIND, 1, true>(c, p, all, parts, blocks, s);
        if constexpr (MT == 1) {
            for (int parts = MAX_CLUSTER / 2; parts > 1; parts--)
                if (tiles >= 4 * parts) {
                    if (all <= clusters_at_once<CHUNKS, MT, KIND, 3>(c, parts)) return launch_numbered<CHUNKS, MT, KIND, 3, true>(c, p, all, parts, blocks, s);
                    if (all <= clusters_at_once<CHUNKS, MT, KIND, 4>(c, parts)) return launch_numbered<CHUNKS, MT, KIND, 4, true>(c, p, all, parts, blocks, s);
                }
            if (all > c->sm_count * 3 && all <= c->sm_count * 4) return launch_numbered<CHUNKS, MT, KIND, 4, false>(c, p, all, 1, blocks, s);
            if (all <= c->sm_count * 3 || tiles <= 128) return launch_numbered<CHUNKS, MT, KIND, 3, false>(c, p, all, 1, blocks, s);
        }
    }
    return launch_tree<CHUNKS, MT, KIND>(c, p, units, unit_rows, unit_keys, s);
}

// The prompt kernel on the rows of trees.
// units: sequences (groups) times heads, with up to unit_tokens tokens and unit_keys keys each.
template <int CHUNKS, int KIND> inline int launch_wide_tree(Context* c, const TreeParams& p, int64_t units, int64_t unit_tokens, int64_t unit_keys, cudaStream_t s) {
    static std::atomic<uint64_t> ready{0};  // devices whose attribute is set
    if (!(ready.load() >> (c->device & 63) & 1)) {
        WF_CUDA(c, cudaFuncSetAttribute(prompt_tiles_kernel<CHUNKS, KIND>, cudaFuncAttributeMaxDynamicSharedMemorySize, PromptShape<CHUNKS>::SMEM));
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
    const int64_t tiles = (unit_keys + PA_KEYS - 1) / PA_KEYS;
    // groups: all of their tokens are p.tokens, and each may have a block that is not full
    if (KIND == ATTEND_PREFIX) units += p.tokens / (2 * t.tile_tokens) * p.cache.kv_heads;
    else units *= (unit_tokens + 2 * t.tile_tokens - 1) / (2 * t.tile_tokens);
    constexpr bool PREFIX = KIND == ATTEND_PREFIX;
    // a prefix is cut where there are fewer units than half of the CTAs' rounds; `cuts` has an entry for each unit, a piece a place for each CTA and round
    t.c.may_cut = PREFIX ? tiles > 1 && units <= (PREFIX_ROUNDS - 1) * c->sm_count : line_is_cut(units, tiles, c->sm_count, PA_CUT_TILES, PA_CUT_ANYWAY);
    t.c.units = (int)std::min<int64_t>(units, (PREFIX_ROUNDS - 1) * c->sm_count);
    const int places = PREFIX ? PREFIX_ROUNDS * c->sm_count : 2 * c->sm_count;
    t.c.piece_rows = unit_tokens <= t.tile_tokens ? PA_ROWS : 2 * PA_ROWS;
    t.c.tile_rows = t.tile_tokens * p.group;
    t.c.tile_room = PA_ROWS;
    t.c.dim = CHUNKS * 64;
    int rc = tree_scratch(c, s, 2 * c->sm_count, t.c.may_cut ? (int64_t)places * t.c.piece_rows * (t.c.dim + 2) : 0, &t.c);
    CUtensorMap q, k, v;
    if (rc == WF_OK) rc = encode_rows(c, &q, p.q, p.cache.dim, p.q_heads, p.tokens, p.cache.dim, p.q_stride, p.group, t.tile_tokens);
    if (rc == WF_OK) rc = encode_cache(c, &k, p.cache.keys, p.cache, t.box_rows);
    if (rc == WF_OK) rc = encode_cache(c, &v, p.cache.values, p.cache, t.box_rows);
    if (rc != WF_OK) return rc;
    const int64_t most = t.c.may_cut ? std::min<int64_t>(units, c->sm_count) * tiles : units;  // CTAs that can have work
    const unsigned grid = (unsigned)std::min<int64_t>(most, c->sm_count);
    rc = launch_attention(c, "tree_attention", prompt_tiles_kernel<CHUNKS, KIND>, grid, PA_THREADS, (size_t)PromptShape<CHUNKS>::SMEM, s, t, q, k, v);
    return rc == WF_OK && t.c.may_cut ? launch_join<KIND, PREFIX>(c, p, t.c, PREFIX ? (unsigned)t.c.units : grid, (int)std::min<int64_t>(unit_tokens, 2 * t.tile_tokens) * p.group, s) : rc;
}

}  // namespace wf

#define ATTENTION_ENTER(ctxh)                                              \
    Context* c = get_context(ctxh);                                        \
    if (!c) return WF_ERR_INVALID_HANDLE;                                  \
    ScopedLock _lk(c);                                                     \
    if (!_lk.ok) return WF_ERR_BUSY;                                       \
    WF_CUDA(c, cudaSetDevice(c->device));                                  \
    cudaStream_t s = resolve_stream(c, stream)
