// Attention that reads less than every key of every sequence: wf_selected_attention (lists of pages for each token and kv head) and wf_shared_prefix_attention (sequences
// that have a prefix in common).  The kernels are those of wf_tree_attention; what a unit is, and what becomes of its rows' sums, is theirs by kind.
//
//   out = softmax(scale q k^T) v, the keys taken in parts: o = sum_t 2^(s_t - m) v_t, l = sum_t 2^(s_t - m) of each, and
//   out = sum_parts 2^(m_part - m) o_part / sum_parts 2^(m_part - m) l_part      m the largest of the parts' maxima
#include "wf_attention_launch.cuh"

using namespace wf;

static int check_attention(Context* c, const char* what, const wf_kv_cache* cache, int layer, int64_t q, int64_t out, int64_t q_stride, int64_t tokens, int seqs, int q_heads, float scale) {
    int rc = check_kv_cache(c, what, cache, layer, false);
    if (rc == WF_OK) rc = check_queries(c, what, q, out, q_stride, tokens, seqs, q_heads, cache);
    if (rc != WF_OK) return rc;
    if (!(scale > 0.f) || scale > 1e30f) return set_error(c, WF_ERR_INVALID_ARGUMENT, "%s: scale %g", what, (double)scale);
    if (cache->pages < 1) return set_error(c, WF_ERR_SHAPE, "%s: a cache without pages", what);
    return WF_OK;
}
static TreeParams attention_params(Context* c, const wf_kv_cache& cache, int layer, int64_t q, int64_t out, int64_t q_stride, int64_t tokens, int q_heads, float scale) {
    TreeParams p{};
    p.cache = cache_layer(cache, layer);
    p.q = reinterpret_cast<const bf16*>(q);
    p.out = reinterpret_cast<bf16*>(out);
    p.q_stride = q_stride;
    p.tokens = tokens;
    p.q_heads = q_heads;
    p.group = q_heads / cache.kv_heads;
    p.group_inverse = p.group == 1 ? 0 : (uint32_t)(((1ull << 32) + p.group - 1) / p.group);
    p.scale_log2 = scale * 1.44269504f;
    p.status = c->d_status;
    return p;
}

// Lists.  More than 32 heads of a group are taken 32 at a time.  Many lists go to small CTAs by number, up to one an SM to large ones that share them out evenly.  Microseconds of the
// large / the small, 32 / 8 heads of 128, lists of 256, 1024, 4096 keys: 8 lists 6.9 / 10.2, 11.0 / 10.2, 12.6 / 16.8; 128 9.3 / 10.2, 18.3 / 19.4, 53 / 50; 160 13.2 / 10.7, 25.8 / 22.0,
// 64 / 59; 384 23.5 / 13.7, 45.8 / 36.6, 133 / 125; 800 44 / 26, 88 / 75, 264 / 262.
template <int CHUNKS> static int launch_lists(Context* c, const TreeParams& p, cudaStream_t s) {
    const int64_t units = p.tokens * p.cache.kv_heads, keys = p.table_stride << p.cache.page_shift;
    if (units * ((p.group + 31) / 32) > c->sm_count && units < UNIT_ITEMS && keys < UNIT_KEYS)
        return p.group <= 16 ? launch_tree<CHUNKS, 1, ATTEND_LISTS, TA_FEW_WARPS>(c, p, units, p.group, keys, s) : launch_tree<CHUNKS, 2, ATTEND_LISTS, TA_FEW_WARPS>(c, p, units, p.group, keys, s);
    return p.group <= 16 ? launch_tree<CHUNKS, 1, ATTEND_LISTS>(c, p, units, p.group, keys, s) : launch_tree<CHUNKS, 2, ATTEND_LISTS>(c, p, units, p.group, keys, s);
}

// Prefixes, then what the sequences have of their own, which begins with the first one's sums.
template <int CHUNKS> static int launch_shared(Context* c, TreeParams p, cudaStream_t s) {
    const int64_t rows = p.tokens * p.q_heads, sums = (rows * (CHUNKS * 64 + 2) * (int64_t)sizeof(float) + 255) & ~255LL;
    // the most cut units and pieces of them that any of the kernels leaves (16: CTAs of an SM times rounds)
    const int64_t most_cuts = 16 * c->sm_count, pieces = (int64_t)c->sm_count * PREFIX_ROUNDS * 2 * PA_ROWS * (CHUNKS * 64 + 2);
    static_assert(4 * UNIT_ROUNDS <= 16 && UNIT_PLACES * 4 * 16 <= PREFIX_ROUNDS * 2 * PA_ROWS, "pieces of small CTAs");
    TreeCuts cuts{};
    uint8_t* more = nullptr;
    int rc = tree_scratch(c, s, most_cuts, pieces, &cuts, sums + p.seqs * (int64_t)sizeof(int2), &more);
    if (rc != WF_OK) return rc;
    p.state = reinterpret_cast<float*>(more);
    p.state_dim = CHUNKS * 64;
    p.prefix_of = reinterpret_cast<int2*>(more + sums);
    rc = launch_wide_tree<CHUNKS, ATTEND_PREFIX>(c, p, (int64_t)p.n_groups * p.cache.kv_heads, p.tokens, p.max_prefix, s);
    if (rc != WF_OK) return rc;
    const int64_t units = (int64_t)p.seqs * p.cache.kv_heads, keys = p.max_context + p.max_drafts;
    const int unit_rows = p.max_drafts * p.group;
    // Tiles of 128 rows where sequences have more than 32; where only the longest of them do, 32 at a time.  Microseconds of the call, tiles of 128 / of 32: 17 sequences with 1 to 12 tokens of
    // 24 / 8 heads of 64 48 / 39; 4, 16, 48 with 12 tokens of 32 / 8 heads of 128 and 400 keys 29.8 / 28.7, 38 / 43, 66 / 85.
    if (unit_rows > 32 && p.tokens * p.group > 20 * (int64_t)p.seqs) return launch_wide_tree<CHUNKS, ATTEND_OWN>(c, p, units, p.max_drafts, keys, s);
    // Small CTAs for many sequences with few rows.  Large / small, one token of 32 / 8 heads of 128 behind 512 in common: 128 units of 50, 400, 2000 keys 18.9 / 18.5, 22.6 / 25.4, 41 / 40; 384 27.9 /
    // 22.8, 37 / 34, 82 / 81; with 20 rows (two small CTAs an SM) 384 43 / 39, 53 / 56, 93 / 136.
    if (unit_rows <= 16 && 2 * units >= 5 * c->sm_count && units < UNIT_ITEMS && keys < UNIT_KEYS) return launch_tree<CHUNKS, 1, ATTEND_OWN, TA_FEW_WARPS>(c, p, units, unit_rows, keys, s);
    return unit_rows <= 16 ? launch_tree<CHUNKS, 1, ATTEND_OWN>(c, p, units, unit_rows, keys, s) : launch_tree<CHUNKS, 2, ATTEND_OWN>(c, p, units, unit_rows, keys, s);
}

extern "C" {

int wf_selected_attention(int64_t ctx, const wf_selected_attention_args* a, const wf_kv_cache* cache, int layer, int64_t stream) {
    ATTENTION_ENTER(ctx);
    const char* what = "selected_attention";
    if (!a || !cache) return set_error(c, WF_ERR_INVALID_ARGUMENT, "%s: null arguments", what);
    if (a->tokens == 0) return WF_OK;
    const int rc = check_attention(c, what, cache, layer, a->q_dev, a->out_dev, a->q_stride, a->tokens, 0, a->q_heads, a->scale);
    if (rc != WF_OK) return rc;
    if (!a->pages_dev || !a->lens_dev || a->pages_dev & 3 || (a->lens_dev | a->ancestors_dev) & 7)
        return set_error(c, WF_ERR_INVALID_ARGUMENT, "%s: pages is a 4-byte aligned device array, lens and ancestors 8-byte aligned ones", what);
    if (a->width < 1 || a->width > (1LL << 31) / cache->page_tokens - 1) return set_error(c, WF_ERR_SHAPE, "%s: width %d", what, a->width);
    TreeParams p = attention_params(c, *cache, layer, a->q_dev, a->out_dev, a->q_stride, a->tokens, a->q_heads, a->scale);
    p.tables = reinterpret_cast<const int*>(a->pages_dev);
    p.table_stride = a->width;
    p.lens = reinterpret_cast<const int2*>(a->lens_dev);
    p.ancestors = reinterpret_cast<const uint64_t*>(a->ancestors_dev);
    return dim_chunks(cache->head_dim) == 1 ? launch_lists<1>(c, p, s) : launch_lists<2>(c, p, s);
}

int wf_shared_prefix_attention(int64_t ctx, const wf_shared_prefix_attention_args* a, const wf_kv_cache* cache, int layer, int64_t stream) {
    ATTENTION_ENTER(ctx);
    const char* what = "shared_prefix_attention";
    if (!a || !cache) return set_error(c, WF_ERR_INVALID_ARGUMENT, "%s: null arguments", what);
    if (a->tokens == 0 || a->seqs == 0) return WF_OK;
    const int rc = check_attention(c, what, cache, layer, a->q_dev, a->out_dev, a->q_stride, a->tokens, a->seqs, a->q_heads, a->scale);
    if (rc != WF_OK) return rc;
    if (a->n_groups < 1 || a->n_groups > a->seqs) return set_error(c, WF_ERR_SHAPE, "%s: %d groups of %d sequences", what, a->n_groups, a->seqs);
    if (!a->tables_dev || !a->context_dev || !a->groups_dev || !a->prefix_dev || (a->tables_dev | a->context_dev | a->q_offsets_dev | a->groups_dev | a->prefix_dev) & 3 ||
        a->ancestors_dev & 7)
        return set_error(c, WF_ERR_INVALID_ARGUMENT, "%s: tables, context, groups and prefix are 4-byte aligned device arrays, ancestors 8-byte aligned", what);
    if (a->max_drafts < 1 || a->max_drafts > TREE_MAX_DRAFTS) return set_error(c, WF_ERR_TOO_LARGE, "%s: max_drafts %d is not 1 .. %d", what, a->max_drafts, TREE_MAX_DRAFTS);
    if (!a->q_offsets_dev && a->tokens != (int64_t)a->seqs * a->max_drafts)
        return set_error(c, WF_ERR_SHAPE, "%s: %lld tokens are not %d for each of %d sequences", what, (long long)a->tokens, a->max_drafts, a->seqs);
    if (a->tokens > WF_SHARED_MAX_TOKENS) return set_error(c, WF_ERR_TOO_LARGE, "%s: %lld tokens, at most %d", what, (long long)a->tokens, WF_SHARED_MAX_TOKENS);
    if (a->table_stride < 1 || a->table_stride > (1LL << 31) / cache->page_tokens - 1 || a->max_prefix < 0 || a->max_prefix > 1LL << 28 || a->max_own < 0 ||
        a->max_own > (1LL << 31) - 1024)
        return set_error(c, WF_ERR_SHAPE, "%s: table_stride %lld, max_prefix %lld, max_own %lld", what, (long long)a->table_stride, (long long)a->max_prefix, (long long)a->max_own);
    TreeParams p = attention_params(c, *cache, layer, a->q_dev, a->out_dev, a->q_stride, a->tokens, a->q_heads, a->scale);
    p.q_offsets = reinterpret_cast<const int*>(a->q_offsets_dev);
    p.tables = reinterpret_cast<const int*>(a->tables_dev);
    p.table_stride = a->table_stride;
    p.context = reinterpret_cast<const int*>(a->context_dev);
    p.ancestors = reinterpret_cast<const uint64_t*>(a->ancestors_dev);
    p.groups = reinterpret_cast<const int*>(a->groups_dev);
    p.prefix = reinterpret_cast<const int*>(a->prefix_dev);
    p.max_context = a->max_own;
    p.max_prefix = a->max_prefix;
    p.seqs = a->seqs;
    p.n_groups = a->n_groups;
    p.max_drafts = a->max_drafts;
    return dim_chunks(cache->head_dim) == 1 ? launch_shared<1>(c, p, s) : launch_shared<2>(c, p, s);
}

}  // extern "C"
