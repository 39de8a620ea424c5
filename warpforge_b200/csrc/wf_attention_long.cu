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

// What rows, 16 at a time in small CTAs, take of an SM: in tiles of 16 keys, eight more for what a block of rows costs in any case.
static double share_of_rows(const Context* c, int64_t units, int64_t rows, int64_t keys) { return (double)units * ((rows + 15) / 16) * ((keys + TA_KEYS - 1) / TA_KEYS + 8) / c->sm_count; }

// Units of more than 16 rows, 16 or 32 of them at a time.  16 read the keys twice as often, out of the L2, but go to clusters and to small CTAs of their own; where that is much, a line is quicker, and where
// units are long and not alike (lists are), too.  Microseconds 32 / 16 at a time: lists of 512, 2048, 4096 keys, 64 heads of 128 for one kv head, one token (share of an SM: 1 to 7) 9.9 / 7.5, 11.5 / 8.7,
// 13.5 / 9.9; 8 (9, 29, 57) 10.2 / 7.8, 13.2 / 9.7, 17.0 / 12.6; 32 (35, 118, 228) 11.5 / 10.4, 17.8 / 18.3, 25.4 / 28.6; 96 (104, 353, 685) 24.3 / 16.2, 44.6 / 41.3, 69 / 74; 256 (277, 941, 1827)
// 48 / 41, 102 / 113, 177 / 331; 40 / 2 heads, 96 tokens (104, 353, 685) 27.6 / 16.8, 48.3 / 43.3, 76.6 / 77.2.  17 sequences of 1 to 1777 keys of their own, 36 rows of 8 heads (331): 39.7 / 47.3.
constexpr double SHARE_LITTLE = 60, SHARE_OF_SHORT = 600;
template <int CHUNKS, int KIND> static int launch_rows(Context* c, const TreeParams& p, int64_t units, int64_t rows, int64_t keys, cudaStream_t s) {
    const double share = share_of_rows(c, units, rows, keys);
    const bool sixteen = rows <= 16 || share <= SHARE_LITTLE || (keys <= (KIND == ATTEND_LISTS ? 2048 : 512) && share <= SHARE_OF_SHORT);
    return sixteen ? launch_units<CHUNKS, 1, KIND>(c, p, units, (int)rows, keys, s) : launch_units<CHUNKS, 2, KIND>(c, p, units, (int)rows, keys, s);
}

// Tiles of 128 rows where sequences have more than 32 each; where only the longest of them do, 32 at a time.  Microseconds of the call, tiles of 128 / of 32: 17 sequences with 1 to 12 tokens of 24 / 8
// heads of 64 48 / 39; 4, 16, 48 with 12 tokens of 32 / 8 heads of 128 and 400 keys 29.8 / 28.7, 38 / 43, 66 / 85.
static bool few_rows(const TreeParams& p) { return p.max_drafts * p.group <= 32 || p.tokens * p.group <= 20 * (int64_t)p.seqs; }
constexpr double AGAIN_BYTES = 270e6, AGAIN_FEW_BYTES = 110e6;
// More than 32 rows go 16 at a time, too, where that is little: the tiles of 128 rows wait longer for the little that they have to do.  Sequences behind a prefix of 4096, 32 / 8 heads of 128, own keys by
// 128 rows / by 16: 8 with 12 tokens and 20, 400, 1500 keys (share 13, 44, 133) 40.6 / 33.5, 43.2 / 38.5, 50.6 / 48.5; 24 with 20, 400 (39, 132) 59.0 / 45.8, 66.0 / 54.7; 48 with 20, 400, 1500 (78, 265, 800)
// 78.0 / 66.5, 90.8 / 87.8, 122 / 146.  With 24 tokens, 96 rows: 8 with 400 (91) 47.2 / 44.6; 24 with 100, 400 (125, 272) 72.3 / 71.5, 80.7 / 87.3; 48 with 20 (171) 109.5 / 111.6.
constexpr double SHARE_48_ROWS = 270, SHARE_MORE_ROWS = 110;
// Prefixes of more than 32 rows in all 16 rows at a time: one token each behind a prefix, tiles of 128 rows / 16 at a time.  32 / 8 heads of 128, 16 sequences behind 1024, 4096, 16384 (share 16, 57, 223)
// 20.1 / 14.5, 26.9 / 19.0, 34.7 / 35.9; 32 (31, 114, 446) 22.1 / 15.8, 28.3 / 24.2, 36.4 / 56.3; 64 (62, 228) 27.0 / 20.6, 32.4 / 34.0; 16 / 2 heads, 16 behind 4096, 16384 (29, 112) 24.7 / 18.4, 41.6 / 33.9.
constexpr double SHARE_OF_PREFIX = 140;
// Each sequence reads the prefix itself, in one kernel, by what that takes of an SM, where a prefix has more than 32 rows.  Microseconds by several kernels / by one.  Where the prefix is read 16 rows at a time, by
// its share and that: 32 / 8 heads of 128, 16 and 32 sequences behind 1024 (16, 68; 31, 135) 14.5 / 12.5, 15.8 / 17.4; 16 / 2 heads, 32 and 64 behind 4096 (57, 116; 114, 232) 18.7 / 17.5, 23.9 / 26.8.  Where it is
// not, sequences with more than 32 rows each (12 and 24 tokens): 32 behind 512 (244) 38.3 / 34.1; 4 behind 4096 (176, 353) 32.0 / 27.5, 35.8 / 47.6; 16 / 2 heads, 32 with 24 behind 512 (248) 38.6 / 34.9.
constexpr double SHARE_MORE_AGAIN = 80, SHARE_AGAIN = 280;

// Prefixes, then what the sequences have of their own, which begins with the first one's sums.
template <int CHUNKS> static int launch_shared(Context* c, TreeParams p, cudaStream_t s) {
    // Where little would be read again, most of it out of the L2, a sequence reads its prefix itself, and there is one kernel; less where a prefix has up to 32 rows in all, whose kernel is quick.  Microseconds
    // by several kernels / by one, one token each with 100 keys of its own, (sequences - groups) x prefix in MB: 64 / 8 heads of 128, 4 sequences behind 1024 in common (13) 15.6 / 8.6; 8 behind 8192 (235)
    // 31.7 / 29.3; 16 behind 4096, 8192 (252, 503) 29.9 / 27.3, 33.3 / 46.3; 64 behind 1024 (264) 30.3 / 29.7; 16 / 2 heads, 32 behind 8192 (260) 41.6 / 28.0; 32 / 8 heads, 64 behind 1024 (264) 28.8 / 28.9.  Up to 32
    // rows: 32 / 8 heads, 8 behind 4096, 8192 (117, 235) 19.7 / 18.0, 25.6 / 29.0; 32 / 32 heads, 4 behind 2048, 4096 (101, 201) 18.0 / 18.4, 24.1 / 28.4; 8 behind 512, 1024 (59, 117) 14.9 / 13.4, 15.9 / 18.6.
    const double again = (double)(p.seqs - p.n_groups) * (double)p.max_prefix * p.cache.kv_heads * p.cache.dim * 4;
    const int64_t units = (int64_t)p.seqs * p.cache.kv_heads, unit_rows = p.max_drafts * p.group, own_keys = p.max_context + p.max_drafts, all_keys = p.max_prefix + own_keys;
    const int64_t prefix_rows = p.tokens * p.group;
    const int64_t prefixes = (int64_t)p.n_groups * p.cache.kv_heads;
    const int64_t rows = p.tokens * p.q_heads, sums = (rows * (CHUNKS * 64 + 2) * (int64_t)sizeof(float) + 255) & ~255LL;
    const double share = share_of_rows(c, units, unit_rows, all_keys), share_of_prefix = share_of_rows(c, prefixes, prefix_rows, p.max_prefix);
    const bool sixteen = prefix_rows > 32 && share_of_prefix <= SHARE_OF_PREFIX;
    if (sixteen ? share <= SHARE_MORE_AGAIN + share_of_prefix : unit_rows > 32 && share <= SHARE_AGAIN) return launch_units<CHUNKS, 1, ATTEND_WHOLE>(c, p, units, (int)unit_rows, all_keys, s);
    if (!sixteen && again <= (prefix_rows > 32 ? AGAIN_BYTES : AGAIN_FEW_BYTES) && few_rows(p)) return launch_rows<CHUNKS, ATTEND_WHOLE>(c, p, units, unit_rows, all_keys, s);
    // more sums than a call may have: without any
    if (sums > ATTN_CALL_BYTES) return launch_rows<CHUNKS, ATTEND_WHOLE>(c, p, units, unit_rows, all_keys, s);
    // the most cut units and pieces of them that any of the kernels leaves
    const int64_t most_cuts = (PREFIX_ROUNDS - 1) * c->sm_count, pieces = (int64_t)c->sm_count * PREFIX_ROUNDS * 2 * PA_ROWS * (CHUNKS * 64 + 2);
    TreeCuts cuts{};
    uint8_t* more = nullptr;
    int rc = tree_scratch(c, s, most_cuts, pieces, &cuts, sums + p.seqs * (int64_t)sizeof(int2), &more);
    if (rc != WF_OK) return rc;
    p.state = reinterpret_cast<float*>(more);
    p.state_dim = CHUNKS * 64;
    p.prefix_of = reinterpret_cast<int2*>(more + sums);
    rc = sixteen             ? launch_units<CHUNKS, 1, ATTEND_PREFIX>(c, p, prefixes, (int)prefix_rows, p.max_prefix, s)
         : prefix_rows > 32 ? launch_wide_tree<CHUNKS, ATTEND_PREFIX>(c, p, prefixes, p.tokens, p.max_prefix, s)
                            : launch_rows<CHUNKS, ATTEND_PREFIX>(c, p, prefixes, prefix_rows, p.max_prefix, s);
    if (rc != WF_OK) return rc;
    if (unit_rows > 32 && share_of_rows(c, units, unit_rows, own_keys) <= (unit_rows <= 48 ? SHARE_48_ROWS : SHARE_MORE_ROWS))
        return launch_units<CHUNKS, 1, ATTEND_OWN>(c, p, units, (int)unit_rows, own_keys, s);
    return few_rows(p) ? launch_rows<CHUNKS, ATTEND_OWN>(c, p, units, unit_rows, own_keys, s) : launch_wide_tree<CHUNKS, ATTEND_OWN>(c, p, units, p.max_drafts, own_keys, s);
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
    // (more than 32 heads of a group are taken 32 at a time)
    const int64_t units = p.tokens * cache->kv_heads, keys = p.table_stride << p.cache.page_shift;
    return dim_chunks(cache->head_dim) == 1 ? launch_rows<1, ATTEND_LISTS>(c, p, units, p.group, keys, s) : launch_rows<2, ATTEND_LISTS>(c, p, units, p.group, keys, s);
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
