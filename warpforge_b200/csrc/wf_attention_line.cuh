// How attention over a cache is cut over the SMs, and how the pieces are joined.
//
// A unit is a block of rows of one sequence and kv head; it reads so many tiles of keys.  All units form one line, a unit `unit_tiles` positions (for
// what it costs in any case) and a position for each tile; the line is cut into even shares, one a CTA.  Where units may be cut, a CTA's pieces
// of cut units go to memory and tree_join_kernel adds them up in the order of the line; where they may not, a unit belongs to the share that it begins in.
#pragma once
#include "wf_attention.cuh"

namespace wf {

// A cut unit, as the CTA that it begins in leaves it for tree_join_kernel.
struct alignas(16) TreeCut {
    int first_cta, last_cta;       // that have pieces of it; first_cta < 0: none begins in this CTA
    int row0, rows, context, seq;  // of the sequence
    int head, first, count;        // kv head; which of the sequence's rows * group, row by row
    int pad[3];
};
struct TreeCuts {
    TreeCut* cuts;      // [CTAs]
    float* pieces;      // [CTAs][2]: of a unit that began earlier, of one that begins here; rows, then their maxima, then their sums
    int piece_rows;     // that a piece has room for
    int tile_rows, tile_room;  // rows come in tiles of tile_rows, which have the room of tile_room
    int dim;            // floats of a row
    int may_cut;
};

// Whether units are cut, by what the host knows: how many there are and how many tiles the longest can have.  Cut, every CTA has the same share, but most
// have parts of two units, and a second kernel joins them; that costs as much as `worth` tiles.  Whole, some CTAs have a unit more than the average.  Where
// most sequences are shorter than the longest, whole units cost up to all of the longest one's tiles: from `anyway` tiles on, that is more than what cutting would
// cost where they are alike.
inline bool line_is_cut(int64_t units, int64_t tiles, int sms, int worth, int anyway) {
    const int64_t rounds = (units + sms - 1) / sms;
    return tiles > anyway || tiles * (rounds * sms - units) > (int64_t)worth * sms;
}

struct LineUnit {
    TreeSeq q;
    int seq, head, first;           // first: of the sequence's rows * group
    int from, to, tiles;            // tiles of the unit that lie in the share
    int first_cta, last_cta;        // whose shares have tiles of it
};

#ifdef __CUDACC__
// Walks the share of this CTA, the whole warp together: f(unit) for every unit that has tiles in it, until it answers false.
template <int KEYS, class F> __device__ __forceinline__ bool walk_line(const TreeParams& p, int unit_rows, int unit_tiles, bool may_cut, F f) {
    const int lane = threadIdx.x & 31, heads = p.cache.kv_heads, group = p.group;
    auto tiles_of = [&](const TreeSeq& q) { return max(1, (q.context + q.rows + KEYS - 1) / KEYS); };
    auto blocks_of = [&](const TreeSeq& q) { return (q.rows * group + unit_rows - 1) / unit_rows; };
    auto info = [&](int s) {
        TreeSeq q{};
        if (s < p.seqs) q = tree_seq(p, s);
        return q;
    };
    auto line_of = [&](const TreeSeq& q) { return q.rows == 0 ? 0 : (int64_t)(tiles_of(q) + unit_tiles) * (heads * blocks_of(q)); };
    // a lane has a sequence at a time
    TreeSeq mine = info(lane);
    int64_t line64 = line_of(mine), total64 = line64;
#pragma unroll 1
    for (int s0 = 32; s0 < p.seqs; s0 += 32) total64 += line_of(info(s0 + lane));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total64 += __shfl_xor_sync(0xFFFFFFFFu, total64, o);
    if (total64 >= (1LL << 31)) {  // 3e10 keys: no cache holds them, some table says so
        report_status(p.status, STATUS_BAD_INDEX);
        return true;
    }
    const int total = (int)total64, share = total / (int)gridDim.x, more = total - share * (int)gridDim.x;  // the first `more` CTAs have a position more
    const int begin = (int)blockIdx.x * share + min((int)blockIdx.x, more), end = begin + share + ((int)blockIdx.x < more);
    auto cta_of = [&](int x) { return x < more * (share + 1) ? x / (share + 1) : more + (x - more * (share + 1)) / share; };
    int at = 0;  // where the lanes' sequences begin on the line
#pragma unroll 1
    for (int s0 = 0; s0 < p.seqs && at < end; s0 += 32) {
        if (s0) {
            mine = info(s0 + lane);
            line64 = line_of(mine);
        }
        const int line = (int)line64;
        int up_to = line;  // of the sequences up to this lane's
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xFFFFFFFFu, up_to, o);
            if (lane >= o) up_to += v;
        }
        const int base = at;
        at += __shfl_sync(0xFFFFFFFFu, up_to, 31);
        uint32_t ours = __ballot_sync(0xFFFFFFFFu, line > 0 && base + up_to > begin && base + up_to - line < end);  // sequences that the share touches
#pragma unroll 1
        for (; ours; ours &= ours - 1) {
            const int l = __ffs(ours) - 1;
            LineUnit u;
            u.q.row0 = __shfl_sync(0xFFFFFFFFu, mine.row0, l);
            u.q.rows = __shfl_sync(0xFFFFFFFFu, mine.rows, l);
            u.q.context = __shfl_sync(0xFFFFFFFFu, mine.context, l);
            u.q.place.table = p.tables + (size_t)(s0 + l) * p.table_stride;
            u.q.place.first = 0;
            u.seq = s0 + l;
            u.tiles = tiles_of(u.q);
            const int start = base + __shfl_sync(0xFFFFFFFFu, up_to - line, l), blocks = blocks_of(u.q), length = u.tiles + unit_tiles;
            int unit = begin > start ? (begin - start) / length : 0;
#pragma unroll 1
            for (int u_at = start + unit * length; unit < blocks * heads && u_at < end; unit++, u_at += length) {
                if (may_cut) {
                    u.from = max(0, begin - u_at - unit_tiles);
                    u.to = min(u.tiles, end - u_at - unit_tiles);
                } else {
                    u.from = 0;
                    u.to = u_at >= begin ? u.tiles : 0;
                }
                if (u.to <= u.from) continue;
                u.head = unit / blocks;
                u.first = (unit - u.head * blocks) * unit_rows;
                const bool whole = u.from == 0 && u.to == u.tiles;
                u.first_cta = whole ? (int)blockIdx.x : cta_of(u_at + unit_tiles);
                u.last_cta = whole ? (int)blockIdx.x : cta_of(u_at + length - 1);
                if (!f(u)) return false;
            }
        }
    }
    return true;
}

// What a CTA leaves for tree_join_kernel: the unit that begins in its share and does not end there, if there is one.
__device__ __forceinline__ void leave_cut(const TreeCuts& c, const LineUnit& u, int count) {
    TreeCut& cut = c.cuts[blockIdx.x];
    cut.first_cta = u.first_cta, cut.last_cta = u.last_cta;
    cut.row0 = u.q.row0, cut.rows = u.q.rows, cut.context = u.q.context, cut.seq = u.seq;
    cut.head = u.head, cut.first = u.first, cut.count = count;
}

__device__ __forceinline__ float line_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The pieces of a cut unit added up, a warp a row, four elements a lane: out = sum_c 2^(m_c - m) o_c / sum_c 2^(m_c - m) l_c.  blockIdx.x: the CTA that
// the unit begins in.  Bound by the latency of cut, pieces and row one after the other, and by how many rows an SM has at a time.  Pieces ahead 2 / 3 / 4 / 5 / 8: 13.3 / 12.5 /
// 12.4 / 13.0 / 12.8 us for one token of 32 heads at 2000 tokens (the kernel before it included), 25.2 / 22.8 / 22.0 / 23.1 / 23.0 of 8 heads at 20,000, 22.4 / 21.6 / 22.0 /
// 21.8 / 22.9 for 8 sequences of 0 to 3000 with up to 24 drafts; CTAs of 2 / 8 / 16 warps, the last of these: 24.5 / 22.3 / 22.9.
constexpr int JOIN_WARPS = 4, JOIN_AHEAD = 4;
__global__ void __launch_bounds__(JOIN_WARPS * 32) tree_join_kernel(const __grid_constant__ TreeParams p, const __grid_constant__ TreeCuts c) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const TreeCut cut = c.cuts[blockIdx.x];
    const int lane = threadIdx.x & 31, row = blockIdx.y * JOIN_WARPS + (threadIdx.x >> 5);
    if (cut.first_cta < 0 || row >= cut.count) return;
    const int tile = row / c.tile_rows, at = tile * c.tile_room + row - tile * c.tile_rows, piece_floats = c.piece_rows * (c.dim + 2);
    const bool mine = 4 * lane < c.dim;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    float top = -INFINITY, sum = 0.f;
    for (int c0 = cut.first_cta; c0 <= cut.last_cta; c0 += JOIN_AHEAD) {
        float4 v[JOIN_AHEAD];
        float m[JOIN_AHEAD], l[JOIN_AHEAD];
#pragma unroll
        for (int i = 0; i < JOIN_AHEAD; i++) {
            const bool real = c0 + i <= cut.last_cta;
            const float* from = c.pieces + ((size_t)(c0 + i) * 2 + (c0 + i == cut.first_cta)) * piece_floats;
            v[i] = real && mine ? ld_once(reinterpret_cast<const float4*>(from + (size_t)at * c.dim) + lane) : make_float4(0.f, 0.f, 0.f, 0.f);
            m[i] = real ? ld_once(from + c.piece_rows * c.dim + at) : -INFINITY;
            l[i] = real ? ld_once(from + c.piece_rows * (c.dim + 1) + at) : 0.f;
        }
        float grown = top;
#pragma unroll
        for (int i = 0; i < JOIN_AHEAD; i++) grown = fmaxf(grown, m[i]);
        const float ref = grown == -INFINITY ? 0.f : grown, keep = line_ex2((top - ref) * p.scale_log2);
        top = grown;
        sum *= keep;
        x.x *= keep, x.y *= keep, x.z *= keep, x.w *= keep;
#pragma unroll
        for (int i = 0; i < JOIN_AHEAD; i++) {
            const float take = line_ex2((m[i] - ref) * p.scale_log2);
            sum += l[i] * take;
            x.x += v[i].x * take, x.y += v[i].y * take, x.z += v[i].z * take, x.w += v[i].w * take;
        }
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int d = p.cache.dim, token = p.token_of(cut.first + row), head = cut.head * p.group + cut.first + row - token * p.group;
    bf16* const to = p.out + ((size_t)(cut.row0 + token) * p.q_heads + head) * d;
    if (4 * lane < d) *reinterpret_cast<uint2*>(to + 4 * lane) = make_uint2(pack_bf16(x.x * inv, x.y * inv), pack_bf16(x.z * inv, x.w * inv));
    // Key by key where an Inf or a NaN may have come from a key that the row does not see, or from a page that is not in the cache.
    const float largest = fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
    const bool odd = !(sum < INFINITY) || scores_too_large(top, p.scale_log2) || !(largest < INFINITY) || x.x != x.x || x.y != x.y || x.z != x.z || x.w != x.w;
    if (__any_sync(0xFFFFFFFFu, odd)) {
        KeyPlace place;
        place.table = p.tables + (size_t)cut.seq * p.table_stride;
        place.first = 0;
        attend_row(p.cache, place, p.q + (size_t)(cut.row0 + token) * p.q_stride + (size_t)head * d, to, cut.head, cut.context < 0 ? 0 : cut.context + cut.rows, p.scale_log2,
                   p.status, SeesAncestors{cut.context, ancestors_of(p, cut.row0 + token, token) & ((uint64_t)-1 >> (64 - cut.rows))});
    }
}
#endif

}  // namespace wf
