// How attention over a cache is cut over the SMs, and how the pieces are joined.
//
// A unit is a block of rows of one sequence and kv head; it reads so many tiles of keys.  Where units are few and of unequal length, all of them form one line, a unit `unit_tiles` positions (for
// what it costs in any case) and a position for each tile; the line is cut into even shares, one a CTA.  Where units may be cut, a CTA's pieces
// of cut units go to memory and tree_join_kernel adds them up in the order of the line; where they may not, a unit belongs to the share that it begins in.
// Where units go by number (walk_units), a CTA or a cluster finds its own without looking at the others, and a cluster's CTAs add their parts up among themselves.  Prefixes (walk_prefixes) are
// cut into parts of at most so many tiles, that many that all CTAs have one; each has a place in memory, and tree_join_kernel adds them up.
#pragma once
#include <algorithm>

#include "wf_attention.cuh"

namespace wf {

constexpr int MAX_CLUSTER = 8;
enum UnitWay { UNITS_ON_A_LINE, UNITS_BY_NUMBER, UNITS_IN_PARTS };
constexpr int64_t UNIT_ITEMS = 1 << 18, UNIT_KEYS = 1 << 27;  // sequences (lists) times heads, of which each may be four blocks of rows, and keys of one: their tiles are numbers for quick_div

// Parts of prefixes: as many as all CTAs have in so many rounds, at most.
constexpr int PREFIX_ROUNDS = 3;

// A cut unit, as the CTA that it begins in leaves it for tree_join_kernel.
struct alignas(16) TreeCut {
    int first_cta, last_cta;       // that have pieces of it; first_cta < 0: none begins in this CTA
    int row0, rows, context, seq;  // of the sequence
    int head, first, count;        // kv head; which of the sequence's rows * group, row by row
    int news;                      // of a list
    int pad[2];
};
struct TreeCuts {
    TreeCut* cuts;      // [CTAs]
    float* pieces;      // [CTAs][2]: of a unit that began earlier, of one that begins here; rows, then their maxima, then their sums
    int piece_rows;     // that a piece has room for
    int tile_rows, tile_room;  // rows come in tiles of tile_rows, which have the room of tile_room
    int dim;            // floats of a row
    int may_cut;
    int parts, blocks;  // units by number: parts of each (CTAs of a cluster), blocks of rows of a sequence and head
    int units;          // by number, how many; prefixes: that `cuts` has an entry for
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
    int unit, part;                 // prefixes: the unit, the place of this part's sums
};

#ifdef __CUDACC__
// Walks the share of this CTA, the whole warp together: f(unit) for every unit that has tiles in it, until it answers false.  none: there are more tiles than a line has, and no unit is walked.
template <int KEYS, int KIND, class F> __device__ __forceinline__ bool walk_share(const TreeParams& p, int unit_rows, int unit_tiles, bool may_cut, bool& none, F f) {
    // a list is a kv head's
    const int lane = threadIdx.x & 31, heads = KIND == ATTEND_LISTS ? 1 : p.cache.kv_heads, group = p.group;
    const int seqs = KIND == ATTEND_LISTS ? (int)p.tokens * p.cache.kv_heads : KIND == ATTEND_PREFIX ? p.n_groups : p.seqs;
    auto tiles_of = [&](const TreeSeq& q) { return max(1, (KIND == ATTEND_TREE ? q.context + q.rows + KEYS - 1 : keys_of<KIND>(q) + KEYS - 1) / KEYS); };
    auto blocks_of = [&](const TreeSeq& q) { return (q.rows * group + unit_rows - 1) / unit_rows; };
    auto info = [&](int s) {
        TreeSeq q{};
        if (s < seqs) q = seq_of<KIND>(p, s);
        return q;
    };
    auto line_of = [&](const TreeSeq& q) { return q.rows == 0 ? 0 : (int64_t)(tiles_of(q) + unit_tiles) * (heads * blocks_of(q)); };
    // a lane has a sequence at a time
    TreeSeq mine = info(lane);
    int64_t line64 = line_of(mine), total64 = line64;
#pragma unroll 1
    for (int s0 = 32; s0 < seqs; s0 += 32) total64 += line_of(info(s0 + lane));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total64 += __shfl_xor_sync(0xFFFFFFFFu, total64, o);
    if (total64 >= (1LL << 31)) {  // 3e10 keys: no cache holds them, some table says so
        report_status(p.status, STATUS_BAD_INDEX);
        none = true;
        return true;
    }
    const int total = (int)total64, share = total / (int)gridDim.x, more = total - share * (int)gridDim.x;  // the first `more` CTAs have a position more
    const int begin = (int)blockIdx.x * share + min((int)blockIdx.x, more), end = begin + share + ((int)blockIdx.x < more);
    auto cta_of = [&](int x) { return x < more * (share + 1) ? x / (share + 1) : more + (x - more * (share + 1)) / share; };
    int at = 0;  // where the lanes' sequences begin on the line
#pragma unroll 1
    for (int s0 = 0; s0 < seqs && at < end; s0 += 32) {
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
            if (KIND == ATTEND_LISTS) u.q.news = __shfl_sync(0xFFFFFFFFu, mine.news, l);
            if (KIND == ATTEND_OWN) {
                u.q.prefix = __shfl_sync(0xFFFFFFFFu, mine.prefix, l);
                u.q.place.table += u.q.prefix >> p.cache.page_shift;
            }
            if (KIND == ATTEND_WHOLE) u.q.prefix = __shfl_sync(0xFFFFFFFFu, mine.prefix, l), u.q.first = __shfl_sync(0xFFFFFFFFu, mine.first, l);
            if (KIND == ATTEND_PREFIX) u.q.place.table = reinterpret_cast<const int*>(__shfl_sync(0xFFFFFFFFu, reinterpret_cast<uint64_t>(mine.place.table), l));
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
                if (KIND == ATTEND_LISTS) u.head = u.seq % p.cache.kv_heads;
                const bool whole = u.from == 0 && u.to == u.tiles;
                u.first_cta = whole ? (int)blockIdx.x : cta_of(u_at + unit_tiles);
                u.last_cta = whole ? (int)blockIdx.x : cta_of(u_at + length - 1);
                if (!f(u)) return false;
            }
        }
    }
    return true;
}

// a / b for 0 <= a < 2^24 (or a < 2 b): by a float, which is off by one at most then, and put right.  Ten instructions where the exact division has thirty; what a CTA does before its
// first load it does once, and waits for every line of its code.
__device__ __forceinline__ int quick_div(int a, int b) {
    int q = (int)__fdividef((float)a, (float)b);
    const int rest = a - q * b;
    return q + (rest >= b) - (rest < 0);
}
// The part'th of `parts` parts of so many tiles begins here.
__device__ __forceinline__ int part_begins(int tiles, int parts, int part) {
    const int each = quick_div(tiles, parts);
    return part * each + min(part, tiles - parts * each);
}

// Walks the units that this CTA has by their number, the whole warp together.
// In a cluster every CTA has a part, if only one without tiles.
template <int KEYS, int KIND, class F> __device__ __forceinline__ bool walk_units(const TreeParams& p, const TreeCuts& c, int unit_rows, F f) {
    const int heads = p.cache.kv_heads, items = c.units * c.parts;  // below 2^23: launch_units
#pragma unroll 1
    for (int item = blockIdx.x; item < items; item += gridDim.x) {
        LineUnit u;
        const int unit = quick_div(item, c.parts), part = item - unit * c.parts;
        const int per_block = quick_div(unit, c.blocks), block = unit - per_block * c.blocks;  // per_block: a sequence's (token's) kv head
        const int seq = quick_div(per_block, heads);
        u.head = per_block - seq * heads;
        u.seq = KIND == ATTEND_LISTS ? per_block : seq;
        u.q = seq_of<KIND>(p, u.seq);
        u.first = block * unit_rows;
        if (u.first >= u.q.rows * p.group) continue;
        u.tiles = max(1, (keys_of<KIND>(u.q) + KEYS - 1) / KEYS);
        u.from = 0, u.to = u.tiles;
        if (c.parts > 1) {
            const int parts = min(c.parts, u.tiles);
            u.from = part < parts ? part_begins(u.tiles, parts, part) : u.tiles, u.to = part < parts ? part_begins(u.tiles, parts, part + 1) : u.tiles;
        }
        if (!f(u)) return false;
    }
    return true;
}

// For the kernel behind the one that reads the prefixes: which prefix a sequence has.  By a warp of every CTA.
__device__ __forceinline__ void leave_prefixes(const TreeParams& p, bool none) {
    const int lane = threadIdx.x & 31;
    for (int g = blockIdx.x; g < p.n_groups; g += gridDim.x) {
        const GroupSeqs of = group_seqs(p, g);
        for (int s = of.first + lane; s < of.stop; s += 32) p.prefix_of[s] = make_int2(none || !rows_in_group(p, of, s) ? -1 : of.prefix, of.first);
    }
    if (blockIdx.x == 0) {  // those that no group has
        const int before = max(0, min(p.groups[0], p.seqs)), behind = max(0, min(p.groups[p.n_groups], p.seqs));
        for (int s = lane; s < before; s += 32) p.prefix_of[s] = make_int2(-1, 0);
        for (int s = behind + lane; s < p.seqs; s += 32) p.prefix_of[s] = make_int2(-1, 0);
    }
}

// Walks this CTA's parts of prefixes.  (64 tokens of 8 x 8 heads behind 16384: 16 units in 18 parts of 7 or 8 tiles of 128 keys, two rounds of 148 CTAs.  On a line most CTAs have pieces of two units
// in one round, of which each waits for its queries, first tile and way out.)  All CTAs have a part of `most` tiles at most in each of one, two or three rounds, whichever takes least: sum ceil(tiles / most) is not more than total /
// most + units, so most = total / (rounds CTAs - units) is enough; where there is one group its units are alike, and rounds CTAs / units parts of each are exactly as many.  Groups
// that overlap may have more rows than there are tokens, and more units than there is room for: nothing is walked then.  Every unit's entry of `cuts` is written, where a wait ran out, too.
template <int KEYS, class F> __device__ __forceinline__ bool walk_prefixes(const TreeParams& p, const TreeCuts& c, int unit_rows, int unit_tiles, F f) {
    const int lane = threadIdx.x & 31, heads = p.cache.kv_heads, ctas = (int)gridDim.x, unit_tokens = quick_div(unit_rows, p.group);
    auto info = [&](int g) {
        TreeSeq q{};
        if (g < p.n_groups) q = prefix_seq(p, g);
        return q;
    };
    auto blocks_of = [&](const TreeSeq& q) { return quick_div(q.rows + unit_tokens - 1, unit_tokens); };
    auto units_of = [&](const TreeSeq& q) { return blocks_of(q) * heads; };
    auto tiles_of = [&](const TreeSeq& q) { return (q.context + KEYS - 1) / KEYS; };
    const TreeSeq first = info(lane);
    int units = units_of(first), total = units * tiles_of(first), rows = first.rows;
#pragma unroll 1
    for (int g0 = 32; g0 < p.n_groups; g0 += 32) {
        const TreeSeq q = info(g0 + lane);
        units += units_of(q), total += units_of(q) * tiles_of(q);
        rows = min(rows + q.rows, 1 << 18);  // (there are 2^17 tokens at most)
    }
    units = __reduce_add_sync(0xFFFFFFFFu, units);
    total = __reduce_add_sync(0xFFFFFFFFu, total);
    const bool too_many = __reduce_add_sync(0xFFFFFFFFu, rows) > p.tokens || (c.may_cut && units > c.units);
    if (units == 0 || too_many) {
        if (c.may_cut && blockIdx.x == 0)
            for (int i = lane; i < c.units; i += 32) c.cuts[i].first_cta = -1;
        if (too_many) report_status(p.status, STATUS_BAD_INDEX);
        leave_prefixes(p, too_many);
        return true;
    }
    bool well = true;
    int most = 1 << 28;  // tiles of a part
    TreeSeq first0 = first;  // the first group's, for all lanes
    first0.context = __shfl_sync(0xFFFFFFFFu, first.context, 0);
    if (c.may_cut) {
        int least = 1 << 30;
#pragma unroll 1
        for (int rounds = 1; rounds <= PREFIX_ROUNDS; rounds++) {
            const int room = rounds * ctas;
            if (units >= room) continue;
            const int each = quick_div(room, units), t = p.n_groups == 1 ? quick_div(tiles_of(first0) + each - 1, each) : (int)((unsigned)(total + room - units - 1) / (unsigned)(room - units));
            if (rounds * (t + unit_tiles) < least) least = rounds * (t + unit_tiles), most = t;
        }
    }
    int at = 0, unit_at = 0;  // items and units of the groups before the lanes'
    int item = (int)blockIdx.x;
#pragma unroll 1
    for (int g0 = 0; g0 < p.n_groups; g0 += 32) {
        TreeSeq mine = first;
        if (g0) mine = info(g0 + lane);
        const int my_units = units_of(mine), my_parts = my_units ? quick_div(tiles_of(mine) + most - 1, most) : 0, my_items = my_units * my_parts;
        int up_to = my_items, units_to = my_units;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xFFFFFFFFu, up_to, o), w = __shfl_up_sync(0xFFFFFFFFu, units_to, o);
            if (lane >= o) up_to += v, units_to += w;
        }
        const int all = __shfl_sync(0xFFFFFFFFu, up_to, 31);
#pragma unroll 1
        for (; item < at + all; item += ctas) {
            const int l = __ffs(__ballot_sync(0xFFFFFFFFu, at + up_to > item)) - 1;  // the group
            LineUnit u;
            u.q.row0 = __shfl_sync(0xFFFFFFFFu, mine.row0, l), u.q.rows = __shfl_sync(0xFFFFFFFFu, mine.rows, l), u.q.context = __shfl_sync(0xFFFFFFFFu, mine.context, l);
            u.q.place.table = reinterpret_cast<const int*>(__shfl_sync(0xFFFFFFFFu, reinterpret_cast<uint64_t>(mine.place.table), l));
            u.q.place.first = 0;
            u.seq = g0 + l;
            u.tiles = tiles_of(u.q);
            const int parts = __shfl_sync(0xFFFFFFFFu, my_parts, l), begin = at + __shfl_sync(0xFFFFFFFFu, up_to - my_items, l), unit = quick_div(item - begin, parts), part = item - begin - unit * parts;
            u.unit = unit_at + __shfl_sync(0xFFFFFFFFu, units_to - my_units, l) + unit;
            const int blocks = blocks_of(u.q);
            u.head = quick_div(unit, blocks);
            u.first = (unit - u.head * blocks) * unit_rows;
            u.from = part_begins(u.tiles, parts, part), u.to = part_begins(u.tiles, parts, part + 1);
            u.first_cta = item - part, u.last_cta = u.first_cta + parts - 1, u.part = item;
            if (c.may_cut && lane == 0 && (parts == 1 || (part == 0 && !well))) c.cuts[u.unit].first_cta = -1;
            if (well) well = f(u);
        }
        at += all;
        unit_at += __shfl_sync(0xFFFFFFFFu, units_to, 31);
    }
    if (c.may_cut && blockIdx.x == 0)
        for (int i = unit_at + lane; i < c.units; i += 32) c.cuts[i].first_cta = -1;  // there are no more
    leave_prefixes(p, false);
    return well;
}

// f(unit) for every unit, or part of one, that this CTA has, the whole warp together, until it answers false.  none: set where a line is too long.
template <int KEYS, int KIND, UnitWay WAY, class F> __device__ __forceinline__ bool walk_line(const TreeParams& p, const TreeCuts& c, int unit_rows, int unit_tiles, bool& none, F f) {
    if constexpr (WAY == UNITS_BY_NUMBER) return walk_units<KEYS, KIND>(p, c, unit_rows, f);
    else if constexpr (WAY == UNITS_IN_PARTS) return walk_prefixes<KEYS>(p, c, unit_rows, unit_tiles, f);
    else return walk_share<KEYS, KIND>(p, unit_rows, unit_tiles, c.may_cut, none, f);
}

// What a CTA leaves for tree_join_kernel: the unit that begins in its share and does not end there, if there is one.
template <int KIND> __device__ __forceinline__ void leave_cut(TreeCut& cut, const LineUnit& u, int count) {
    cut.first_cta = u.first_cta, cut.last_cta = u.last_cta;
    cut.row0 = u.q.row0, cut.rows = u.q.rows, cut.context = u.q.context, cut.seq = u.seq;
    cut.head = u.head, cut.first = u.first, cut.count = count;
    if (KIND == ATTEND_LISTS) cut.news = u.q.news;
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
// PARTS: the pieces are parts of prefixes, one place each; blockIdx.x is the unit.  (64 rows of 8 heads and one prefix in 18 parts, 22 MB of pieces out of the L2: 6 us.)
constexpr int JOIN_WARPS = 4, JOIN_AHEAD = 4;
template <int KIND, bool PARTS> __global__ void __launch_bounds__(JOIN_WARPS * 32) tree_join_kernel(const __grid_constant__ TreeParams p, const __grid_constant__ TreeCuts c) {
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
            const float* from = c.pieces + (PARTS ? (size_t)(c0 + i) : (size_t)(c0 + i) * 2 + (c0 + i == cut.first_cta)) * piece_floats;
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
    const int d = p.cache.dim, token = p.token_of(cut.first + row), head = cut.head * p.group + cut.first + row - token * p.group;
    const size_t place = (size_t)(cut.row0 + token) * p.q_heads + head;
    if (KIND == ATTEND_PREFIX) {  // the keys behind the prefix are another kernel's
        if (mine) *reinterpret_cast<float4*>(p.state + place * p.state_dim + 4 * lane) = x;
        if (lane == 0) p.state_maxima()[place] = top, p.state_weights()[place] = sum;
        return;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    bf16* const to = p.out + place * d;
    if (4 * lane < d) *reinterpret_cast<uint2*>(to + 4 * lane) = make_uint2(pack_bf16(x.x * inv, x.y * inv), pack_bf16(x.z * inv, x.w * inv));
    // Key by key where an Inf or a NaN may have come from a key that the row does not see, or from a page that is not in the cache.
    const float largest = fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
    const bool odd = !(sum < INFINITY) || scores_too_large(top, p.scale_log2) || !(largest < INFINITY) || x.x != x.x || x.y != x.y || x.z != x.z || x.w != x.w;
    if (__any_sync(0xFFFFFFFFu, odd)) attend_again<KIND>(p, cut, token, cut.head, p.q + (size_t)(cut.row0 + token) * p.q_stride + (size_t)head * d, to);
}
#endif

}  // namespace wf
