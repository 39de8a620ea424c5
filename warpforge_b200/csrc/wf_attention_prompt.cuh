// Attention on the 5th-generation tensor cores: whole prompts, and trees of drafted tokens with many rows.
//
//   S = Q K^T   [128 rows x 128 keys] fp32 in TMEM, Q and K in shared memory
//   P = 2^(S scale log2 e - m)        bf16, written over S in TMEM
//   O += P V    [128 rows x dim] fp32 in TMEM, P in TMEM, V in shared memory
//
// A CTA works on two tiles of rows of one kv head at a time, so that the tensor core has the one tile's products to do while the other
// tile's exponentials are taken; where there is one tile of rows, on every other tile of keys of it in turn.  The rows of a tile are the heads of the group for some tokens, token by
// token: keys and values are read once for the whole group.  A thread of the softmax warps has a row: its maximum and sum need no exchange.
//
// Bound by a chain: weights lie where the scores lay, so a group's next scores wait for its products, those for its exponentials, and a tile of keys is load of the scores, maxima,
// exponentials, stores, products, scores one after the other, with the other group's beside it.  A pair of tiles takes about 3300 cycles at dim 128 (2048 of products; tensor
// pipe 63 % busy, issue slots 52 %, special functions 40 %) and 3200 at dim 64 (1024; 33 %, 54 %, 42 %).  8192 tokens, 32 / 8 heads of 128: 440 us in a burst (1.25 PFLOP/s of
// the products that the mask leaves, 0.76 of the measured rate), 505 to 515 over seconds under the power limit; of 64: 386 us in a burst.
// 512 tokens, 32 / 32 heads: 12.2 us, a launch, 2 us until the first item is known (code and arguments come from memory), two pairs of tiles and the rows' way out.  Two threads a row
// (16 softmax warps): 604 us, where one took 521 at the time.
#pragma once
#include "wf_attention_line.cuh"
#include "wf_gemm_core.cuh"

namespace wf {

constexpr int PA_ROWS = 128, PA_KEYS = 128;  // of a tile
constexpr int PA_SOFTMAX_WARPS = 8;          // four a tile
constexpr int PA_LOAD_WARP = 8, PA_MMA_WARP = 9, PA_SCHED_WARP = 10;  // and one that has nothing to do: setmaxnreg wants four
constexpr int PA_THREADS = 12 * 32;
// Registers: 168 a thread at launch; the softmax warps, which hold a row of S, take what the others give back (256 x 224 + 128 x 56 = 384 x 168).
constexpr int PA_SOFTMAX_REGS = 224, PA_OTHER_REGS = 56;
constexpr int PA_CHUNK = PA_KEYS * 128;      // bytes of 128 rows x 64 elements
constexpr int PA_ITEMS = 2;                  // items announced ahead
// Which of the 32 pairs of weights of 64 keys are taken by the cubic: two in five, so that the special function unit and the fp32 units are through at about the same time
// (none / one in five / one in three / two in five: 449 / 433 / 431 / 435 us for 8192 tokens, 32 / 8 heads of 128; none / two in five: 429 / 372 of 64).
__host__ __device__ constexpr bool PA_CUBIC(int pair) { return pair % 5 == 1 || pair % 5 == 3; }
constexpr float PA_RESCALE = 8.f;            // the running maximum is followed when it has grown by this many powers of two
constexpr int PA_MAX_STAGES = 12;

// Two tiles of rows of one sequence and kv head.
struct PromptItem {
    int seq, head;
    int row0, rows, keys;  // of the sequence
    int token0;            // first token of tile 0
    int from, n0, n1;      // key tiles: the first, and where the tiles of rows end
    int split;             // one tile of rows: both groups work on it, n0 is where it ends, group g takes the key tiles from + g, from + g + 2, ..
    int context;           // tree: tokens before the new ones, -1: a sequence that cannot be
    int piece;             // tree: the unit is cut; 1: this piece is not the one it begins with, 2: it is
    int last;              // no more work (1), or a wait ran out
    // key tiles of group g
    __device__ __forceinline__ int tiles(int g) const { return split ? (n0 - from - g + 1) >> 1 : max(0, (g ? n1 : n0) - from); }
    __device__ __forceinline__ int all() const { return max(n0, n1) - from; }
};

struct PromptTiles {
    PromptParams p;
    int tile_tokens;   // tokens of a tile: 128 / group
    int box_rows;      // rows of keys that one TMA load brings: those of a page, at most 128
    int split;         // prompt: items have one tile of rows
    int wide_rows;     // rows of the output are made of aligned 32-byte pieces
    unsigned int* sched;  // prompt: [0] items taken beyond the first of each CTA, [1] CTAs that are done
    TreeParams tree;
    TreeCuts c;
};

// By the thread whose `issue` is non-zero; the whole warp comes here with the same operands, which then sit in uniform registers.
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar, uint32_t issue) {
    asm volatile("{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %6, 0;\n\t"
                 "@e cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n\t}" ::"r"(dst), "l"(map),
                 "r"(x), "r"(y), "r"(z), "r"(bar), "r"(issue)
                 : "memory");
}
__device__ __forceinline__ void mbar_expect_if(uint32_t bar, uint32_t bytes, uint32_t issue) {
    asm volatile("{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %2, 0;\n\t@e mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t}" ::"r"(bar), "r"(bytes), "r"(issue) : "memory");
}
// Operand of 16-bit elements with the other dimension contiguous (V: a row is a key, its elements run along N), 128-byte swizzle: 64 elements x 8
// rows are 1024 bytes, the next 8 rows follow, the next 64 elements lie `chunk` bytes on.
__device__ __forceinline__ uint64_t smem_desc_sw128_n(uint32_t saddr, uint32_t chunk) {
    return (uint64_t)((saddr & 0x3FFFF) >> 4) | (uint64_t)(chunk >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// Four MMAs over 64 elements of the heads: both operands in shared memory, 32 bytes apart in the swizzled rows.
__device__ __forceinline__ void pa_mma_qk(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate, uint32_t issue) {
    asm volatile(
        "{\n\t.reg .pred p, e, t;\n\t.reg .b64 a1, a2, a3, b1, b2, b3;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %5, 0;\n\tsetp.eq.b32 t, 0, 0;\n\t"
        "add.s64 a1, %1, 2;\n\tadd.s64 a2, %1, 4;\n\tadd.s64 a3, %1, 6;\n\t"
        "add.s64 b1, %2, 2;\n\tadd.s64 b2, %2, 4;\n\tadd.s64 b3, %2, 6;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a1, b1, %3, t;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a2, b2, %3, t;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a3, b3, %3, t;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(issue)
        : "memory");
}
// Four MMAs over 64 keys: weights in TMEM, eight columns each; values 16 rows (2048 bytes) apart.
__device__ __forceinline__ void pa_mma_pv(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate, uint32_t issue) {
    asm volatile(
        "{\n\t.reg .pred p, e, t;\n\t.reg .b32 a1, a2, a3;\n\t.reg .b64 b1, b2, b3;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %5, 0;\n\tsetp.eq.b32 t, 0, 0;\n\t"
        "add.s32 a1, %1, 8;\n\tadd.s32 a2, %1, 16;\n\tadd.s32 a3, %1, 24;\n\t"
        "add.s64 b1, %2, 128;\n\tadd.s64 b2, %2, 256;\n\tadd.s64 b3, %2, 384;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], b1, %3, t;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a2], b2, %3, t;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a3], b3, %3, t;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(issue)
        : "memory");
}
__device__ __forceinline__ void tc_commit_if(void* bar, uint32_t issue) {
    asm volatile(
        "{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %1, 0;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(g_smem_u32(bar)),
        "r"(issue)
        : "memory");
}
// 32 columns of this warp's 32 lanes, without the wait
__device__ __forceinline__ void tmem_ld32_start(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
// ... and the wait: what uses the columns stays behind it
__device__ __forceinline__ void tmem_wait_ld32(uint32_t* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                   "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]),
                   "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
        "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
        "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3_or_nan(float a, float b, float c) {  // the largest, or NaN where one of them is
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\tfma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
// 2^x for x <= PA_RESCALE without the special function unit, which has 16 of them a cycle and would be what a tile waits for: x = n + f with n the nearest
// integer (adding 1.5 * 2^23 leaves it in the low bits), 2^f by a cubic on [-1/2, 1/2], 1 at 0, with the smallest largest relative error (1.0e-4, 1/38 of
// what a weight may be off by its rounding to bf16), n added to the exponent.  0 from -127 on, and for NaN: a row that sees one is marked by its maxima.
__device__ __forceinline__ float2 add2(float2 a, float2 b);
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 w, x, y;\n\tmov.b64 {%0, %1}, w;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 ex2_by_cubic(float2 x) {
    x.x = fmaxf(x.x, -127.f);
    x.y = fmaxf(x.y, -127.f);
    const float2 big = make_float2(12582912.f, 12582912.f), less = make_float2(-12582912.f, -12582912.f);
    const float2 t = add2(x, big), n = add2(t, less), f = fma2(n, make_float2(-1.f, -1.f), x);
    float2 y = fma2(f, make_float2(0.05500893f, 0.05500893f), make_float2(0.24221095f, 0.24221095f));
    y = fma2(y, f, make_float2(0.6932829f, 0.6932829f));
    y = fma2(y, f, make_float2(1.f, 1.f));
    return make_float2(__uint_as_float(__float_as_uint(y.x) + (__float_as_uint(t.x) << 23)), __uint_as_float(__float_as_uint(y.y) + (__float_as_uint(t.y) << 23)));
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 w, x, y;\n\tmov.b64 {%0, %1}, w;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

// Waits for a barrier, the whole warp with one answer.
__device__ __forceinline__ bool pa_wait(uint64_t* bar, uint32_t parity) { return __all_sync(0xFFFFFFFFu, g_mbar_wait(bar, parity)); }

// 32 bytes, aligned: a sector in one store (a thread stores its own row: each of a warp's stores touches 32 lines, which is what it costs)
__device__ __forceinline__ void store_32(void* to, const uint32_t* w) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}

struct PromptShared {
    uint64_t q_full[2], q_empty[2];
    uint64_t s_full[2], p_half[2], p_full[2], o_full[2];  // scores; weights of the first 64 keys, of all; sums
    uint64_t half_ready, half_taken;  // one tile of rows, two groups: their maxima and sums lie in half_max and half_sum; both O have been read
    float half_max[2][PA_ROWS], half_sum[2][PA_ROWS];
    uint32_t half_odd[4];  // rows that the second group has seen to be not finite
    uint64_t kv_full[PA_MAX_STAGES], kv_empty[PA_MAX_STAGES];
    uint64_t item_full[PA_ITEMS], item_empty[PA_ITEMS];
    PromptItem items[PA_ITEMS];
    int bad_pages[2][2 * PA_ITEMS];  // group g's key tiles of an item (ItemCursor::mark) have pages outside the cache
    uint32_t tmem;
};

template <int CHUNKS> struct PromptShape {  // by the head's dimension in 64 elements, rounded up
    static constexpr int STAGES = CHUNKS == 2 ? 5 : 12, STAGE_BYTES = CHUNKS * PA_CHUNK, Q_BYTES = 2 * CHUNKS * PA_CHUNK;
    static constexpr int SMEM = Q_BYTES + STAGES * STAGE_BYTES + (int)sizeof(PromptShared);
    static_assert(SMEM <= 227 * 1024, "shared memory");
};

// The next item of the ring; false: no more, or a wait ran out.
struct ItemCursor {
    int slot = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ bool next(PromptShared* sh, PromptItem& it, bool& failed) {
        if (!pa_wait(&sh->item_full[slot], phase)) {
            failed = true;
            return false;
        }
        it = sh->items[slot];
        __syncwarp();
        if ((threadIdx.x & 31) == 0) g_mbar_arrive(&sh->item_empty[slot]);
        if (++slot == PA_ITEMS) slot = 0, phase ^= 1;
        return it.last == 0;
    }
    // A place for what the load warp finds out about the item.  It is at most PA_ITEMS items ahead of the softmax warps: twice as many places are enough.
    __device__ __forceinline__ int mark() const { return slot + PA_ITEMS * (int)phase; }
};

// Which items there are, the longest first (a CTA's numbers are taken up to four items ahead, so the order evens out calls with many items a CTA, not those with
// three): tiles of a sequence count from where its past ends, v = block + past / block tokens, and v goes down
// over all sequences at once.  Every lane has every 32nd sequence.
struct PromptSchedule {
    const PromptTiles& t;
    int block;       // tokens of an item
    int v;           // where the cursor is
    int before;      // items with a larger v
    int count;       // sequences that have this v
    PromptSeq mine;  // of the first 32 sequences, this lane's; the others are looked up when they are needed
    int mine_lo, mine_hi;
    __device__ __forceinline__ PromptSeq look(int s, int& lo, int& hi) const {  // a sequence and its v: [lo, hi)
        PromptSeq q{};
        lo = hi = 0;
        if (s >= t.p.seqs) return q;
        q = prompt_seq(t.p, s);
        lo = max(0, q.keys - q.rows) / block;
        hi = lo + (q.rows + block - 1) / block;
        return q;
    }
    __device__ __forceinline__ uint32_t with(int s0, int value, int& lo, PromptSeq& q) const {  // which of 32 sequences have it
        int hi = mine_hi;
        lo = mine_lo;
        q = mine;
        if (s0) q = look(s0 + (threadIdx.x & 31), lo, hi);
        return __ballot_sync(0xFFFFFFFFu, value >= lo && value < hi);
    }
    __device__ __forceinline__ int have(int value) const {
        int n = 0, lo;
        PromptSeq q;
#pragma unroll 1
        for (int s0 = 0; s0 < t.p.seqs; s0 += 32) n += __popc(with(s0, value, lo, q));
        return n;
    }
    // the largest v below this one that any sequence has, -1: none
    __device__ __forceinline__ int below(int value) const {
        int best = -1;
#pragma unroll 1
        for (int s0 = 0; s0 < t.p.seqs; s0 += 32) {
            int lo = mine_lo, hi = mine_hi;
            if (s0) look(s0 + (threadIdx.x & 31), lo, hi);
            if (min(hi, value) > lo) best = max(best, min(hi, value) - 1);
        }
        return __reduce_max_sync(0xFFFFFFFFu, best);
    }
    __device__ __forceinline__ void begin() {
        block = (t.split ? 1 : 2) * t.tile_tokens;
        mine = look(threadIdx.x & 31, mine_lo, mine_hi);
        int top = mine_hi;
#pragma unroll 1
        for (int s = 32 + (threadIdx.x & 31); s < t.p.seqs; s += 32) {
            int lo, hi;
            look(s, lo, hi);
            top = max(top, hi);
        }
        v = __reduce_max_sync(0xFFFFFFFFu, top) - 1;
        before = 0;
        count = v >= 0 ? have(v) : 0;
    }
    // item i (they come in ascending order); false: there is none
    __device__ __forceinline__ bool find(int i, PromptItem& it) {
        const int heads = t.p.cache.kv_heads;
#pragma unroll 1
        while (v >= 0 && i >= before + count * heads) {
            before += count * heads;
            if (--v < 0) break;
            count = have(v);
            if (count) continue;
            // None, as between one sequence's long past and the others' ends: at once to the next v that there is.  (One by one, a token behind 100,000 others took
            // 1.2 ms with 8 query heads for its kv head and 16 with 128, where it now takes 0.66.)
            v = below(v);
            if (v >= 0) count = have(v);
        }
        if (v < 0) return false;
        int nth = (i - before) / heads;
        it.head = i - before - nth * heads;
#pragma unroll 1
        for (int s0 = 0; s0 < t.p.seqs; s0 += 32) {
            int lo;
            PromptSeq q;
            uint32_t which = with(s0, v, lo, q);
            const int n = __popc(which);
            if (nth >= n) {
                nth -= n;
                continue;
            }
            for (; nth > 0; nth--) which &= which - 1;
            const int lane = __ffs(which) - 1;
            it.seq = s0 + lane;
            it.row0 = __shfl_sync(0xFFFFFFFFu, q.row0, lane);
            it.rows = __shfl_sync(0xFFFFFFFFu, q.rows, lane);
            it.keys = __shfl_sync(0xFFFFFFFFu, q.keys, lane);
            it.token0 = (v - __shfl_sync(0xFFFFFFFFu, lo, lane)) * block;
            break;
        }
        auto tiles = [&](int token) {  // key tiles that a tile of rows starting at this token sees
            if (token >= it.rows) return 0;
            const int last = it.keys - it.rows + min(it.rows, token + t.tile_tokens) - 1;
            return last < 0 ? 0 : last / PA_KEYS + 1;
        };
        it.from = it.piece = it.last = 0;
        it.split = t.split;
        it.n0 = tiles(it.token0);
        it.n1 = t.split ? 0 : tiles(it.token0 + t.tile_tokens);
        return true;
    }
};

// The items of a CTA's share of a tree call.
// What a unit costs beyond its key tiles, in key tiles: with 0 / 1 / 2 / 3 / 4 / 6, eight sequences of 0 to 3000 tokens and up to 24 drafts take 27.5 / 24.3 / 24.2 / 22.9 /
// 23.0 / 23.4 us.
constexpr int PA_UNIT_TILES = 3;
// When units are cut (line_is_cut).  Microseconds whole / cut, 12 drafts of 32 / 8 heads of 128: 16 sequences with 700, 1000, 1400, 1800 tokens 16.3 / 23.9, 19.6 / 27.4,
// 26.5 / 32.7, 31.2 / 37.7; 8 with 1000, 1400 17.0 / 19.2, 22.5 / 22.4; 20 with 1000, 1400 31.9 / 30.7, 42.8 / 37.9; 4 with 600, 1000 12.8 / 14.5, 15.9 / 15.7.
constexpr int PA_CUT_TILES = 6, PA_CUT_ANYWAY = 15;
template <class F> __device__ __forceinline__ bool tree_items(const PromptTiles& t, F f) {
    const TreeParams& p = t.tree;
    bool cut = false;
    const bool ok = walk_line<PA_KEYS>(p, 2 * t.tile_tokens * p.group, PA_UNIT_TILES, t.c.may_cut, [&](const LineUnit& u) {
        PromptItem it{};
        it.seq = u.seq, it.head = u.head, it.row0 = u.q.row0, it.rows = u.q.rows, it.context = u.q.context;
        it.keys = u.q.context < 0 ? 0 : u.q.context + u.q.rows;
        it.token0 = u.first / p.group;
        it.from = u.from;
        it.n0 = u.to;
        it.split = it.rows - it.token0 <= t.tile_tokens;
        it.n1 = it.split ? u.from : u.to;
        it.piece = u.from == 0 && u.to == u.tiles ? 0 : u.from == 0 ? 2 : 1;
        if (it.piece == 2) {
            cut = true;
            if ((threadIdx.x & 31) == 0) leave_cut(t.c, u, min(2 * t.tile_tokens, it.rows - it.token0) * p.group);
        }
        return f(it);
    });
    if (t.c.may_cut && !cut && (threadIdx.x & 31) == 0) t.c.cuts[blockIdx.x].first_cta = -1;
    return ok;
}

template <int CHUNKS, bool TREE>
__global__ void __launch_bounds__(PA_THREADS, 1) prompt_tiles_kernel(const __grid_constant__ PromptTiles t, const __grid_constant__ CUtensorMap q_map,
                                                                    const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
    constexpr int DIM = CHUNKS * 64, STAGES = PromptShape<CHUNKS>::STAGES, STAGE_BYTES = PromptShape<CHUNKS>::STAGE_BYTES;
    constexpr uint32_t IDESC = 1u << 4 | 1u << 7 | 1u << 10 | (uint32_t)(PA_ROWS / 16) << 24;  // fp32 += bf16 x bf16, 128 rows
    constexpr uint32_t IDESC_QK = IDESC | (uint32_t)(PA_KEYS / 8) << 17, IDESC_PV = IDESC | 1u << 16 | (uint32_t)(DIM / 8) << 17;
    constexpr uint32_t O_COLUMN = 2 * PA_KEYS;  // TMEM: S of tile 0, S of tile 1, O of tile 0, O of tile 1
    extern __shared__ __align__(1024) uint8_t raw[];  // the kernel has no other shared memory: it begins where the swizzle wants it to
    PromptShared* const sh = reinterpret_cast<PromptShared*>(raw + PromptShape<CHUNKS>::Q_BYTES + STAGES * STAGE_BYTES);
    const uint32_t smem = g_smem_u32(raw), kv_smem = smem + PromptShape<CHUNKS>::Q_BYTES;
    const PromptParams& p = t.p;
    const int warp = __shfl_sync(0xFFFFFFFFu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    if (warp == PA_LOAD_WARP && lane == 0) {
        for (int g = 0; g < 2; g++) {
            g_mbar_init(&sh->q_full[g], 1);
            g_mbar_init(&sh->q_empty[g], 1);
            g_mbar_init(&sh->s_full[g], 1);
            g_mbar_init(&sh->p_half[g], 4);
            g_mbar_init(&sh->p_full[g], 4);
            g_mbar_init(&sh->o_full[g], 1);
        }
        g_mbar_init(&sh->half_ready, 8);
        g_mbar_init(&sh->half_taken, 8);
        for (int i = 0; i < STAGES; i++) {
            g_mbar_init(&sh->kv_full[i], 1);
            g_mbar_init(&sh->kv_empty[i], 1);
        }
        for (int i = 0; i < PA_ITEMS; i++) {
            g_mbar_init(&sh->item_full[i], 1);
            g_mbar_init(&sh->item_empty[i], PA_SOFTMAX_WARPS + 2);
        }
        for (int i = 0; i < 2 * PA_ITEMS; i++) sh->bad_pages[0][i] = sh->bad_pages[1][i] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        prefetch_tensormap(&q_map);
        prefetch_tensormap(&k_map);
        prefetch_tensormap(&v_map);
    }
    if (warp == PA_MMA_WARP) tmem_alloc(&sh->tmem, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh->tmem;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");

    bool failed = false;
    PromptItem it;
    ItemCursor items;
    if (warp < PA_SOFTMAX_WARPS) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(PA_SOFTMAX_REGS));
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PA_OTHER_REGS));
    if (warp < PA_SOFTMAX_WARPS) {
        const int g = warp >> 2, r = (warp & 3) * 32 + lane;  // the tile, the row of it
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, s_at = tmem + lanes + (uint32_t)(g * PA_KEYS), o_at = tmem + lanes + O_COLUMN + (uint32_t)(g * DIM);
        const int group = p.group, tile_tokens = t.tile_tokens;
        const int my_token = r / group, my_head = r % group;
        const float scale = p.scale_log2;
        uint32_t s_phase = 0, o_phase[2] = {0, 0}, half_phase = 0;
        while (items.next(sh, it, failed)) {
            const int n = it.tiles(g), step = it.split ? 2 : 1;
            const int first = it.token0 + (it.split ? 0 : g * tile_tokens), token = first + my_token;
            const bool mine = r < group * tile_tokens && token < it.rows;
            const int last_key = it.keys - it.rows + token;  // prompt: that the row sees
            const int all_see = TREE ? it.context - 1 : it.keys - it.rows + first + (warp & 3) * 32 / group;  // that every row of this warp sees
            const uint64_t word = TREE && mine && it.keys > 0 ? ancestors_of(t.tree, it.row0 + token, token) & ((uint64_t)-1 >> (64 - it.rows)) : 0;
            float m = -INFINITY, l = 0.f;
            int j = it.from + (it.split ? g : 0);  // the key tile
            for (int i_tile = 0; i_tile < n; i_tile++, j += step) {
                if (!pa_wait(&sh->s_full[g], s_phase)) {
                    failed = true;
                    break;
                }
                s_phase ^= 1;
                tc_fence_after();
                uint32_t s[PA_KEYS];
                float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                auto maxima = [&](int c) {  // of 32 keys
#pragma unroll
                    for (int i = 32 * c; i < 32 * c + 32; i += 8)
#pragma unroll
                        for (int e = 0; e < 4; e++) top[e] = max3_or_nan(top[e], __uint_as_float(s[i + 2 * e]), __uint_as_float(s[i + 2 * e + 1]));
                };
                tmem_ld32_start(s_at, s);
                tmem_wait_ld32(s);
                const bool masked = j * PA_KEYS + PA_KEYS - 1 > all_see;  // keys that some row of the warp does not see
#pragma unroll
                for (int c = 1; c < 4; c++) {
                    tmem_ld32_start(s_at + 32 * c, s + 32 * c);
                    if (!masked) maxima(c - 1);  // under the load
                    tmem_wait_ld32(s + 32 * c);
                }
                if (masked) {
                    if (TREE) {
                        // bit i of the four words: the row sees key i of the tile.  Below `old` it does, from there on the ancestors say so.
                        const int old = it.context - j * PA_KEYS;
#pragma unroll
                        for (int c = 0; c < 4; c++) {
                            const int at = old - 32 * c;  // where the word begins, seen from this one
                            uint32_t bits = it.context < 0 || at <= 0 ? 0u : at >= 32 ? 0xFFFFFFFFu : (1u << at) - 1;
                            if (at > -64 && at < 32) bits |= at >= 0 ? (uint32_t)(word << at) : (uint32_t)(word >> -at);
#pragma unroll
                            for (int i = 0; i < 32; i++)
                                if (!(bits >> i & 1)) s[32 * c + i] = 0xFF800000u;
                        }
                    } else {
                        const int limit = last_key - j * PA_KEYS;
#pragma unroll
                        for (int i = 0; i < PA_KEYS; i++)
                            if (i > limit) s[i] = 0xFF800000u;
                    }
#pragma unroll
                    for (int c = 0; c < 3; c++) maxima(c);
                }
                maxima(3);
                float tile_top = max3_or_nan(max3_or_nan(top[0], top[1], top[2]), top[3], -INFINITY);
                if (tile_top != tile_top) {  // a score that the row sees is NaN: so is its sum from here on, whatever the cubic makes of it
                    l = tile_top;
                    tile_top = -INFINITY;
                }
                if (i_tile == 0) {
                    m = tile_top;
                } else if (__any_sync(0xFFFFFFFFu, (tile_top - m) * scale > PA_RESCALE)) {
                    // O is at rest: the MMAs that made it ran before those that made S
                    const float grown = fmaxf(m, tile_top), ref = grown == -INFINITY ? 0.f : grown;
                    const float keep = ex2((m - ref) * scale);
                    m = grown;
                    l *= keep;
#pragma unroll
                    for (int c = 0; c < DIM; c += 32) {
                        uint32_t o[32];
                        tmem_ld32_start(o_at + c, o);
                        tmem_wait_ld32(o);
#pragma unroll
                        for (int i = 0; i < 32; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * keep);
                        tmem_st32(o_at + c, o);
                    }
                }
                const float ref = m == -INFINITY ? 0.f : m * scale;
                const float2 sc = make_float2(scale, scale), off = make_float2(-ref, -ref);
                float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
                uint32_t w[32];
#pragma unroll
                for (int h = 0; h < 2; h++) {
#pragma unroll
                    for (int i = 0; i < 32; i++) {
                        const int k = 64 * h + 2 * i;
                        float2 x = fma2(make_float2(__uint_as_float(s[k]), __uint_as_float(s[k + 1])), sc, off);
                        if (PA_CUBIC(i)) {
                            x = ex2_by_cubic(x);
                        } else {
                            x.x = ex2(x.x);
                            x.y = ex2(x.y);
                        }
                        sum[i & 1] = add2(sum[i & 1], x);
                        w[i] = pack_bf16(x.x, x.y);
                    }
                    tmem_st32(s_at + 32 * h, w);
                    if (h == 0) {  // the products of these keys may begin
                        tmem_wait_st();
                        tc_fence_before();
                        if (lane == 0) g_mbar_arrive(&sh->p_half[g]);
                    }
                }
                const float2 both = add2(sum[0], sum[1]);
                l += both.x + both.y;
                tmem_wait_st();
                tc_fence_before();
                if (lane == 0) g_mbar_arrive(&sh->p_full[g]);
            }
            if (failed) break;
            const int row = it.row0 + token, head = it.head * group + my_head;
            const int d = p.cache.dim;
            bool odd = false;  // something is not finite
            const bool halves = it.split && it.tiles(1) > 0;
            if (n > 0) {
                if (!pa_wait(&sh->o_full[g], o_phase[g])) {
                    failed = true;
                    break;
                }
                tc_fence_after();
            }
            if (TREE && *reinterpret_cast<volatile int*>(&sh->bad_pages[g][items.mark()])) l = __uint_as_float(0x7FC00000u);
            float keep = 1.f, take = 0.f, top = m;
            if (halves) {  // both groups add both up, half of the columns each
                sh->half_max[g][r] = m;
                sh->half_sum[g][r] = l;
                __syncwarp();
                if (lane == 0) g_mbar_arrive(&sh->half_ready);
                if (!pa_wait(&sh->half_ready, half_phase) || !pa_wait(&sh->o_full[g ^ 1], o_phase[g ^ 1])) {
                    failed = true;
                    break;
                }
                tc_fence_after();
                const float other = sh->half_max[g ^ 1][r];
                top = fmaxf(m, other);
                const float ref = top == -INFINITY ? 0.f : top;
                keep = ex2((m - ref) * scale), take = ex2((other - ref) * scale);
                l = l * keep + sh->half_sum[g ^ 1][r] * take;
            }
#pragma unroll
            for (int e = 0; e < 2; e++) o_phase[e] ^= it.tiles(e) > 0;  // the other group's, too
            const bool whole = !(TREE && it.piece);
            if (n > 0) {
                const float inv = l == 0.f ? 0.f : __frcp_rn(l);
                const float2 f0 = make_float2(whole ? keep * inv : keep, whole ? keep * inv : keep), f1 = make_float2(whole ? take * inv : take, whole ? take * inv : take);
                const int rows = t.c.piece_rows, at = it.split ? r : g * PA_ROWS + r;
                float* const piece = t.c.pieces + ((size_t)blockIdx.x * 2 + (it.piece == 2)) * rows * (DIM + 2);
                if (!whole && r < group * tile_tokens && !(halves && g)) {
                    piece[rows * DIM + at] = top;
                    piece[rows * (DIM + 1) + at] = l;
                }
                // Few instructions and a small loop: it runs once an item, by one warp a scheduler at about three cycles an instruction.  (Transposed among four lanes, so that
                // a store touches 8 rows and not 32, it took twice as long.)
                float2 finite = make_float2(0.f, 0.f);  // the sum: an Inf or a NaN stays in it
                const uint32_t other_at = o_at + (uint32_t)(g ? -DIM : DIM);
#pragma unroll 1
                for (int c = halves && g ? DIM / 2 : 0; c < (halves && !g ? DIM / 2 : DIM); c += 32) {
                    uint32_t o[32];
                    tmem_ld32_start(o_at + c, o);
                    tmem_wait_ld32(o);
                    float2* const x = reinterpret_cast<float2*>(o);
#pragma unroll
                    for (int i = 0; i < 16; i++) x[i] = mul2(x[i], f0);
                    if (halves) {
                        uint32_t o1[32];
                        tmem_ld32_start(other_at + c, o1);
                        tmem_wait_ld32(o1);
#pragma unroll
                        for (int i = 0; i < 16; i++) x[i] = fma2(reinterpret_cast<float2*>(o1)[i], f1, x[i]);
                    }
                    if (TREE && !whole) {
                        if (mine)
#pragma unroll
                            for (int i = 0; i < 4; i++) store_32(piece + (size_t)at * DIM + c + 8 * i, o + 8 * i);
                        continue;
                    }
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        finite = add2(finite, x[i]);
                        o[i] = pack_bf16(x[i].x, x[i].y);
                    }
                    bf16* const to = p.out + ((size_t)row * p.q_heads + head) * d + c;
                    if (t.wide_rows) {
#pragma unroll
                        for (int i = 0; i < 2; i++)
                            if (mine && c + 16 * i < d) store_32(to + 16 * i, o + 8 * i);
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            if (mine && c + 8 * i < d) *reinterpret_cast<uint4*>(to + 8 * i) = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                    }
                }
                odd = whole && (!(l < INFINITY) || scores_too_large(top, scale) || !(fabsf(finite.x + finite.y) < INFINITY));
                tc_fence_before();
            } else if (!TREE && mine && !(it.split && g)) {
                for (int i = 0; i < d; i += 8) *reinterpret_cast<uint4*>(p.out + ((size_t)row * p.q_heads + head) * d + i) = make_uint4(0u, 0u, 0u, 0u);
            }
            if (halves) {
                const uint32_t which = __ballot_sync(0xFFFFFFFFu, odd);
                if (g && lane == 0) sh->half_odd[warp & 3] = which;
                if (lane == 0) g_mbar_arrive(&sh->half_taken);
                if (!pa_wait(&sh->half_taken, half_phase)) {
                    failed = true;
                    break;
                }
                half_phase ^= 1;
                odd = !g && (odd || (sh->half_odd[warp & 3] >> lane & 1));  // the first group's
            }
            // Rows with an Inf or a NaN in their sums, and rows whose pages are not in the cache, go key by key: the first may have
            // come from a key that the row does not see (0 x Inf), the second's keys were not read.
            if (!TREE) odd |= !(it.split && g) && *reinterpret_cast<volatile int*>(&sh->bad_pages[g][items.mark()]);
            uint32_t again = __ballot_sync(0xFFFFFFFFu, mine && odd);
            while (again) {
                const int l2 = __ffs(again) - 1;
                again &= again - 1;
                const int tok = __shfl_sync(0xFFFFFFFFu, token, l2), hd = __shfl_sync(0xFFFFFFFFu, head, l2), last = it.keys - it.rows + tok;
                KeyPlace place;
                place.table = p.tables ? p.tables + (size_t)it.seq * p.table_stride : nullptr;
                place.first = it.row0;
                const bf16* q_row = p.q + (size_t)(it.row0 + tok) * p.q_stride + (size_t)hd * d;
                bf16* out_row = p.out + ((size_t)(it.row0 + tok) * p.q_heads + hd) * d;
                if (TREE)
                    attend_row(p.cache, place, q_row, out_row, it.head, it.keys, p.scale_log2, p.status,
                               SeesAncestors{it.context, ancestors_of(t.tree, it.row0 + tok, tok) & ((uint64_t)-1 >> (64 - it.rows))});
                else attend_row(p.cache, place, q_row, out_row, it.head, min(it.keys, last + 1), p.scale_log2, p.status, SeesUpTo{last});
            }
        }
    } else if (warp == PA_LOAD_WARP) {
        const uint32_t issue = elect_one();
        StageCursor ring;
        uint32_t q_phase[2] = {1, 1};
        const int boxes = PA_KEYS / t.box_rows;
        while (items.next(sh, it, failed)) {
            const int n = it.all();
            const int* table = p.tables ? p.tables + (size_t)it.seq * p.table_stride : nullptr;
            // the rows of a key tile's boxes, a lane each, and how many there are
            auto find = [&](int j, int& z) {
                if (!table) {
                    z = it.row0 + j * PA_KEYS;
                    return 1;
                }
                const int key = j * PA_KEYS + lane * t.box_rows;
                int page = 0;
                const bool valid = lane < boxes && (key < it.keys || (TREE && lane == 0));  // a sequence that cannot be reads something, and sees nothing
                if (valid && key < it.keys) page = table[key >> p.cache.page_shift];
                if (page < 0 || page >= p.cache.pages) {  // never followed: these rows go key by key
                    report_status(p.status, STATUS_BAD_INDEX);
                    for (int g = 0; g < 2; g++)
                        if (it.split || j < (g ? it.n1 : it.n0)) *reinterpret_cast<volatile int*>(&sh->bad_pages[g][items.mark()]) = 1;
                    page = 0;
                }
                __syncwarp();  // the mark is there before a tile that this warp loads
                z = (int)((((int64_t)page * p.cache.kv_heads + it.head) << p.cache.page_shift) + (key & ((1 << p.cache.page_shift) - 1)));
                return __popc(__ballot_sync(0xFFFFFFFFu, valid));
            };
            auto load = [&](const CUtensorMap* map, int z, int loads) {
                if (!pa_wait(&sh->kv_empty[ring.s], ring.phase ^ 1)) {
                    failed = true;
                    return;
                }
                const uint32_t bar = g_smem_u32(&sh->kv_full[ring.s]);
                mbar_expect_if(bar, (uint32_t)(loads * CHUNKS * 128 * t.box_rows), issue);
                for (int i = 0; i < loads; i++) {
                    const int row = __shfl_sync(0xFFFFFFFFu, z, i);
#pragma unroll
                    for (int c = 0; c < CHUNKS; c++)
                        tma_load_3d(kv_smem + (uint32_t)(ring.s * STAGE_BYTES + c * PA_CHUNK + i * t.box_rows * 128), map, 64 * c, table ? 0 : it.head, row, bar, issue);
                }
                ring.advance(STAGES);
            };
            int z = 0, z_before = 0, loads = 0, loads_before = 0;
            for (int j = 0; j < n && !failed; j++) {  // keys 0, keys 1, values 0, keys 2, values 1, ..
                loads = find(it.from + j, z);
                auto queries = [&](int g) {
                    if (it.tiles(g) == 0) return;
                    if (!pa_wait(&sh->q_empty[g], q_phase[g])) failed = true;
                    q_phase[g] ^= 1;
                    if (failed) return;
                    const uint32_t bar = g_smem_u32(&sh->q_full[g]);
                    mbar_expect_if(bar, (uint32_t)(CHUNKS * 128 * p.group * t.tile_tokens), issue);
                    const int first = it.row0 + it.token0 + (it.split ? 0 : g * t.tile_tokens);
#pragma unroll
                    for (int c = 0; c < CHUNKS; c++) tma_load_3d(smem + (uint32_t)((g * CHUNKS + c) * PA_CHUNK), &q_map, 64 * c, it.head * p.group, first, bar, issue);
                };
                if (j == 0) queries(0);
                if (!failed) load(&k_map, z, loads);
                if (j == 0 && !failed) queries(1);
                if (j > 0 && !failed) load(&v_map, z_before, loads_before);
                z_before = z;
                loads_before = loads;
            }
            if (n > 0 && !failed) load(&v_map, z_before, loads_before);
            if (failed) break;
            if (lane < 2) *reinterpret_cast<volatile int*>(&sh->bad_pages[lane][(items.mark() + 1) % (2 * PA_ITEMS)]) = 0;  // the next item's
            __syncwarp();
        }
    } else if (warp == PA_MMA_WARP) {
        // Everything here is laid out for the pace of the issuing thread: the group is a constant in every place (as a variable the kernel lost 10 %).
        const uint32_t issue = elect_one();
        uint32_t q_phase[2] = {0, 0}, p_phase[2] = {0, 0};
        struct Place {  // in the ring
            int s = 0;
            uint32_t phase = 0;
            __device__ __forceinline__ void advance(int by) {
                s += by;
                if (s >= STAGES) s -= STAGES, phase ^= 1;
            }
        } begin;
        typedef std::integral_constant<int, 0> Group0;
        typedef std::integral_constant<int, 1> Group1;
        auto there = [&](const Place& at) {  // its keys or values have arrived
            if (!pa_wait(&sh->kv_full[at.s], at.phase)) failed = true;
            tc_fence_after();
            return !failed;
        };
        auto scores = [&](auto group, int stage) {  // S = Q K^T
            constexpr int g = decltype(group)::value;
            const uint64_t a = smem_desc_sw128(smem + (uint32_t)(g * CHUNKS * PA_CHUNK)), b = smem_desc_sw128(kv_smem + (uint32_t)(stage * STAGE_BYTES));
#pragma unroll
            for (int c = 0; c < CHUNKS; c++)
                pa_mma_qk(tmem + (uint32_t)(g * PA_KEYS), a + (uint64_t)(c * (PA_CHUNK >> 4)), b + (uint64_t)(c * (PA_CHUNK >> 4)), IDESC_QK, c > 0, issue);
            tc_commit_if(&sh->s_full[g], issue);
        };
        auto first_scores = [&](auto group, int stage, int tiles) {
            constexpr int g = decltype(group)::value;
            if (!pa_wait(&sh->q_full[g], q_phase[g])) {
                failed = true;
                return false;
            }
            q_phase[g] ^= 1;
            tc_fence_after();
            scores(group, stage);
            if (tiles == 1) tc_commit_if(&sh->q_empty[g], issue);
            return true;
        };
        auto products = [&](auto group, int stage, bool accumulate) {  // O += P V
            constexpr int g = decltype(group)::value;
            const uint64_t b = smem_desc_sw128_n(kv_smem + (uint32_t)(stage * STAGE_BYTES), PA_CHUNK);
#pragma unroll
            for (int h = 0; h < 2; h++) {
                if (!pa_wait(h ? &sh->p_full[g] : &sh->p_half[g], p_phase[g])) {
                    failed = true;
                    return false;
                }
                tc_fence_after();
                pa_mma_pv(tmem + O_COLUMN + (uint32_t)(g * DIM), tmem + (uint32_t)(g * PA_KEYS + 32 * h), b + (uint64_t)(h * 512), IDESC_PV, accumulate || h > 0, issue);
            }
            p_phase[g] ^= 1;
            return true;
        };
        while (items.next(sh, it, failed)) {
            const int n = it.all(), nt[2] = {it.tiles(0), it.tiles(1)};
            if (n == 0) continue;
            const bool tail = max(it.n0, it.n1) * PA_KEYS > it.keys;
            auto zero_tail = [&](int stage, int j) {  // values behind the last key: their weights are 0, and 0 x whatever lies there has to be 0
                if (!tail || j != n - 1) return;
                for (int c = 0; c < CHUNKS; c++)
                    for (int i = max(0, it.keys - (it.from + j) * PA_KEYS) * 8 + lane; i < PA_KEYS * 8; i += 32)
                        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(kv_smem + (uint32_t)(stage * STAGE_BYTES + c * PA_CHUNK + i * 16)), "r"(0) : "memory");
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
            };
            Place keys = begin, values = begin;  // keys 0, keys 1, values 0, keys 2, values 1, .., the last two values
            values.advance(n > 1 ? 2 : 1);
            if (!there(keys)) break;
            if (!it.split) {
                if ((nt[0] && !first_scores(Group0{}, keys.s, nt[0])) || (nt[1] && !first_scores(Group1{}, keys.s, nt[1]))) break;
                tc_commit_if(&sh->kv_empty[keys.s], issue);
                keys.advance(1);
                for (int j = 0; j < n; j++) {
                    if (!there(values)) break;
                    zero_tail(values.s, j);
                    bool more = false;
                    auto step = [&](auto group) {
                        constexpr int g = decltype(group)::value;
                        if (!products(group, values.s, j > 0)) return;
                        if (j + 1 == nt[g]) return tc_commit_if(&sh->o_full[g], issue);
                        if (!more && !there(keys)) return;
                        more = true;
                        scores(group, keys.s);
                        if (j + 2 == nt[g]) tc_commit_if(&sh->q_empty[g], issue);
                    };
                    if (j < nt[0]) step(Group0{});
                    if (j < nt[1] && !failed) step(Group1{});
                    if (failed) break;
                    tc_commit_if(&sh->kv_empty[values.s], issue);
                    if (more) {
                        tc_commit_if(&sh->kv_empty[keys.s], issue);
                        keys.advance(2);
                    }
                    values.advance(j + 2 < n ? 2 : 1);
                }
            } else {  // a key tile is one group's, and the next one the other's
                if (!first_scores(Group0{}, keys.s, nt[0])) break;
                tc_commit_if(&sh->kv_empty[keys.s], issue);
                keys.advance(1);
                if (n > 1) {
                    if (!there(keys) || !first_scores(Group1{}, keys.s, nt[1])) break;
                    tc_commit_if(&sh->kv_empty[keys.s], issue);
                    keys.advance(2);
                }
                for (int j = 0; j < n; j++) {
                    if (!there(values)) break;
                    zero_tail(values.s, j);
                    auto step = [&](auto group) {
                        constexpr int g = decltype(group)::value;
                        if (!products(group, values.s, j >= 2)) return;
                        tc_commit_if(&sh->kv_empty[values.s], issue);
                        if (j + 2 >= n) return tc_commit_if(&sh->o_full[g], issue);
                        if (!there(keys)) return;
                        scores(group, keys.s);
                        tc_commit_if(&sh->kv_empty[keys.s], issue);
                        keys.advance(2);
                        if (j + 4 >= n) tc_commit_if(&sh->q_empty[g], issue);
                    };
                    if (j & 1) step(Group1{});
                    else step(Group0{});
                    if (failed) break;
                    values.advance(j + 2 < n ? 2 : 1);
                }
            }
            if (failed) break;
            const int on = begin.s + 2 * n;
            begin.s = on % STAGES;
            begin.phase ^= (uint32_t)(on / STAGES) & 1;
        }
    } else if (warp == PA_SCHED_WARP) {
        int slot = 0;
        uint32_t phase = 1;
        auto announce = [&](const PromptItem& item) {
            if (!pa_wait(&sh->item_empty[slot], phase)) {
                failed = true;
                return false;
            }
            if (lane == 0) {
                sh->items[slot] = item;
                g_mbar_arrive(&sh->item_full[slot]);
            }
            if (++slot == PA_ITEMS) slot = 0, phase ^= 1;
            return true;
        };
        if (TREE) {
            tree_items(t, announce);
        } else {
            PromptSchedule schedule{t};
            schedule.begin();
            for (int i = blockIdx.x; schedule.find(i, it);) {
                unsigned int ahead = 0;
                if (lane == 0) ahead = atomicAdd(&t.sched[0], 1u);
                if (!announce(it)) break;
                i = (int)(gridDim.x + __shfl_sync(0xFFFFFFFFu, ahead, 0));
            }
            __threadfence();
            if (lane == 0 && atomicAdd(&t.sched[1], 1u) == gridDim.x - 1) {  // the last one leaves the counters as it found them
                t.sched[0] = 0;
                t.sched[1] = 0;
            }
        }
        if (!failed) {
            it = PromptItem{};
            it.last = 1;
            announce(it);
        }
    }
    if (failed) {
        if (lane == 0) report_status(p.status, STATUS_GEMM_PIPE_TIMEOUT);
        drain_after_abort();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == PA_MMA_WARP) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

}  // namespace wf
