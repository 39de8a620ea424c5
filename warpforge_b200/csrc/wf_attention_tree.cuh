// Attention of a few new tokens per sequence over a long cache.
//
// Bound by HBM: every key and value is read once, 4 dim bytes for 4 dim flops a row.  The rows of a sequence and kv head (its new tokens times the
// heads of the group) are padded to 16 or 32 and multiplied by mma.sync, 16 keys at a time; a tile of 5th-generation tensor cores has 128 rows, of which
// one decoded token fills one to eight.  More than 32 rows go to the kernel of wf_attention_prompt.cuh.  (One token of 48 sequences of 31 to 4000 tokens, 64 / 8 heads of
// 128: 419 MB in 73 us, 5.7 TB/s, 0.88 of a copy's rate.  One of 32 / 32 heads at 512 tokens: 9.3 us, of which 3.5 are a launch and the rest one SM's walk through 33 tiles.)
//
// The units are cut as wf_attention_line.cuh says.  Inside a CTA four warps walk its share and have TMA fill a ring of tiles ahead, across the ends of
// units too; eight others take the tiles of a piece in turn.
#pragma once
#include "wf_attention_line.cuh"
#include "wf_gemm_core.cuh"

namespace wf {

constexpr int TA_KEYS = 16;  // of a tile
constexpr int TA_WARPS = 8, TA_LOADERS = 4;  // warps that multiply, warps that walk and load
constexpr int TA_THREADS = (TA_WARPS + TA_LOADERS) * 32;
// Registers: 168 a thread at launch; the warps that multiply take what the others give back (256 x 216 + 128 x 72 = 384 x 168).
constexpr int TA_MULTIPLY_REGS = 216, TA_WALK_REGS = 72;
constexpr int TA_MERGE_BYTES = 64 * 1024;
constexpr int TA_SEGMENTS = 2;     // announced ahead
// When units are cut (line_is_cut).  Microseconds whole / cut, heads of 128: one sequence of 32 heads with 300, 600, 1000, 2000 tokens 7.2 / 8.7, 9.4 / 9.1, 11.9 / 10.7,
// 20.3 / 12.8; 8, 16, 18, 20, 24 sequences of 8 heads with 1000 tokens 12.8 / 13.4, 15.5 / 20.1, 16.6 / 21.5, 24.9 / 22.5, 25.7 / 25.8; 16 with 1800 23.4 / 28.2; one with
// 1250 beside 15 with 200 14.4 / 12.3.
constexpr int TA_CUT_TILES = 40, TA_CUT_ANYWAY = 96;
constexpr float TA_RESCALE = 8.f;  // the running maximum is followed when it has grown by this many powers of two
// CHUNKS of 64 elements of the head's dimension; MT blocks of 16 rows
template <int CHUNKS, int MT> struct TreeShape {
    static constexpr int DIM = CHUNKS * 64, ROWS = 16 * MT;
    static constexpr int SLOT_BYTES = 2 * CHUNKS * TA_KEYS * 128;  // keys and values of a tile
    static constexpr int Q_BYTES = ROWS * DIM * 2;
    static constexpr int FIT = (227 * 1024 - TA_MERGE_BYTES - TA_SEGMENTS * Q_BYTES - 4 * 1024) / SLOT_BYTES;
    // A slot belongs to one loader, and within a segment to one warp, lap after lap: a barrier's parity tells the laps apart only for those that wait for every one.
    static constexpr int SLOTS = FIT > 32 ? 32 : FIT / TA_WARPS * TA_WARPS;
    static constexpr int SETS = TA_MERGE_BYTES / (ROWS * DIM * 4) < TA_WARPS ? TA_MERGE_BYTES / (ROWS * DIM * 4) : TA_WARPS;  // warps whose sums lie in shared memory at a time
    static constexpr int SMEM = SLOTS * SLOT_BYTES + TA_MERGE_BYTES + TA_SEGMENTS * Q_BYTES + 1024;
    static constexpr int PIECE = ROWS * (DIM + 2);  // floats of a piece in memory
    // What a unit costs beyond its tiles, in tiles (queries, first tile's way, the fold over eight warps).  16 rows, with 2 / 4 / 8 / 12 / 16 / 24: 91 / 85 / 75 / 73 / 73 / 75 us
    // for one token of 48 sequences of 31 to 4000 tokens; 32 rows of 30 sequences of 10 to 5000, with 16 / 24 / 32 / 48: 72 / 65 / 63 / 61, but 33.2 / 32.8 / 33.2 / 33.3 for 20 alike.
    static constexpr int UNIT_TILES = 16 * MT;
    static_assert(SETS == TA_WARPS || 2 * SETS == TA_WARPS, "one round of folding");
    static_assert(SLOTS >= TA_WARPS && SLOTS % TA_WARPS == 0 && SLOTS % TA_LOADERS == 0, "slots for every warp and loader");
};
// What a CTA has of a unit.
struct alignas(16) TreeSegment {
    int row0, rows, context, seq;  // of the sequence; context < 0: a sequence that cannot be, its rows are zeros
    int head, first;               // first of the sequence's rows * group that the unit has
    int from, to, tiles;           // of the unit
    int slot, phase;               // of the first tile in the ring
    int last;                      // no more work
};

struct TreeTiles {
    TreeParams p;
    TreeCuts c;
};

// By the thread whose `issue` is non-zero; the whole warp comes here with the same operands, which then sit in uniform registers (issued by four
// lanes with operands of their own, the loads of a tile took 670 cycles and set the pace; HBM gives an SM a tile in 345).
__device__ __forceinline__ void ta_load(uint32_t dst, const CUtensorMap* map, int x, int z, uint32_t bar, uint32_t issue) {
    asm volatile("{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %6, 0;\n\t"
                 "@e cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n\t}" ::"r"(dst), "l"(map),
                 "r"(x), "r"(0), "r"(z), "r"(bar), "r"(issue)
                 : "memory");
}
__device__ __forceinline__ void ta_expect(uint32_t bar, uint32_t bytes, uint32_t issue) {
    asm volatile("{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %2, 0;\n\t@e mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t}" ::"r"(bar), "r"(bytes), "r"(issue) : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ta_copy16(uint32_t dst, const void* src, bool real) {  // zeros where there is nothing
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void ta_sync() { asm volatile("barrier.cta.sync 1, %0;" ::"n"(TA_WARPS * 32) : "memory"); }
__device__ __forceinline__ bool ta_sync_or(bool v) {  // the same answer for all warps that multiply
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(r) : "r"((uint32_t)v), "n"(TA_WARPS * 32) : "memory");
    return r != 0;
}

template <int CHUNKS, int MT> struct TreeShared {
    typedef TreeShape<CHUNKS, MT> Shape;
    uint64_t full[Shape::SLOTS], empty[Shape::SLOTS];
    uint64_t seg_full[TA_SEGMENTS], seg_empty[TA_SEGMENTS];
    TreeSegment segments[TA_SEGMENTS];
    float warp_max[Shape::SETS][Shape::ROWS], warp_sums[Shape::SETS][Shape::ROWS];
    unsigned long long odd_rows;
    // [number % ..] = number: the segment of that number has pages outside the cache; nobody is more than TA_SEGMENTS ahead of another
    int bad_pages[2 * TA_SEGMENTS];
    __device__ __forceinline__ volatile int& bad_page(int number) { return *reinterpret_cast<volatile int*>(&bad_pages[(unsigned)number % (2 * TA_SEGMENTS)]); }
};

// The warps that walk the line: the first announces this CTA's segments, all fetch their queries and have their tiles loaded, by turns.  True: all went
// well.
template <int CHUNKS, int MT>
__device__ __forceinline__ bool tree_load(const TreeTiles& t, TreeShared<CHUNKS, MT>* sh, const CUtensorMap* k_map, const CUtensorMap* v_map, uint32_t ring, uint32_t q_smem, int loader) {
    typedef TreeShape<CHUNKS, MT> Shape;
    constexpr int ROWS = Shape::ROWS, DIM = Shape::DIM;
    const TreeParams& p = t.p;
    const int lane = threadIdx.x & 31, heads = p.cache.kv_heads, group = p.group;
    const uint32_t issue = elect_one();
    int seg = 0, slot = 0, number = 0;
    uint32_t seg_phase = 1, phase = 1;
    bool cut = false;  // a unit that begins here goes on in the next share
    const bool ok = walk_line<TA_KEYS>(p, ROWS, Shape::UNIT_TILES, t.c.may_cut, [&](const LineUnit& u) {
        const int keys = u.q.context < 0 ? 0 : u.q.context + u.q.rows, count = min(ROWS, u.q.rows * group - u.first);
        // the page of a lane's tile, asked for before anything is waited for
        const int* const table = u.q.place.table;
        int tile = u.from + lane, page = 0;
        if (tile < u.to && keys > 0) page = table[tile * TA_KEYS >> p.cache.page_shift];
        if (!__all_sync(0xFFFFFFFFu, g_mbar_wait(&sh->seg_empty[seg], seg_phase))) return false;
        if (loader == 0 && lane == 0) {
            TreeSegment& d = sh->segments[seg];
            d.row0 = u.q.row0, d.rows = u.q.rows, d.context = u.q.context, d.seq = u.seq, d.head = u.head, d.first = u.first;
            d.from = u.from, d.to = u.to, d.tiles = u.tiles, d.slot = slot, d.phase = (int)phase ^ 1, d.last = 0;
            g_mbar_arrive(&sh->seg_full[seg]);
            if (u.from == 0 && u.to < u.tiles) leave_cut(t.c, u, count);
        }
        cut |= u.from == 0 && u.to < u.tiles;
        __syncwarp();
        // the queries: rows of 16-byte pieces, swizzled by the row
        const bf16* q0 = p.q + (size_t)u.q.row0 * p.q_stride + (size_t)u.head * group * p.cache.dim;
#pragma unroll 1
        for (int i = loader * 32 + lane; i < ROWS * (DIM / 8); i += 32 * TA_LOADERS) {
            const int r = i / (DIM / 8), piece = i % (DIM / 8), token = p.token_of(u.first + r);
            const bool real = r < count && piece * 8 < p.cache.dim;
            ta_copy16(q_smem + (uint32_t)(seg * Shape::Q_BYTES + r * DIM * 2 + ((piece ^ (r & 7)) << 4)),
                      real ? q0 + (size_t)token * p.q_stride + (size_t)((u.first + r) - token * group) * p.cache.dim + piece * 8 : p.q, real);
        }
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(g_smem_u32(&sh->seg_full[seg])) : "memory");
#pragma unroll 1
        for (int t0 = u.from; t0 < u.to; t0 += 32) {
            if (t0 > u.from) {
                tile = t0 + lane;
                page = tile < u.to && keys > 0 ? table[tile * TA_KEYS >> p.cache.page_shift] : 0;
            }
            if (page < 0 || page >= p.cache.pages) {  // never followed: the unit's rows go key by key
                sh->bad_page(number) = number;
                page = 0;
            }
            __syncwarp();  // the mark is there before a tile that this warp has loaded
            const int z = ((page * heads + u.head) << p.cache.page_shift) + (tile * TA_KEYS & ((1 << p.cache.page_shift) - 1));  // below 2^31: check_cache
            const int n = min(32, u.to - t0);
#pragma unroll 1
            for (int i = 0; i < n; i++) {
                const int row = __shfl_sync(0xFFFFFFFFu, z, i);
                if (slot % TA_LOADERS == loader) {
                    if (!__all_sync(0xFFFFFFFFu, g_mbar_wait(&sh->empty[slot], phase))) return false;
                    const uint32_t bar = g_smem_u32(&sh->full[slot]), to_slot = ring + (uint32_t)(slot * Shape::SLOT_BYTES);
                    ta_expect(bar, Shape::SLOT_BYTES, issue);
#pragma unroll
                    for (int c = 0; c < 2 * CHUNKS; c++) ta_load(to_slot + (uint32_t)(c * TA_KEYS * 128), c < CHUNKS ? k_map : v_map, 64 * (c % CHUNKS), row, bar, issue);
                }
                if (++slot == Shape::SLOTS) slot = 0, phase ^= 1;
            }
        }
        number++;
        if (++seg == TA_SEGMENTS) seg = 0, seg_phase ^= 1;
        return true;
    });
    if (t.c.may_cut && !cut && loader == 0 && lane == 0) t.c.cuts[blockIdx.x].first_cta = -1;  // where a wait ran out, too: tree_join_kernel follows it
    if (!ok || !__all_sync(0xFFFFFFFFu, g_mbar_wait(&sh->seg_empty[seg], seg_phase))) return false;
    if (loader == 0 && lane == 0) {
        sh->segments[seg].last = 1;
        g_mbar_arrive(&sh->seg_full[seg]);
    }
    g_mbar_arrive(&sh->seg_full[seg]);
    return true;
}

template <int CHUNKS, int MT>
__global__ void __launch_bounds__(TA_THREADS, 1) tree_tiles_kernel(const __grid_constant__ TreeTiles t, const __grid_constant__ CUtensorMap k_map,
                                                                   const __grid_constant__ CUtensorMap v_map) {
    typedef TreeShape<CHUNKS, MT> Shape;
    constexpr int DIM = Shape::DIM, ROWS = Shape::ROWS, SLOTS = Shape::SLOTS, SLOT_BYTES = Shape::SLOT_BYTES, N_TILES = DIM / 8, SETS = Shape::SETS;
    constexpr bool Q_KEPT = MT * CHUNKS <= 2;  // queries stay in registers; else they are read again with every tile
    extern __shared__ uint8_t raw[];
    __shared__ TreeShared<CHUNKS, MT> sh_;
    TreeShared<CHUNKS, MT>* const sh = &sh_;
    const TreeParams& p = t.p;
    const int tid = threadIdx.x, warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0), lane = tid & 31, g = lane >> 2, quad = lane & 3;
    const uint32_t ring = (g_smem_u32(raw) + 1023u) & ~1023u, q_smem = ring + SLOTS * SLOT_BYTES;
    float* const merge = reinterpret_cast<float*>(raw + (ring - g_smem_u32(raw)) + SLOTS * SLOT_BYTES + TA_SEGMENTS * Shape::Q_BYTES);
    if (tid < SLOTS) {
        g_mbar_init(&sh->full[tid], 1);
        g_mbar_init(&sh->empty[tid], 1);
    } else if (tid >= 32 && tid < 32 + TA_SEGMENTS) {
        g_mbar_init(&sh->seg_full[tid - 32], 32 * TA_LOADERS + 1);  // every lane's copies of queries, and the words
        g_mbar_init(&sh->seg_empty[tid - 32], TA_WARPS);
    } else if (tid == 64) {
        sh->odd_rows = 0;
        for (int i = 0; i < 2 * TA_SEGMENTS; i++) sh->bad_pages[i] = -1;
        prefetch_tensormap(&k_map);
        prefetch_tensormap(&v_map);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    __syncthreads();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (warp >= TA_WARPS) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(TA_WALK_REGS));
        if (!tree_load<CHUNKS, MT>(t, sh, &k_map, &v_map, ring, q_smem, warp - TA_WARPS)) {
            if (lane == 0) report_status(p.status, STATUS_GEMM_PIPE_TIMEOUT);
            drain_after_abort();
        }
        return;
    }

    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(TA_MULTIPLY_REGS));
    const float scale = p.scale_log2;
    const int d = p.cache.dim, group = p.group;
    // ldmatrix: a lane's row and 16-byte piece, swizzled
    const int matrix = lane >> 3, mrow = lane & 7;
    const uint32_t k_row = (uint32_t)(((matrix >> 1) * 8 + mrow) * 128), v_row = (uint32_t)(((matrix & 1) * 8 + mrow) * 128) + CHUNKS * TA_KEYS * 128;
    const uint32_t q_row = (uint32_t)(((matrix & 1) * 8 + mrow) * DIM * 2);
    int seg = 0;
    uint32_t seg_phase = 0;
    bool failed = false;
#pragma unroll 1
    for (int number = 0;; number++) {
        failed |= !g_mbar_wait(&sh->seg_full[seg], seg_phase);
        if (ta_sync_or(failed)) {  // `merge` is free again, too
            failed = true;
            break;
        }
        const TreeSegment w = sh->segments[seg];
        if (w.last) break;
        const int keys = w.context < 0 ? 0 : w.context + w.rows, count = min(ROWS, w.rows * group - w.first);
        const uint32_t q_at = q_smem + (uint32_t)(seg * Shape::Q_BYTES) + q_row;
        auto load_q = [&](int i, int k, uint32_t(&a)[4]) { ldmatrix4(q_at + (uint32_t)(i * 16 * DIM * 2) + (uint32_t)(((2 * k + (matrix >> 1)) ^ mrow) << 4), a); };
        uint32_t q[MT][Q_KEPT ? DIM / 16 : 1][4];
        if (Q_KEPT)
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int k = 0; k < DIM / 16; k++) load_q(i, k, q[i][Q_KEPT ? k : 0]);
        float o[MT][N_TILES][4], m[MT][2], l[MT][2];
#pragma unroll
        for (int i = 0; i < MT; i++) {
            m[i][0] = m[i][1] = -INFINITY;
            l[i][0] = l[i][1] = 0.f;
#pragma unroll
            for (int n = 0; n < N_TILES; n++) o[i][n][0] = o[i][n][1] = o[i][n][2] = o[i][n][3] = 0.f;
        }
        int slot = w.slot + warp;
        uint32_t phase = (uint32_t)w.phase;
        if (slot >= SLOTS) slot -= SLOTS, phase ^= 1;
#pragma unroll 1
        for (int tile = w.from + warp; tile < w.to; tile += TA_WARPS) {
            if (!__all_sync(0xFFFFFFFFu, g_mbar_wait(&sh->full[slot], phase))) {
                failed = true;
                break;
            }
            const uint32_t base = ring + (uint32_t)(slot * SLOT_BYTES);
            float s[MT][2][4] = {};
#pragma unroll
            for (int k0 = 0; k0 < DIM / 16; k0 += 4) {
                uint32_t b[4][4];
#pragma unroll
                for (int k = 0; k < 4; k++) ldmatrix4(base + (uint32_t)(k0 / 4 * TA_KEYS * 128) + k_row + (uint32_t)(((2 * k + (matrix & 1)) ^ mrow) << 4), b[k]);
#pragma unroll
                for (int k = 0; k < 4; k++)
#pragma unroll
                    for (int i = 0; i < MT; i++) {
                        if (!Q_KEPT) load_q(i, k0 + k, q[i][0]);
                        mma_bf16(s[i][0], q[i][Q_KEPT ? k0 + k : 0], b[k][0], b[k][1]);
                        mma_bf16(s[i][1], q[i][Q_KEPT ? k0 + k : 0], b[k][2], b[k][3]);
                    }
            }
            const int key0 = tile * TA_KEYS;
            if (key0 + TA_KEYS > w.context) {  // new tokens, or none
#pragma unroll
                for (int i = 0; i < MT; i++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const int r = 16 * i + g + 8 * e, token = p.token_of(w.first + r);
                        const uint64_t sees = r < count && keys > 0 ? ancestors_of(p, w.row0 + token, token) & ((uint64_t)-1 >> (64 - w.rows)) : 0;
#pragma unroll
                        for (int c = 0; c < 4; c++) {
                            const int j = key0 + 8 * (c >> 1) + 2 * quad + (c & 1) - w.context;
                            if (!(w.context >= 0 && (j < 0 || (j < TREE_MAX_DRAFTS && (sees >> j & 1))))) s[i][c >> 1][2 * e + (c & 1)] = -INFINITY;
                        }
                    }
                if (key0 + TA_KEYS > keys) {  // values behind the last key: their weights are 0, and 0 x whatever lies there has to be 0
#pragma unroll 1
                    for (int e = max(0, keys - key0) * 8 * CHUNKS + lane; e < TA_KEYS * 8 * CHUNKS; e += 32) {
                        const int row = e / (8 * CHUNKS), piece = e % (8 * CHUNKS);
                        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(base + (uint32_t)((CHUNKS + piece / 8) * TA_KEYS * 128 + row * 128 + piece % 8 * 16)), "r"(0) : "memory");
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                }
            }
            bool grows = false;
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int e = 0; e < 2; e++)
                    grows |= (fmaxf(fmaxf(s[i][0][2 * e], s[i][0][2 * e + 1]), fmaxf(s[i][1][2 * e], s[i][1][2 * e + 1])) - m[i][e]) * scale > TA_RESCALE;
            if (__any_sync(0xFFFFFFFFu, grows)) {
#pragma unroll
                for (int i = 0; i < MT; i++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float top = fmaxf(fmaxf(s[i][0][2 * e], s[i][0][2 * e + 1]), fmaxf(s[i][1][2 * e], s[i][1][2 * e + 1]));
                        top = fmaxf(m[i][e], top);
                        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
                        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
                        const float keep = line_ex2((m[i][e] - (top == -INFINITY ? 0.f : top)) * scale);
                        m[i][e] = top;
                        l[i][e] *= keep;
#pragma unroll
                        for (int n = 0; n < N_TILES; n++) {
                            o[i][n][2 * e] *= keep;
                            o[i][n][2 * e + 1] *= keep;
                        }
                    }
            }
            uint32_t a[MT][4];
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const float ref = m[i][e] == -INFINITY ? 0.f : m[i][e] * scale;
#pragma unroll
                    for (int n = 0; n < 2; n++) {
                        const float x = line_ex2(fmaf(s[i][n][2 * e], scale, -ref)), y = line_ex2(fmaf(s[i][n][2 * e + 1], scale, -ref));
                        l[i][e] += x + y;
                        a[i][2 * n + e] = pack_bf16(x, y);
                    }
                }
#pragma unroll
            for (int n0 = 0; n0 < N_TILES / 2; n0 += 4) {
                uint32_t b[4][4];
#pragma unroll
                for (int n = 0; n < 4; n++) ldmatrix4_trans(base + (uint32_t)(n0 / 4 * TA_KEYS * 128) + v_row + (uint32_t)(((2 * n + (matrix >> 1)) ^ mrow) << 4), b[n]);
#pragma unroll
                for (int n = 0; n < 4; n++)
#pragma unroll
                    for (int i = 0; i < MT; i++) {
                        mma_bf16(o[i][2 * (n0 + n)], a[i], b[n][0], b[n][1]);
                        mma_bf16(o[i][2 * (n0 + n) + 1], a[i], b[n][2], b[n][3]);
                    }
            }
            __syncwarp();
            if (lane == 0) g_mbar_arrive(&sh->empty[slot]);
            slot += TA_WARPS;
            if (slot >= SLOTS) slot -= SLOTS, phase ^= 1;
        }
        __syncwarp();
        if (lane == 0) g_mbar_arrive(&sh->seg_empty[seg]);  // the queries
        if (++seg == TA_SEGMENTS) seg = 0, seg_phase ^= 1;
        if (sh->bad_page(number) == number) l[0][0] = l[0][1] = l[MT - 1][0] = l[MT - 1][1] = __uint_as_float(0x7FC00000u);

        // The warps' sums together.  Where they do not all fit shared memory the upper half hands its to the lower half first.
        auto write_sums = [&](int set) {
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    // the threads of a row have followed the same maximum
                    l[i][e] += __shfl_xor_sync(0xFFFFFFFFu, l[i][e], 1);
                    l[i][e] += __shfl_xor_sync(0xFFFFFFFFu, l[i][e], 2);
                    const int r = 16 * i + g + 8 * e;
                    if (quad == 0) {
                        sh->warp_max[set][r] = m[i][e];
                        sh->warp_sums[set][r] = l[i][e];
                    }
                    float2* row = reinterpret_cast<float2*>(merge + (size_t)(set * ROWS + r) * DIM);
#pragma unroll
                    for (int n = 0; n < N_TILES; n++) row[(n ^ (r & 3)) * 4 + quad] = make_float2(o[i][n][2 * e], o[i][n][2 * e + 1]);
                }
        };
        if (SETS < TA_WARPS) {
            if (warp >= SETS) write_sums(warp - SETS);
            ta_sync();
            if (warp < SETS) {
#pragma unroll
                for (int i = 0; i < MT; i++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const int r = 16 * i + g + 8 * e;
                        const float other = sh->warp_max[warp][r], top = fmaxf(m[i][e], other), ref = top == -INFINITY ? 0.f : top;
                        const float keep = line_ex2((m[i][e] - ref) * scale), take = line_ex2((other - ref) * scale);
                        m[i][e] = top;
                        l[i][e] = l[i][e] * keep + (quad == 0 ? sh->warp_sums[warp][r] * take : 0.f);
                        const float2* row = reinterpret_cast<const float2*>(merge + (size_t)(warp * ROWS + r) * DIM);
#pragma unroll
                        for (int n = 0; n < N_TILES; n++) {
                            const float2 v = row[(n ^ (r & 3)) * 4 + quad];
                            o[i][n][2 * e] = o[i][n][2 * e] * keep + v.x * take;
                            o[i][n][2 * e + 1] = o[i][n][2 * e + 1] * keep + v.y * take;
                        }
                    }
            }
            ta_sync();
        }
        if (warp < SETS) write_sums(warp);
        ta_sync();
        const bool whole = w.from == 0 && w.to == w.tiles;
        // a CTA has at most two pieces of cut units: one that began before its share, one that begins in it
        float* const piece = t.c.pieces + ((size_t)blockIdx.x * 2 + (w.from == 0)) * Shape::PIECE;
        auto store = [&](int r, int col, const float4& x, float sum, float top) {  // four elements of a row, or zeros where it sees nothing
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            uint32_t largest = sum < INFINITY && !scores_too_large(top, scale) ? 0 : 0x7F800000u;
            largest = max(max(largest, __float_as_uint(x.x) & 0x7FFFFFFFu), max(__float_as_uint(x.y) & 0x7FFFFFFFu, max(__float_as_uint(x.z) & 0x7FFFFFFFu, __float_as_uint(x.w) & 0x7FFFFFFFu)));
            if (largest >= 0x7F800000u) atomicOr(&sh->odd_rows, 1ull << r);
            const int token = p.token_of(w.first + r);
            bf16* to = p.out + ((size_t)(w.row0 + token) * p.q_heads + w.head * group + (w.first + r) - token * group) * d + col;
            *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16(x.x * inv, x.y * inv), pack_bf16(x.z * inv, x.w * inv));
        };
        constexpr int PER_ROW = DIM / 4;  // threads of a row
#pragma unroll 1
        for (int i = tid; i < count * PER_ROW; i += TA_WARPS * 32) {
            const int r = i / PER_ROW, n = i % PER_ROW;
            float top = -INFINITY, sum = 0.f, tops[SETS];
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int c = 0; c < SETS; c++) top = fmaxf(top, tops[c] = sh->warp_max[c][r]);
            const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
            for (int c = 0; c < SETS; c++) {
                const float keep = line_ex2((tops[c] - ref) * scale);
                sum += sh->warp_sums[c][r] * keep;
                const float4 v = *reinterpret_cast<const float4*>(merge + (size_t)(c * ROWS + r) * DIM + ((n >> 1) ^ (r & 3)) * 8 + (n & 1) * 4);
                x.x += v.x * keep, x.y += v.y * keep, x.z += v.z * keep, x.w += v.w * keep;
            }
            if (whole) {
                if (4 * n < d) store(r, 4 * n, x, sum, top);
            } else {
                *reinterpret_cast<float4*>(piece + r * DIM + 4 * n) = x;
                if (n == 0) {
                    piece[ROWS * DIM + r] = top;
                    piece[ROWS * (DIM + 1) + r] = sum;
                }
            }
        }
        ta_sync();
        const unsigned long long odd = sh->odd_rows;
        if (odd) {
            // An Inf or a NaN in a row's sums may have come from a key that it does not see (0 x Inf), or from a page that is not in the cache: key by key.
            ta_sync();
            if (tid == 0) sh->odd_rows = 0;
            KeyPlace place;
            place.table = p.tables + (size_t)w.seq * p.table_stride;
            place.first = 0;
#pragma unroll 1
            for (int r = warp; r < count; r += TA_WARPS) {
                if (!(odd >> r & 1)) continue;
                const int token = p.token_of(w.first + r), h = w.head * group + (w.first + r) - token * group;
                attend_row(p.cache, place, p.q + (size_t)(w.row0 + token) * p.q_stride + (size_t)h * d, p.out + ((size_t)(w.row0 + token) * p.q_heads + h) * d, w.head, keys,
                           scale, p.status, SeesAncestors{w.context, ancestors_of(p, w.row0 + token, token) & ((uint64_t)-1 >> (64 - w.rows))});
            }
        }
    }
    if (failed) {
        if (lane == 0) report_status(p.status, STATUS_GEMM_PIPE_TIMEOUT);
        drain_after_abort();
    }
}

}  // namespace wf
