// wf_qk_norm_rope: what happens to q, k and v between their projections and the attention, in one pass.  Per token and head of q and k
//   x' = x / sqrt(mean(x^2) + eps) * gamma,   (a, b) -> (a c - b s, b c + a s) for the pairs of the first rot elements
// in fp32, rounded once to bf16; v is rounded only; k and v go to their slots in the cache.
// Bound by HBM for fp32 rows (2048 tokens of 64 + 2 x 8 heads of 128: 127 MB in 24.6 us, 5.15 TB/s, 0.79 of a copy's rate), by the launch and one chain of
// loads (slot and position, table row, store) for a token alone: 3.4 us.
#include <algorithm>

#include "wf_attention.cuh"

namespace wf {

CacheView cache_layer(const wf_kv_cache& cache, int layer);
int check_kv_cache(Context* c, const char* what, const wf_kv_cache* cache, int layer, bool packed_too);

struct RopeParams {
    const void *q, *k, *v;
    int64_t q_stride, k_stride, v_stride;
    const float *gamma_q, *gamma_k;
    const float2* rope;
    int64_t rope_rows;
    const int* positions;
    const int64_t* slots;
    bf16* q_out;
    CacheView cache;
    int64_t tokens;
    int q_heads, k_heads;  // 0: that part is not wanted
    int rot, norm, adjacent;
    int sets, batches;  // warps of a token, batches of heads of a warp
    float eps;
    int* status;
};

// Two neighbouring elements.
template <class X, bool VEC> __device__ __forceinline__ float2 load_pair(const X* p) {
    if (!VEC) return make_float2((float)p[0], (float)p[1]);
    float2 v;
    if (sizeof(X) == 4) {
        asm volatile("ld.global.cs.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "l"(p));
        return v;
    }
    uint32_t w;
    asm volatile("ld.global.cs.u32 %0, [%1];" : "=r"(w) : "l"(p));
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}

__device__ __forceinline__ float2 mul_pair(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 w, x, y;\n\tmov.b64 {%0, %1}, w;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 fma_pair(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\tfma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}

// A group of LANES lanes has a head, four elements a lane: two pairs that are rotated, (i, i + rot/2) and (i + 1, i + 1 + rot/2) or two adjacent ones, so
// that no lane needs another's, or four that are not.  A warp takes HEADS heads of one token and of one kind (q, k or v) at a time: what the kinds differ in
// is settled outside, and four elements are two operations on pairs.  (With the kinds mixed, a head took 121 instructions a lane and the kernel was bound by
// them: 27.9 us at the size above, 8.6 instead of 6.0 us at 777 tokens of 28 + 2 x 4 bf16 heads of 96.)
constexpr int ROPE_WARPS = 4, ROPE_UNROLL = 4, ROPE_WARPS_PER_SM = 64, ROPE_MOST_BATCHES = 5;
// DIM: 4 * LANES where all of the head is rotated or nothing, else 0.  The test whether a lane turns costs registers: in the kernel for whole heads 26.4 instead of
// 24.7 us at the size above; with half of each head rotated that size takes 27.3.
template <class X, bool VEC, int LANES, int DIM>
__global__ void __launch_bounds__(ROPE_WARPS * 32) qk_norm_rope_kernel(const __grid_constant__ RopeParams p) {
    constexpr int SIDE = 32 / LANES, HEADS = ROPE_UNROLL * SIDE;  // heads beside one another in a warp, heads of a batch
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int lane = threadIdx.x & (LANES - 1), side = (threadIdx.x & 31) / LANES;
    const int d = DIM ? DIM : p.cache.dim;
    const bool mine = DIM || 4 * lane < d;
    const int64_t unit = (int64_t)blockIdx.x * ROPE_WARPS + (threadIdx.x >> 5);
    const int64_t t = unit / p.sets;
    if (t >= p.tokens) return;
    const int q_batches = (p.q_heads + HEADS - 1) / HEADS, k_batches = (p.k_heads + HEADS - 1) / HEADS;
    const int first = (int)(unit - t * p.sets) * p.batches, end = min(q_batches + 2 * k_batches, first + p.batches);
    // the elements: a0, a0 + 1 and b0, b0 + 1
    const bool turns = 4 * lane < p.rot, apart = turns && !p.adjacent;
    const int a0 = !mine ? 0 : apart ? 2 * lane : 4 * lane, b0 = !mine ? 0 : apart ? p.rot / 2 + 2 * lane : 4 * lane + 2;
    int64_t slot = p.slots ? p.slots[t] : t;
    int64_t pos = p.rot ? p.positions[t] : 0;
    float2 x[ROPE_UNROLL][2];
    auto ask = [&](int batch) {
        const int kind = batch < q_batches ? 0 : batch < q_batches + k_batches ? 1 : 2, h0 = (batch - (kind == 0 ? 0 : kind == 1 ? q_batches : q_batches + k_batches)) * HEADS + side;
        const int last = (kind ? p.k_heads : p.q_heads) - 1;
        const X* const token = kind == 0 ? static_cast<const X*>(p.q) + t * p.q_stride : kind == 1 ? static_cast<const X*>(p.k) + t * p.k_stride : static_cast<const X*>(p.v) + t * p.v_stride;
#pragma unroll
        for (int u = 0; u < ROPE_UNROLL; u++) {
            const int at = min(h0 + u * SIDE, last) * d;  // heads behind the last are read as the last, and not stored
            x[u][0] = load_pair<X, VEC>(token + (at + a0));
            x[u][1] = load_pair<X, VEC>(token + (at + b0));
        }
    };
    ask(first);
    const bool bad = (p.rot && (pos < 0 || pos >= p.rope_rows)) || (p.k_heads && slot >= p.cache.pages << p.cache.page_shift);
    if (bad) {
        if ((threadIdx.x & 31) == 0) report_status(p.status, STATUS_BAD_INDEX);
        slot = -1;
        pos = 0;
    }
    float4 cs = make_float4(1.f, 0.f, 1.f, 0.f);  // cosine and sine of the lane's two pairs, if they turn: 16 bytes of the row either way
    if (turns) cs = *reinterpret_cast<const float4*>(p.rope + (size_t)pos * (p.rot / 2) + 2 * lane);
    const int64_t place = slot < 0 ? 0 : (int64_t)p.cache.at(slot >> p.cache.page_shift, 0, (int)(slot & ((1 << p.cache.page_shift) - 1)));
#pragma unroll 1
    for (int batch = first; batch < end; batch++) {
        if (batch > first) ask(batch);
        const int kind = batch < q_batches ? 0 : batch < q_batches + k_batches ? 1 : 2, h0 = (batch - (kind == 0 ? 0 : kind == 1 ? q_batches : q_batches + k_batches)) * HEADS + side;
        if (kind < 2 && p.norm) {
            // The sums of squares of four heads in ten exchanges instead of twenty: with every exchange at a distance a lane passes on half of the sums that it has and adds
            // to the others, until it has one; that one is then brought to all lanes of the head.
            float s[ROPE_UNROLL];
#pragma unroll
            for (int u = 0; u < ROPE_UNROLL; u++) {
                const float2 sq = fma_pair(x[u][1], x[u][1], mul_pair(x[u][0], x[u][0]));
                s[u] = mine ? sq.x + sq.y : 0.f;
            }
            const bool hi = lane & (LANES / 2), hi2 = lane & (LANES / 4);
            float t0 = hi ? s[2] : s[0], t1 = hi ? s[3] : s[1];
            t0 += __shfl_xor_sync(0xFFFFFFFFu, hi ? s[0] : s[2], LANES / 2);
            t1 += __shfl_xor_sync(0xFFFFFFFFu, hi ? s[1] : s[3], LANES / 2);
            float r = hi2 ? t1 : t0;
            r += __shfl_xor_sync(0xFFFFFFFFu, hi2 ? t0 : t1, LANES / 4);
#pragma unroll
            for (int o = LANES / 8; o > 0; o >>= 1) r += __shfl_xor_sync(0xFFFFFFFFu, r, o);
            r = rsqrtf(r / (float)d + p.eps);
            const float* const gamma = kind ? p.gamma_k : p.gamma_q;
            const float2 ga = gamma ? make_float2(gamma[a0], gamma[a0 + 1]) : make_float2(1.f, 1.f), gb = gamma ? make_float2(gamma[b0], gamma[b0 + 1]) : make_float2(1.f, 1.f);
#pragma unroll
            for (int u = 0; u < ROPE_UNROLL; u++) {
                const float inv = __shfl_sync(0xFFFFFFFFu, r, (u >> 1) * (LANES / 2) + (u & 1) * (LANES / 4), LANES);
                x[u][0] = mul_pair(mul_pair(x[u][0], make_float2(inv, inv)), ga);
                x[u][1] = mul_pair(mul_pair(x[u][1], make_float2(inv, inv)), gb);
            }
        }
        if (kind < 2 && (DIM ? p.rot != 0 : turns)) {  // a lane that does not turn is left alone: 0 x Inf would make a NaN of its others
            const float2 c = make_float2(cs.x, cs.z), s = make_float2(cs.y, cs.w), minus = make_float2(-cs.y, -cs.w);
#pragma unroll
            for (int u = 0; u < ROPE_UNROLL; u++) {
                const float2 a = x[u][0], b = x[u][1];
                if (p.adjacent) {
                    x[u][0] = make_float2(a.x * cs.x - a.y * cs.y, a.y * cs.x + a.x * cs.y);
                    x[u][1] = make_float2(b.x * cs.z - b.y * cs.w, b.y * cs.z + b.x * cs.w);
                } else {
                    x[u][0] = fma_pair(b, minus, mul_pair(a, c));
                    x[u][1] = fma_pair(a, s, mul_pair(b, c));
                }
            }
        }
        bf16* const to = kind == 0 ? p.q_out + t * p.q_heads * d : kind == 1 ? p.cache.keys + place : p.cache.values + place;
        const int64_t apart_heads = kind == 0 ? d : (int64_t)d << p.cache.page_shift;
        const int heads = !mine || (kind && slot < 0) ? 0 : kind ? p.k_heads : p.q_heads;
#pragma unroll
        for (int u = 0; u < ROPE_UNROLL; u++) {
            const int h = h0 + u * SIDE;
            if (h >= heads) continue;
            bf16* const row = to + h * apart_heads;
            *reinterpret_cast<uint32_t*>(row + a0) = bad ? 0u : pack_bf16(x[u][0].x, x[u][0].y);
            *reinterpret_cast<uint32_t*>(row + b0) = bad ? 0u : pack_bf16(x[u][1].x, x[u][1].y);
        }
    }
}

}  // namespace wf

using namespace wf;

extern "C" int wf_qk_norm_rope(int64_t ctx, const wf_qk_norm_rope_args* a, const wf_kv_cache* cache, int layer, int64_t stream) {
    Context* c = get_context(ctx);
    if (!c) return WF_ERR_INVALID_HANDLE;
    ScopedLock lock(c);
    if (!lock.ok) return WF_ERR_BUSY;
    WF_CUDA(c, cudaSetDevice(c->device));
    cudaStream_t s = resolve_stream(c, stream);
    const char* what = "qk_norm_rope";
    if (!a || !cache) return set_error(c, WF_ERR_INVALID_ARGUMENT, "%s: null arguments", what);
    if (a->tokens == 0) return WF_OK;
    const int rc = check_kv_cache(c, what, cache, layer, true);
    if (rc != WF_OK) return rc;
    if (a->x_dtype != WF_DTYPE_F32 && a->x_dtype != WF_DTYPE_BF16) return set_error(c, WF_ERR_INVALID_ARGUMENT, "%s: x_dtype %d", what, a->x_dtype);
    if (!a->k_dev != !a->v_dev || (!a->q_dev && !a->k_dev)) return set_error(c, WF_ERR_INVALID_ARGUMENT, "%s: q, or k and v, or all three", what);
    const int d = cache->head_dim, size = a->x_dtype == WF_DTYPE_F32 ? 4 : 2;
    if ((a->q_dev | a->k_dev | a->v_dev) & (size - 1)) return set_error(c, WF_ERR_INVALID_ARGUMENT, "%s: misaligned q, k or v", what);
    if (a->q_dev && (!a->q_out_dev || a->q_out_dev & 7)) return set_error(c, WF_ERR_INVALID_ARGUMENT, "%s: q_out must be an 8-byte aligned device address", what);
    if (a->tokens < 0 || a->tokens > (1LL << 31) - 1 || (a->q_dev && (a->q_heads < 1 || a->q_heads > 8192)))
        return set_error(c, WF_ERR_SHAPE, "%s: tokens=%lld q_heads=%d", what, (long long)a->tokens, a->q_heads);
    if ((a->q_dev && a->q_stride < (int64_t)a->q_heads * d) || (a->k_dev && (a->k_stride < (int64_t)cache->kv_heads * d || a->v_stride < (int64_t)cache->kv_heads * d)))
        return set_error(c, WF_ERR_SHAPE, "%s: a stride is shorter than a token", what);
    if (a->rot_dim < 0 || a->rot_dim > d || a->rot_dim % 8) return set_error(c, WF_ERR_SHAPE, "%s: rot_dim %d is not a multiple of 8 up to %d", what, a->rot_dim, d);
    if (a->rot_dim && (!a->rope_dev || a->rope_dev & 15 || a->rope_rows < 1 || !a->positions_dev || a->positions_dev & 3))
        return set_error(c, WF_ERR_INVALID_ARGUMENT, "%s: a rotation needs a 16-byte aligned table and positions", what);
    if ((a->gamma_q_dev | a->gamma_k_dev) & 3 || a->slots_dev & 7) return set_error(c, WF_ERR_INVALID_ARGUMENT, "%s: misaligned gamma or slots", what);
    if (a->flags & ~(WF_QK_NORM | WF_ROPE_ADJACENT)) return set_error(c, WF_ERR_INVALID_ARGUMENT, "%s: unknown flags %d", what, a->flags);
    RopeParams p{};
    p.q = reinterpret_cast<const void*>(a->q_dev), p.k = reinterpret_cast<const void*>(a->k_dev), p.v = reinterpret_cast<const void*>(a->v_dev);
    p.q_stride = a->q_stride, p.k_stride = a->k_stride, p.v_stride = a->v_stride;
    p.gamma_q = reinterpret_cast<const float*>(a->gamma_q_dev), p.gamma_k = reinterpret_cast<const float*>(a->gamma_k_dev);
    p.rope = reinterpret_cast<const float2*>(a->rope_dev);
    p.rope_rows = a->rope_rows;
    p.positions = reinterpret_cast<const int*>(a->positions_dev);
    p.slots = reinterpret_cast<const int64_t*>(a->slots_dev);
    p.q_out = reinterpret_cast<bf16*>(a->q_out_dev);
    p.cache = cache_layer(*cache, layer);
    p.tokens = a->tokens;
    p.q_heads = a->q_dev ? a->q_heads : 0;
    p.k_heads = a->k_dev ? cache->kv_heads : 0;
    p.rot = a->rot_dim, p.norm = a->flags & WF_QK_NORM, p.adjacent = (a->flags & WF_ROPE_ADJACENT) != 0;
    p.eps = a->eps;
    p.status = c->d_status;
    // 8-byte (bf16: 4-byte) loads where every head of every token allows them; head_dim is a multiple of 8
    const int64_t piece = 2 * size;
    const bool vec = ((a->q_dev | a->k_dev | a->v_dev) % piece) == 0 && (!a->q_dev || a->q_stride % 2 == 0) && (!a->k_dev || (a->k_stride % 2 == 0 && a->v_stride % 2 == 0));
    // Batches of heads of a warp: first every SM has its 64 warps (3.4 us for one token), then a warp takes up to five batches, which share the token's table row
    // and the loads of slot and position.  At 2048 tokens 24 / 32 / 48 / 64 / 96 warps an SM: 26.0 / 25.2 / 25.3 / 24.6 / 25.2 us; CTAs of 8 warps: 26.1.
    const int side = d <= 64 ? 2 : 1, per = ROPE_UNROLL * side, all = (p.q_heads + per - 1) / per + 2 * ((p.k_heads + per - 1) / per);
    p.batches = (int)std::max<int64_t>(1, std::min<int64_t>({a->tokens * all / ((int64_t)c->sm_count * ROPE_WARPS_PER_SM), all, ROPE_MOST_BATCHES}));
    p.sets = (all + p.batches - 1) / p.batches;
    const int64_t grid = (a->tokens * p.sets + ROPE_WARPS - 1) / ROPE_WARPS;
    if (grid > (1LL << 31) - 1) return set_error(c, WF_ERR_TOO_LARGE, "%s: %lld tokens of %d heads", what, (long long)a->tokens, p.q_heads + 2 * p.k_heads);
    void (*kernel)(RopeParams);
    const int whole = p.rot == 0 || p.rot == d ? d : 0;
#define WF_ROPE_DIM(X, V) (whole == 128 ? qk_norm_rope_kernel<X, V, 32, 128> : whole == 64 ? qk_norm_rope_kernel<X, V, 16, 64> : side == 2 ? qk_norm_rope_kernel<X, V, 16, 0> : qk_norm_rope_kernel<X, V, 32, 0>)
    if (size == 4) kernel = vec ? WF_ROPE_DIM(float, true) : WF_ROPE_DIM(float, false);
    else kernel = vec ? WF_ROPE_DIM(bf16, true) : WF_ROPE_DIM(bf16, false);
#undef WF_ROPE_DIM
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(ROPE_WARPS * 32);
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
