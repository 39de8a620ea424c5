// wf_qk_norm_rope: what happens to q, k and v between their projections and the attention, in one pass.  Per token and head of q and k
//   x' = x / sqrt(mean(x^2) + eps) * gamma,   (a, b) -> (a c - b s, b c + a s) for the pairs of the first rot elements
// in fp32, rounded once to bf16; v is rounded only; k and v go to their slots in the cache.
// Bound by HBM: one read of the projections' rows, one write of half their size.
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
    int q_heads, k_heads, v_heads;  // 0: that part is not wanted
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

// A group of LANES lanes has a head, four elements a lane: two pairs that are rotated, (i, i + rot/2) and (i + 1, i + 1 + rot/2) or two adjacent ones, so
// that no lane needs another's, or four that are not. A warp takes HEADS heads of one token at a time.
constexpr int ROPE_WARPS = 4, ROPE_UNROLL = 4, ROPE_WARPS_PER_SM = 48, ROPE_MOST_BATCHES = 5;
template <class X, bool VEC, int LANES> __global__ void __launch_bounds__(ROPE_WARPS * 32) qk_norm_rope_kernel(const __grid_constant__ RopeParams p) {
    constexpr int SIDE = 32 / LANES, HEADS = ROPE_UNROLL * SIDE;  // heads beside one another in a warp, heads of a batch
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int lane = threadIdx.x & (LANES - 1), side = (threadIdx.x & 31) / LANES;
    const int d = p.cache.dim, heads = p.q_heads + p.k_heads + p.v_heads, rotated = p.q_heads + p.k_heads;
    const bool mine = 4 * lane < d;
    const int64_t unit = (int64_t)blockIdx.x * ROPE_WARPS + (threadIdx.x >> 5);
    const int64_t t = unit / p.sets;
    if (t >= p.tokens) return;
    const int set = (int)(unit - t * p.sets), h_first = set * p.batches * HEADS + side;
    const int h_end = min(heads, (set + 1) * p.batches * HEADS);
    // the elements: a0, a0 + 1 and b0, b0 + 1
    const bool turns = 4 * lane < p.rot, apart = turns && !p.adjacent;
    const int a0 = apart ? 2 * lane : 4 * lane, b0 = apart ? p.rot / 2 + 2 * lane : 4 * lane + 2;
    // where the token's heads lie, as if all were heads of one tensor: head h is h * d elements on
    const X* const in_q = static_cast<const X*>(p.q) + t * p.q_stride;
    const X* const in_k = static_cast<const X*>(p.k) + t * p.k_stride - (int64_t)p.q_heads * d;
    const X* const in_v = static_cast<const X*>(p.v) + t * p.v_stride - (int64_t)rotated * d;
    auto ask = [&](int h0, float2 (&x)[ROPE_UNROLL][2]) {
#pragma unroll
        for (int u = 0; u < ROPE_UNROLL; u++) {
            const int h = h0 + u * SIDE;
            x[u][0] = x[u][1] = make_float2(0.f, 0.f);
            if (h >= h_end || !mine) continue;
            const X* const from = (h < p.q_heads ? in_q : h < rotated ? in_k : in_v) + h * d;
            x[u][0] = load_pair<X, VEC>(from + a0);
            x[u][1] = load_pair<X, VEC>(from + b0);
        }
    };
    float2 x[ROPE_UNROLL][2];
    ask(h_first, x);
    int64_t slot = p.slots ? p.slots[t] : t;
    int64_t pos = p.rot ? p.positions[t] : 0;
    float2 gq[2] = {make_float2(1.f, 1.f), make_float2(1.f, 1.f)}, gk[2] = {make_float2(1.f, 1.f), make_float2(1.f, 1.f)};
    if (p.norm && mine) {
        if (p.gamma_q) gq[0] = make_float2(p.gamma_q[a0], p.gamma_q[a0 + 1]), gq[1] = make_float2(p.gamma_q[b0], p.gamma_q[b0 + 1]);
        if (p.gamma_k) gk[0] = make_float2(p.gamma_k[a0], p.gamma_k[a0 + 1]), gk[1] = make_float2(p.gamma_k[b0], p.gamma_k[b0 + 1]);
    }
    const bool bad = (p.rot && (pos < 0 || pos >= p.rope_rows)) || (p.k_heads && slot >= p.cache.pages << p.cache.page_shift);
    if (bad) {
        if ((threadIdx.x & 31) == 0) report_status(p.status, STATUS_BAD_INDEX);
        slot = -1;
        pos = 0;
    }
    float4 cs = make_float4(1.f, 0.f, 1.f, 0.f);  // cosine and sine of the lane's two pairs: 16 bytes of the row either way
    if (turns) cs = *reinterpret_cast<const float4*>(p.rope + (size_t)pos * (p.rot / 2) + 2 * lane);
    bf16* const out_q = p.q_out + t * p.q_heads * d;
    const int64_t place = slot < 0 ? 0 : (int64_t)p.cache.at(slot >> p.cache.page_shift, 0, (int)(slot & ((1 << p.cache.page_shift) - 1)));
    const int apart_heads = d << p.cache.page_shift;  // elements between heads of the cache
    for (int h0 = h_first; h0 - side < h_end; h0 += HEADS) {
        if (h0 > h_first) ask(h0, x);
        float inv[ROPE_UNROLL];
        if (p.norm) {
            // The sums of squares of four heads in ten exchanges instead of twenty: with every exchange at a distance a lane passes on half of the sums that it has and adds
            // to the others, until it has one; that one is then brought to all lanes of the head.
            float s[ROPE_UNROLL];
#pragma unroll
            for (int u = 0; u < ROPE_UNROLL; u++) s[u] = x[u][0].x * x[u][0].x + x[u][0].y * x[u][0].y + x[u][1].x * x[u][1].x + x[u][1].y * x[u][1].y;
            const bool hi = lane & (LANES / 2), hi2 = lane & (LANES / 4);
            float t0 = hi ? s[2] : s[0], t1 = hi ? s[3] : s[1];
            t0 += __shfl_xor_sync(0xFFFFFFFFu, hi ? s[0] : s[2], LANES / 2);
            t1 += __shfl_xor_sync(0xFFFFFFFFu, hi ? s[1] : s[3], LANES / 2);
            float r = hi2 ? t1 : t0;
            r += __shfl_xor_sync(0xFFFFFFFFu, hi2 ? t0 : t1, LANES / 4);
#pragma unroll
            for (int o = LANES / 8; o > 0; o >>= 1) r += __shfl_xor_sync(0xFFFFFFFFu, r, o);
            r = rsqrtf(r / (float)d + p.eps);
#pragma unroll
            for (int u = 0; u < ROPE_UNROLL; u++) inv[u] = __shfl_sync(0xFFFFFFFFu, r, (u >> 1) * (LANES / 2) + (u & 1) * (LANES / 4), LANES);
        }
#pragma unroll
        for (int u = 0; u < ROPE_UNROLL; u++) {
            const int h = h0 + u * SIDE;
            if (h >= h_end || !mine) continue;
            float2 a = x[u][0], b = x[u][1];
            if (h < rotated) {
                if (p.norm) {
                    const bool is_q = h < p.q_heads;
                    const float2 ga = is_q ? gq[0] : gk[0], gb = is_q ? gq[1] : gk[1];
                    a = make_float2(a.x * inv[u] * ga.x, a.y * inv[u] * ga.y);
                    b = make_float2(b.x * inv[u] * gb.x, b.y * inv[u] * gb.y);
                }
                if (apart) {
                    const float2 a1 = make_float2(a.x * cs.x - b.x * cs.y, a.y * cs.z - b.y * cs.w);
                    b = make_float2(b.x * cs.x + a.x * cs.y, b.y * cs.z + a.y * cs.w);
                    a = a1;
                } else if (turns) {
                    a = make_float2(a.x * cs.x - a.y * cs.y, a.y * cs.x + a.x * cs.y);
                    b = make_float2(b.x * cs.z - b.y * cs.w, b.y * cs.z + b.x * cs.w);
                }
            }
            const uint32_t wa = bad ? 0u : pack_bf16(a.x, a.y), wb = bad ? 0u : pack_bf16(b.x, b.y);
            bf16* to = out_q + h * d;
            if (h >= p.q_heads) to = (h < rotated ? p.cache.keys + (int64_t)(h - p.q_heads) * apart_heads : p.cache.values + (int64_t)(h - rotated) * apart_heads) + place;
            if (h < p.q_heads || slot >= 0) {
                *reinterpret_cast<uint32_t*>(to + a0) = wa;
                *reinterpret_cast<uint32_t*>(to + b0) = wb;
            }
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
    p.k_heads = p.v_heads = a->k_dev ? cache->kv_heads : 0;
    p.rot = a->rot_dim, p.norm = a->flags & WF_QK_NORM, p.adjacent = (a->flags & WF_ROPE_ADJACENT) != 0;
    p.eps = a->eps;
    p.status = c->d_status;
    // 8-byte (bf16: 4-byte) loads where every head of every token allows them; head_dim is a multiple of 8
    const int64_t piece = 2 * size;
    const bool vec = ((a->q_dev | a->k_dev | a->v_dev) % piece) == 0 && (!a->q_dev || a->q_stride % 2 == 0) && (!a->k_dev || (a->k_stride % 2 == 0 && a->v_stride % 2 == 0));
    // Batches of heads of a warp: as many warps as the device holds come first, then fewer that share a token's table row and scales.
    const int heads = p.q_heads + p.k_heads + p.v_heads, side = d <= 64 ? 2 : 1, all = (heads + ROPE_UNROLL * side - 1) / (ROPE_UNROLL * side);
    p.batches = (int)std::max<int64_t>(1, std::min<int64_t>({a->tokens * all / ((int64_t)c->sm_count * ROPE_WARPS_PER_SM), all, ROPE_MOST_BATCHES}));
    p.sets = (all + p.batches - 1) / p.batches;
    const int64_t grid = (a->tokens * p.sets + ROPE_WARPS - 1) / ROPE_WARPS;
    if (grid > (1LL << 31) - 1) return set_error(c, WF_ERR_TOO_LARGE, "%s: %lld tokens of %d heads", what, (long long)a->tokens, heads);
    void (*kernel)(RopeParams);
#define WF_ROPE_PICK(X, V) (side == 2 ? qk_norm_rope_kernel<X, V, 16> : qk_norm_rope_kernel<X, V, 32>)
    if (size == 4) kernel = vec ? WF_ROPE_PICK(float, true) : WF_ROPE_PICK(float, false);
    else kernel = vec ? WF_ROPE_PICK(bf16, true) : WF_ROPE_PICK(bf16, false);
#undef WF_ROPE_PICK
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
