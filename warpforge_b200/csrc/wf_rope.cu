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
    float eps;
    int* status;
};

template <class X, bool VEC> __device__ __forceinline__ void load_x(const void* base, size_t i, float (&f)[4]) {
    const X* p = static_cast<const X*>(base) + i;
    if (VEC && sizeof(X) == 4) {
        const float4 v = ld_once(reinterpret_cast<const float4*>(p));
        f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
    } else if (VEC) {
        load4(reinterpret_cast<const bf16*>(p), f);
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++) f[e] = (float)p[e];
    }
}

// A group of LANES lanes has a head, four elements a lane; a warp takes HEADS heads of one token at a time, all requested before the
// first is used.  The partner of a pair (i, i + rot/2) lies rot / 8 lanes away (rot is a multiple of 8).
constexpr int ROPE_WARPS = 4, ROPE_UNROLL = 4;
template <class X, bool VEC, int LANES> __global__ void __launch_bounds__(ROPE_WARPS * 32) qk_norm_rope_kernel(const __grid_constant__ RopeParams p) {
    constexpr int SIDE = 32 / LANES, HEADS = ROPE_UNROLL * SIDE;  // heads beside one another in a warp, heads of a warp
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int lane = threadIdx.x & (LANES - 1), side = (threadIdx.x & 31) / LANES;
    const int d = p.cache.dim, i = 4 * lane, heads = p.q_heads + p.k_heads + p.v_heads, sets = (heads + HEADS - 1) / HEADS;
    const bool mine = i < d;
    const int64_t unit = (int64_t)blockIdx.x * ROPE_WARPS + (threadIdx.x >> 5);
    const int64_t t = unit / sets;
    if (t >= p.tokens) return;
    const int h0 = (int)(unit % sets) * HEADS + side;
    float x[ROPE_UNROLL][4] = {};
#pragma unroll
    for (int u = 0; u < ROPE_UNROLL; u++) {
        const int h = h0 + u * SIDE;
        if (h >= heads || !mine) continue;
        if (h < p.q_heads) load_x<X, VEC>(p.q, t * p.q_stride + (size_t)h * d + i, x[u]);
        else if (h < p.q_heads + p.k_heads) load_x<X, VEC>(p.k, t * p.k_stride + (size_t)(h - p.q_heads) * d + i, x[u]);
        else load_x<X, VEC>(p.v, t * p.v_stride + (size_t)(h - p.q_heads - p.k_heads) * d + i, x[u]);
    }
    int64_t slot = p.slots ? p.slots[t] : t;
    int64_t pos = p.rot ? p.positions[t] : 0;
    const bool bad = (p.rot && (pos < 0 || pos >= p.rope_rows)) || (p.k_heads && slot >= p.cache.pages << p.cache.page_shift);
    if (bad) {
        if ((threadIdx.x & 31) == 0) report_status(p.status, STATUS_BAD_INDEX);
        slot = -1;
        pos = 0;
    }
    float c[4] = {1.f, 1.f, 1.f, 1.f}, s[4] = {};
    const int half = p.rot / 2;
    const bool upper = !p.adjacent && i >= half;  // the second of its pairs
    if (i < p.rot) {  // rows of the table are rot * 4 bytes: 16-byte pieces
        if (p.adjacent) {
            const float4 w = *reinterpret_cast<const float4*>(p.rope + (size_t)pos * half + i / 2);
            c[0] = c[1] = w.x, s[0] = s[1] = w.y, c[2] = c[3] = w.z, s[2] = s[3] = w.w;
        } else {
            const float4* row = reinterpret_cast<const float4*>(p.rope + (size_t)pos * half + (upper ? i - half : i));
            const float4 a = row[0], b = row[1];
            c[0] = a.x, s[0] = a.y, c[1] = a.z, s[1] = a.w, c[2] = b.x, s[2] = b.y, c[3] = b.z, s[3] = b.w;
        }
    }
    float gq[4] = {1.f, 1.f, 1.f, 1.f}, gk[4] = {1.f, 1.f, 1.f, 1.f};
    if (p.norm && mine) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (p.gamma_q) gq[e] = p.gamma_q[i + e];
            if (p.gamma_k) gk[e] = p.gamma_k[i + e];
        }
    }
    const int64_t page = slot >> p.cache.page_shift;
    const int row = (int)(slot & ((1 << p.cache.page_shift) - 1));
    const int away = p.rot / 8;
#pragma unroll
    for (int u = 0; u < ROPE_UNROLL; u++) {
        const int h = h0 + u * SIDE;
        const bool is_q = h < p.q_heads, turned = h < p.q_heads + p.k_heads;  // the same for the lanes of a head, not for a warp's
        float y[4];
        float inv = 1.f;
        if (p.norm) {
            float sum = x[u][0] * x[u][0] + x[u][1] * x[u][1] + x[u][2] * x[u][2] + x[u][3] * x[u][3];
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
            if (turned) inv = rsqrtf(sum / (float)d + p.eps);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) y[e] = turned && p.norm ? x[u][e] * inv * (is_q ? gq[e] : gk[e]) : x[u][e];
        if (p.rot) {
            float other[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float far = __shfl_sync(0xFFFFFFFFu, y[e], upper ? lane - away : lane + away, LANES);
                other[e] = p.adjacent ? y[e ^ 1] : far;
            }
            if (turned && i < p.rot) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const bool second = p.adjacent ? e & 1 : upper;
                    y[e] = second ? y[e] * c[e] + other[e] * s[e] : y[e] * c[e] - other[e] * s[e];
                }
            }
        }
        if (h >= heads || !mine) continue;
        const uint2 w = bad ? make_uint2(0u, 0u) : make_uint2(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]));
        if (is_q) *reinterpret_cast<uint2*>(p.q_out + ((size_t)t * p.q_heads + h) * d + i) = w;
        else if (slot >= 0) {
            bf16* to = turned ? p.cache.keys + p.cache.at(page, h - p.q_heads, row) : p.cache.values + p.cache.at(page, h - p.q_heads - p.k_heads, row);
            *reinterpret_cast<uint2*>(to + i) = w;
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
    // 16-byte (bf16: 8-byte) loads where every head of every token allows them; head_dim is a multiple of 8
    const int64_t piece = 4 * size;
    const bool vec = ((a->q_dev | a->k_dev | a->v_dev) % piece) == 0 && (!a->q_dev || a->q_stride % 4 == 0) && (!a->k_dev || (a->k_stride % 4 == 0 && a->v_stride % 4 == 0));
    const int heads = p.q_heads + p.k_heads + p.v_heads, side = d <= 64 ? 2 : 1, sets = (heads + ROPE_UNROLL * side - 1) / (ROPE_UNROLL * side);
    const int64_t grid = (a->tokens * sets + ROPE_WARPS - 1) / ROPE_WARPS;
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
