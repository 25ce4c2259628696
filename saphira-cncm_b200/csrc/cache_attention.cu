// Attention of a row's new tokens -- one, a run, or a tree of drafted ones -- to its key/value cache
// (ncmb_cache_attention, include/ncm_b200.h), and the scratch and checks that the cache operators share.
//
// For query head h of kv head h / G and node t:  s_j = scale q.k_j over the slots j that t sees, p_j = exp(s_j - max s) /
// sum, out = sum p_j v_j; weights_j (+)= sum over the G heads and the T nodes of p_j.
#include "cache.cuh"

#include <stdarg.h>

namespace ncmb {

int cache_refuse(const char *who, const char *fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    fprintf(stderr, "[ncm_b200] %s: ", who);
    vfprintf(stderr, fmt, ap);
    fprintf(stderr, "\n");
    va_end(ap);
    return -1;
}

int cache_check(const char *who, const NcmbCache *c, CacheDev &d) {
    if (!c) return cache_refuse(who, "no cache");
    if (c->type != NCMB_F32 && c->type != NCMB_BF16) return cache_refuse(who, "cache type %d", c->type);
    if (c->rows < 0 || c->n_kv < 1 || c->capacity < 1) return cache_refuse(who, "%d rows, %d kv heads, capacity %d", c->rows, c->n_kv, c->capacity);
    if (c->rows > 65535 || c->n_kv > 65535) return cache_refuse(who, "%d rows, %d kv heads: at most 65535", c->rows, c->n_kv);
    if (c->hd < 8 || c->hd > 128 || c->hd % 8) return cache_refuse(who, "head dim %d: a multiple of 8 up to 128", c->hd);
    const int64_t es = cache_elem(c);
    if (!c->k || !c->v || (c->rows && !c->len)) return cache_refuse(who, "a null pointer in the cache");
    if (((uintptr_t)c->k | (uintptr_t)c->v) % 16 || ((uintptr_t)c->len) % 4) return cache_refuse(who, "keys and values have to be 16-byte aligned");
    if (c->row_stride < 0 || c->head_stride < 0 || c->token_stride < 0 || (c->row_stride * es) % 16 || (c->head_stride * es) % 16 || (c->token_stride * es) % 16)
        return cache_refuse(who, "strides have to be positive multiples of 16 bytes");
    if ((c->capacity > 1 && c->token_stride < c->hd) || (c->n_kv > 1 && c->head_stride < c->hd) || (c->rows > 1 && c->row_stride < c->hd))
        return cache_refuse(who, "a stride is smaller than the head dim");
    d = CacheDev{(const char *)c->k, (const char *)c->v, c->row_stride * es, c->head_stride * es, c->token_stride * es, c->rows, c->n_kv, c->hd, c->capacity, c->len};
    return 0;
}

void *cache_scratch(const char *who, size_t bytes) {
    static void *base = nullptr;
    static size_t cap = 0;
    if (bytes <= cap) return base;
    if (base) { CUDA_CHECK(cudaStreamSynchronize(stream())); CUDA_CHECK(cudaFree(base)); base = nullptr; cap = 0; }
    const size_t want = (bytes + (bytes >> 2) + ((size_t)1 << 20)) & ~(size_t)255;
    for (size_t b : {want, (bytes + 255) & ~(size_t)255}) {
        if (cudaMalloc(&base, b) == cudaSuccess) { cap = b; return base; }
        (void)cudaGetLastError();
        base = nullptr;
    }
    cache_refuse(who, "no device memory for %.1f MB of scratch", bytes / 1048576.0);
    return nullptr;
}

namespace {

struct AttnCache {
    CacheDev c;
    const char *q; char *out;
    int64_t ldq, ldo;                // bytes
    int H, G, T;
    const int *parents;
    float scale;
    float *weights;
    float *lse;                      // [rows][T][H]
};

template <class E> __device__ __forceinline__ float get(const char *p, int d) { return (float)((const E *)p)[d]; }
__device__ __forceinline__ void put(float *p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16 *p, float v) { *p = __float2bfloat16(v); }

__device__ __forceinline__ bool node_used(const int *par, int t) { return !par || (par[t] >= -1 && par[t] < t); }

// a node's ancestors and itself as bits, 32 per lane: lane w holds nodes 32 w ... 32 w + 31
__device__ __forceinline__ uint32_t node_mask(const int *par, int t, int lane) {
    uint32_t m = 0;
    for (int at = t; at >= 0 && node_used(par, at); at = par ? par[at] : at - 1)
        if ((at >> 5) == lane) m |= 1u << (at & 31);
    return m;
}

// one warp per (row, node, head), one key at a time
template <class KE, class QE>
__global__ void __launch_bounds__(128) k_cache_attention_plain(AttnCache a) {
    const int lane = threadIdx.x & 31;
    const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (w >= (int64_t)a.c.rows * a.T * a.H) return;
    const int h = (int)(w % a.H), t = (int)(w / a.H % a.T), b = (int)(w / a.H / a.T);
    const int len = cache_len(a.c, b, a.T);
    const int *par = a.parents ? a.parents + (int64_t)b * a.T : nullptr;
    QE *o = (QE *)(a.out + ((int64_t)b * a.T + t) * a.ldo) + (int64_t)h * a.c.hd;
    const bool used = node_used(par, t);
    const uint32_t mask = used ? node_mask(par, t, lane) : 0;
    const char *q = a.q + ((int64_t)b * a.T + t) * a.ldq + (int64_t)h * a.c.hd * sizeof(QE);
    const char *k = a.c.k + b * a.c.rs + (h / a.G) * a.c.hs, *v = a.c.v + b * a.c.rs + (h / a.G) * a.c.hs;
    float qr[4], acc[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < 4; i++) qr[i] = lane + 32 * i < a.c.hd ? get<QE>(q, lane + 32 * i) * a.scale : 0.f;
    for (int j = 0; used && j < len + a.T; j++) {
        if (j >= len && !((__shfl_sync(0xffffffffu, mask, (j - len) >> 5) >> ((j - len) & 31)) & 1u)) continue;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 4; i++) if (lane + 32 * i < a.c.hd) s = fmaf(qr[i], get<KE>(k + j * a.c.ts, lane + 32 * i), s);
#pragma unroll
        for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        const float n = fmaxf(m, s), al = m == -INFINITY ? 0.f : expf(m - n), p = expf(s - n);
        l = l * al + p;
        m = n;
#pragma unroll
        for (int i = 0; i < 4; i++) if (lane + 32 * i < a.c.hd) acc[i] = acc[i] * al + p * get<KE>(v + j * a.c.ts, lane + 32 * i);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) if (lane + 32 * i < a.c.hd) put(o + lane + 32 * i, l > 0.f ? acc[i] / l : 0.f);
    if (a.lse && lane == 0) a.lse[w] = l > 0.f ? m + logf(l) : INFINITY;
}

// one warp per (row, kv head, slot)
template <class KE, class QE>
__global__ void __launch_bounds__(128) k_cache_weights_plain(AttnCache a) {
    const int lane = threadIdx.x & 31, j = blockIdx.x * 4 + (threadIdx.x >> 5), kvh = blockIdx.y, b = blockIdx.z;
    const int len = cache_len(a.c, b, a.T);
    if (j >= len + a.T) return;
    const int *par = a.parents ? a.parents + (int64_t)b * a.T : nullptr;
    const char *k = a.c.k + b * a.c.rs + kvh * a.c.hs + j * a.c.ts;
    float kr[4], sum = 0.f;
#pragma unroll
    for (int i = 0; i < 4; i++) kr[i] = lane + 32 * i < a.c.hd ? get<KE>(k, lane + 32 * i) : 0.f;
    for (int t = 0; t < a.T; t++) {
        if (!node_used(par, t)) continue;
        const uint32_t mask = node_mask(par, t, lane);
        if (j >= len && !((__shfl_sync(0xffffffffu, mask, (j - len) >> 5) >> ((j - len) & 31)) & 1u)) continue;
        for (int g = 0; g < a.G; g++) {
            const char *q = a.q + ((int64_t)b * a.T + t) * a.ldq + (int64_t)(kvh * a.G + g) * a.c.hd * sizeof(QE);
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < 4; i++) if (lane + 32 * i < a.c.hd) s = fmaf(get<QE>(q, lane + 32 * i) * a.scale, kr[i], s);
#pragma unroll
            for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
            sum += expf(s - a.lse[((int64_t)b * a.T + t) * a.H + kvh * a.G + g]);
        }
    }
    float *w = a.weights + ((int64_t)b * a.c.nkv + kvh) * a.c.cap + j;
    if (lane == 0) *w = j < len ? *w + sum : sum;
}

} // namespace
} // namespace ncmb

using namespace ncmb;

extern "C" int ncmb_cache_attention(const NcmbCache *c, const void *q, int64_t ldq, void *out, int64_t ldo, int act_type, int n_head,
                                    int T, const int *parents, float scale, int max_len, float *weights) {
    const char *who = "ncmb_cache_attention";
    AttnCache a;
    if (cache_check(who, c, a.c)) return -1;
    if (act_type != NCMB_F32 && !(act_type == NCMB_BF16 && c->type == NCMB_BF16)) return cache_refuse(who, "activations of type %d with a cache of type %d", act_type, c->type);
    if (n_head < 1 || n_head % c->n_kv) return cache_refuse(who, "%d heads over %d kv heads", n_head, c->n_kv);
    if (T < 1 || T > NCMB_MAX_NODES || T > c->capacity) return cache_refuse(who, "%d new tokens: 1 to %d, and no more than the capacity", T, NCMB_MAX_NODES);
    const int64_t es = act_type == NCMB_BF16 ? 2 : 4;
    if (!q || !out || ((uintptr_t)q | (uintptr_t)out) % 16 || (ldq * es) % 16 || (ldo * es) % 16 || ldq < (int64_t)n_head * c->hd || ldo < (int64_t)n_head * c->hd)
        return cache_refuse(who, "q and out have to be 16-byte aligned, with rows of n_head * hd at multiples of 16 bytes");
    if (!(fabsf(scale) < INFINITY)) return cache_refuse(who, "scale %g", scale);
    if (c->rows == 0) return 0;
    ensure_device();
    a.q = (const char *)q; a.out = (char *)out; a.ldq = ldq * es; a.ldo = ldo * es;
    a.H = n_head; a.G = n_head / c->n_kv; a.T = T; a.parents = parents; a.weights = weights;
    a.scale = scale == 0.f ? 1.0f / sqrtf((float)c->hd) : scale;
    if (max_len <= 0 || max_len > c->capacity - T) max_len = c->capacity - T;
    a.lse = nullptr;
    const int64_t warps = (int64_t)c->rows * T * n_head;
    if (weights && !(a.lse = (float *)cache_scratch(who, warps * 4))) return -1;
    const unsigned grid = grid1d(warps, 4);
    const dim3 gw((unsigned)cdiv(c->capacity, 4), c->n_kv, c->rows);
    if (c->type == NCMB_F32) {
        LAUNCH((k_cache_attention_plain<float, float>), grid, 128, 0, a);
        if (weights) LAUNCH((k_cache_weights_plain<float, float>), gw, 128, 0, a);
    } else if (act_type == NCMB_F32) {
        LAUNCH((k_cache_attention_plain<__nv_bfloat16, float>), grid, 128, 0, a);
        if (weights) LAUNCH((k_cache_weights_plain<__nv_bfloat16, float>), gw, 128, 0, a);
    } else {
        LAUNCH((k_cache_attention_plain<__nv_bfloat16, __nv_bfloat16>), grid, 128, 0, a);
        if (weights) LAUNCH((k_cache_weights_plain<__nv_bfloat16, __nv_bfloat16>), gw, 128, 0, a);
    }
    return 0;
}
