// Attention of a row's new tokens -- one, a run, or a tree of drafted ones -- to its key/value cache
// (ncmb_cache_attention, include/ncm_b200.h), and the scratch and checks that the cache operators share.
//
// For query head h of kv head h / G and node t:  s_j = scale q.k_j over the slots j that t sees, p_j = exp(s_j - max s) /
// sum, out = sum p_j v_j; weights_j (+)= sum over the G heads and the T nodes of p_j.
#include "cache_tc.cuh"

#include <new>
#include <unordered_map>

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

int cache_device(const char *who) {
    ensure_device();
    int dev = -1;
    if (cudaGetDevice(&dev) != cudaSuccess) (void)cudaGetLastError();
    return dev == ctx().device ? 0 : cache_refuse(who, "device %d is current, the library runs on %d", dev, ctx().device);
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

// Areas of each stream: calls on one stream are ordered, calls on two are not. A captured call's area is in the graph for good: it is
// replaced when a call needs more, but not freed.
void *cache_scratch(const char *who, size_t bytes, int area) {
    struct Area { void *base = nullptr; size_t cap = 0; bool in_graph = false; };
    struct Areas { Area of[SCRATCH_AREAS]; };
    static std::unordered_map<cudaStream_t, Areas> streams;
    static cudaStream_t last = nullptr;
    static Areas *mine = nullptr;                    // of `last`
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    cudaError_t e = cudaStreamIsCapturing(stream(), &capture);
    const bool captured = capture != cudaStreamCaptureStatusNone;
    if (e != cudaSuccess) { (void)cudaGetLastError(); cache_refuse(who, "the stream: %s", cudaGetErrorString(e)); return nullptr; }
    if (!mine || last != stream()) {
        try { mine = &streams[stream()]; } catch (const std::bad_alloc &) { cache_refuse(who, "no memory"); return nullptr; }
        last = stream();
    }
    Area *a = &mine->of[area];
    if (bytes <= a->cap) {
        a->in_graph |= captured;
        return a->base;
    }
    if (captured) { cache_refuse(who, "%.1f MB of scratch while the stream is captured: make the same call on it before", bytes / 1048576.0); return nullptr; }
    if (a->base && !a->in_graph) {
        e = cudaStreamSynchronize(stream());         // refused where another thread's capture forbids it
        if (e != cudaSuccess) { (void)cudaGetLastError(); cache_refuse(who, "scratch has to grow: %s", cudaGetErrorString(e)); return nullptr; }
        CUDA_CHECK(cudaFree(a->base));
    }
    *a = Area();
    const size_t want = (bytes + (bytes >> 2) + ((size_t)1 << 20)) & ~(size_t)255;
    for (size_t b : {want, (bytes + 255) & ~(size_t)255}) {
        if (cudaMalloc(&a->base, b) == cudaSuccess) {
            if (area == SCRATCH_DONE) CUDA_CHECK(cudaMemsetAsync(a->base, 0, b, stream()));
            a->cap = b;
            // what the wide tiles report into is made here too, not by a captured call, and is zero for every stream
            (void)tc_err_flag();
            CUDA_CHECK(cudaStreamSynchronize(stream()));
            return a->base;
        }
        (void)cudaGetLastError();
        a->base = nullptr;
    }
    cache_refuse(who, "no device memory for %.1f MB of scratch", bytes / 1048576.0);
    return nullptr;
}

int ct_map(const char *who, const CacheDev &c, const char *p, int kt, CUtensorMap &m) {
    using Encode = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static Encode encode = nullptr;
    if (!encode) {
        cudaDriverEntryPointQueryResult found;
        void *f = nullptr;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found) != cudaSuccess || !f) return cache_refuse(who, "the driver has no tensor maps");
        encode = (Encode)f;
    }
    // a dim of one element has a stride that is not used: any valid one
    const cuuint64_t dims[4] = {(cuuint64_t)c.hd, (cuuint64_t)c.cap, (cuuint64_t)c.nkv, (cuuint64_t)c.rows};
    const cuuint64_t strides[3] = {(cuuint64_t)(c.cap > 1 ? c.ts : 256), (cuuint64_t)(c.nkv > 1 ? c.hs : 256), (cuuint64_t)(c.rows > 1 ? c.rs : 256)};
    const cuuint32_t box[4] = {64, (cuuint32_t)kt, 1, 1}, one[4] = {1, 1, 1, 1};
    const CUresult r = encode(&m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<char *>(p), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : cache_refuse(who, "tensor map: %d (strides of 2^40 bytes or more?)", (int)r);
}

int cache_variant = 0;

namespace {

template <class KE, class QE, int HDP>
int run_attention_hd(const char *who, const CmArgs &a, int max_keys) {
    // (the terms of an fp32 cache's keys of more than 64 dims do not fit shared memory beside the queries')
    if constexpr (sizeof(KE) == 2 || HDP == 64) { if (takes_wide<KE, QE, HDP>(a, max_keys)) return ct_run_as<KE, QE, HDP>(who, a, max_keys); }
    auto none = [] {};
    return a.M <= 8 ? cm_run_as<KE, QE, HDP, 8, false>(who, a, max_keys, none) : cm_run_as<KE, QE, HDP, 16, false>(who, a, max_keys, none);
}
template <class KE, class QE>
int run_attention(const char *who, const CmArgs &a, int max_keys) {
    return a.c.hd <= 64 ? run_attention_hd<KE, QE, 64>(who, a, max_keys) : run_attention_hd<KE, QE, 128>(who, a, max_keys);
}

} // namespace
} // namespace ncmb

using namespace ncmb;

extern "C" void ncmb_set_cache_variant(int variant) { ncmb::cache_variant = variant; }

extern "C" int ncmb_cache_attention(const NcmbCache *c, const void *q, int64_t ldq, void *out, int64_t ldo, int act_type, int n_head,
                                    int T, const int *parents, float scale, int max_len, float *weights) {
    const char *who = "ncmb_cache_attention";
    CmArgs a = {};
    if (cache_check(who, c, a.c)) return -1;
    if (act_type != NCMB_F32 && !(act_type == NCMB_BF16 && c->type == NCMB_BF16)) return cache_refuse(who, "activations of type %d with a cache of type %d", act_type, c->type);
    if (n_head < 1 || n_head % c->n_kv) return cache_refuse(who, "%d heads over %d kv heads", n_head, c->n_kv);
    if (T < 1 || T > NCMB_MAX_NODES || T > c->capacity) return cache_refuse(who, "%d new tokens: 1 to %d, and no more than the capacity", T, NCMB_MAX_NODES);
    if ((int64_t)T * (n_head / c->n_kv) > 1 << 30) return cache_refuse(who, "%d new tokens of %d heads a kv head", T, n_head / c->n_kv);
    const int64_t es = act_type == NCMB_BF16 ? 2 : 4;
    if (!q || !out || ((uintptr_t)q | (uintptr_t)out) % 16 || (ldq * es) % 16 || (ldo * es) % 16 || ldq < (int64_t)n_head * c->hd || ldo < (int64_t)n_head * c->hd)
        return cache_refuse(who, "q and out have to be 16-byte aligned, with rows of n_head * hd at multiples of 16 bytes");
    if (!(fabsf(scale) < INFINITY)) return cache_refuse(who, "scale %g", scale);
    if (c->rows == 0) return 0;
    ensure_device();
    a.q = (const char *)q; a.out = (char *)out; a.ldq = ldq * es; a.ldo = ldo * es;
    a.H = n_head; a.G = n_head / c->n_kv; a.T = T; a.M = T * a.G; a.parents = parents; a.weights = weights;
    a.c2 = (scale == 0.f ? 1.0f / sqrtf((float)c->hd) : scale) * 1.44269504f;
    if (max_len <= 0 || max_len > c->capacity - T) max_len = c->capacity - T;
    const double keys = (double)c->rows * c->n_kv * (max_len + T);      // by the bound: lengths are on the device
    ProfScope prof(NCMB_K_ATTN, 4.0 * keys * a.M * c->hd, 2.0 * keys * c->hd * cache_elem(c));
    if (c->type == NCMB_F32) return run_attention<float, float>(who, a, max_len + T);
    if (act_type == NCMB_F32) return run_attention<__nv_bfloat16, float>(who, a, max_len + T);
    return run_attention<__nv_bfloat16, __nv_bfloat16>(who, a, max_len + T);
}
