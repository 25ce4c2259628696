// Attention over blocks of the cache that a cheap score picks for each query (ncmb_block_summaries and
// ncmb_block_attention, include/ncm_b200.h).
#include "cache_mma.cuh"

namespace ncmb {
namespace {

template <class E> __device__ __forceinline__ float get(const char *p, int d) { return (float)((const E *)p)[d]; }

// one warp per (row, kv head, block); a lane has the dims lane, lane + 32, ...
template <class KE>
__global__ void __launch_bounds__(128) k_block_summaries(CacheDev c, int n_new, const int *first, int block, int nb, signed char *codes, float *scales) {
    const int lane = threadIdx.x & 31, i = blockIdx.x * 4 + (threadIdx.x >> 5), kvh = blockIdx.y, b = blockIdx.z;
    const int n = cache_len(c, b, n_new) + n_new, f = first ? first[b] : 0;
    if (i >= nb || i * (int64_t)block >= n || (i + 1) * (int64_t)block <= f) return;
    const int s0 = i * block, cnt = min(block, n - s0);
    const char *k = c.k + b * c.rs + kvh * c.hs + s0 * c.ts;
    float mean[4], top = 0.f;
#pragma unroll
    for (int x = 0; x < 4; x++) {
        const int d = lane + 32 * x;
        mean[x] = 0.f;
        if (d >= c.hd) continue;
        // by halves: slot j of what is left plus slot j + half. In the order of a binary counter over bit-reversed slots, so
        // that one partial sum a level is enough.
        float part[8];
        const int bits = 31 - __clz(block);
        for (int j = 0; j < block; j++) {
            const int s = (int)(__brev((unsigned)j) >> (32 - bits));
            float v = s < cnt ? get<KE>(k + s * c.ts, d) : 0.f;
            int lev = 0;
            for (int jj = j; jj & 1; jj >>= 1, lev++) v = __fadd_rn(part[lev], v);
            part[lev] = v;
        }
        mean[x] = __fdiv_rn(part[bits], (float)cnt);
        top = fmaxf(top, fabsf(mean[x]));
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float sc = __fdiv_rn(top, 127.f);
    const int64_t at = ((int64_t)b * c.nkv + kvh) * nb + i;
#pragma unroll
    for (int x = 0; x < 4; x++) {
        const int d = lane + 32 * x;
        if (d < c.hd) codes[at * c.hd + d] = sc > 0.f ? (signed char)(int)rintf(__fdiv_rn(mean[x], sc)) : 0;
    }
    if (lane == 0) scales[at] = sc;
}

struct BlockArgs {
    CacheDev c;
    const char *q; char *out;
    int64_t ldq, ldo;
    int H, G, T, block, nb, n_sel, n_first, n_last;
    float scale;
    const signed char *codes; const float *scales;
    int *picks;                      // [rows][T][nkv][n_sel]
    uint32_t *keys;                  // scratch [rows][T][nkv][nb] when they do not fit shared memory, else null
};

constexpr int BP_THREADS = 256;
constexpr int BP_KEYS = 16384;       // keys a CTA holds in shared memory

// picks of one (row, token, kv head)
template <class QE>
__global__ void __launch_bounds__(BP_THREADS) k_block_pick(BlockArgs a) {
    extern __shared__ __align__(16) char dyn[];
    __shared__ SelShared sel;
    __shared__ int wtie[BP_THREADS / 32], wkeep[BP_THREADS / 32];
    const int t = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, hd = a.c.hd;
    const int cur = (cache_len(a.c, b, a.T) + t) / a.block, n = cur + 1, k = min(n, a.n_sel);
    const int64_t u = ((int64_t)b * a.T + t) * a.c.nkv + kvh;
    int *picks = a.picks + u * a.n_sel;
    for (int i = k + tid; i < a.n_sel; i += BP_THREADS) picks[i] = -1;
    if (n <= a.n_sel) {
        for (int i = tid; i < n; i += BP_THREADS) picks[i] = i;
        return;
    }
    float *qs = (float *)dyn;                                                // [G]
    signed char *q8 = (signed char *)(qs + ((a.G + 3) & ~3));                // [G][hd]
    uint32_t *keys = a.keys ? a.keys + u * a.nb : (uint32_t *)(q8 + ((a.G * hd + 15) & ~15));
    for (int g = warp; g < a.G; g += BP_THREADS / 32) {
        const char *q = a.q + ((int64_t)b * a.T + t) * a.ldq + (int64_t)(kvh * a.G + g) * hd * sizeof(QE);
        float v[4], top = 0.f;
#pragma unroll
        for (int x = 0; x < 4; x++) { v[x] = lane + 32 * x < hd ? get<QE>(q, lane + 32 * x) : 0.f; top = fmaxf(top, fabsf(v[x])); }
#pragma unroll
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float sc = __fdiv_rn(top, 127.f);
        if (lane == 0) qs[g] = sc;
#pragma unroll
        for (int x = 0; x < 4; x++)
            if (lane + 32 * x < hd) q8[g * hd + lane + 32 * x] = sc > 0.f ? (signed char)(int)rintf(__fdiv_rn(v[x], sc)) : 0;
    }
    __syncthreads();
    const signed char *codes = a.codes + ((int64_t)b * a.c.nkv + kvh) * a.nb * hd;
    const float *scales = a.scales + ((int64_t)b * a.c.nkv + kvh) * a.nb;
    for (int i = tid; i < n; i += BP_THREADS) {
        uint32_t key = 0xffffffffu;
        if (i >= a.n_first && i <= cur - a.n_last) {
            int2 c[16];                                                      // up to 128 codes
#pragma unroll
            for (int x = 0; x < 16; x++) if (x * 8 < hd) c[x] = *(const int2 *)(codes + (int64_t)i * hd + x * 8);
            float best = -INFINITY;
            for (int g = 0; g < a.G; g++) {
                int dot = 0;
#pragma unroll
                for (int x = 0; x < 16; x++)
                    if (x * 8 < hd) {
                        const int2 q = *(const int2 *)(q8 + g * hd + x * 8);
                        dot = __dp4a(c[x].x, q.x, dot);
                        dot = __dp4a(c[x].y, q.y, dot);
                    }
                const float s = __fmul_rn((float)dot, qs[g]);
                best = s > best || !(s == s) ? s : best;
            }
            key = float_key(__fmul_rn(best, scales[i]));
        }
        keys[i] = key;
    }
    __syncthreads();
    uint32_t ties;
    const uint32_t bound = select_kth<BP_THREADS>(sel, n, (uint32_t)k, ties, [&](int i) { return keys[i]; });
    const int per = ((n + BP_THREADS - 1) / BP_THREADS) * 32, w0 = min(n, warp * per), w1 = min(n, w0 + per);
    int nt = 0, above = 0;
    for (int s = w0; s < w1; s += 32) {
        const uint32_t x = s + lane < w1 ? keys[s + lane] : 0;
        nt += __popc(__ballot_sync(0xffffffffu, s + lane < w1 && x == bound));
        above += __popc(__ballot_sync(0xffffffffu, s + lane < w1 && x > bound));
    }
    if (lane == 0) { wtie[warp] = nt; wkeep[warp] = above; }
    __syncthreads();
    int tb = 0, at = 0;                          // ties before this warp; picks before it
    for (int i = 0; i < warp; i++) { at += wkeep[i]; tb += wtie[i]; }
    at += min(tb, (int)ties);
    for (int s = w0; s < w1; s += 32) {
        const bool in = s + lane < w1;
        const uint32_t x = in ? keys[s + lane] : 0, lt = (1u << lane) - 1;
        const uint32_t tm = __ballot_sync(0xffffffffu, in && x == bound);
        const bool keep = in && (x > bound || (x == bound && tb + __popc(tm & lt) < (int)ties));
        const uint32_t km = __ballot_sync(0xffffffffu, keep);
        if (keep) picks[at + __popc(km & lt)] = s + lane;
        at += __popc(km);
        tb += __popc(tm);
    }
}

} // namespace
} // namespace ncmb

using namespace ncmb;

extern "C" int ncmb_block_summaries(const NcmbCache *c, int n_new, const int *first, int block, int max_len, signed char *codes, float *scales) {
    const char *who = "ncmb_block_summaries";
    CacheDev d;
    if (cache_check(who, c, d)) return -1;
    if (block != 16 && block != 32 && block != 64 && block != 128) return cache_refuse(who, "blocks of %d: 16, 32, 64 or 128", block);
    if (n_new < 0 || n_new > c->capacity) return cache_refuse(who, "%d new tokens in a cache of %d", n_new, c->capacity);
    if (!codes || !scales || (uintptr_t)codes % 16) return cache_refuse(who, "codes and scales: not null, codes 16-byte aligned");
    if (c->rows == 0) return 0;
    ensure_device();
    const int nb = (int)cdiv(c->capacity, block);
    const dim3 grid((unsigned)cdiv(nb, 4), c->n_kv, c->rows);
    if (c->type == NCMB_F32) LAUNCH(k_block_summaries<float>, grid, 128, 0, d, n_new, first, block, nb, codes, scales);
    else LAUNCH(k_block_summaries<__nv_bfloat16>, grid, 128, 0, d, n_new, first, block, nb, codes, scales);
    (void)max_len;
    return 0;
}

extern "C" int ncmb_block_attention(const NcmbCache *c, const void *q, int64_t ldq, void *out, int64_t ldo, int act_type, int n_head, int T,
                                    int block, const signed char *codes, const float *scales, int n_sel, int n_first, int n_last,
                                    float scale, int max_len, int *picks) {
    const char *who = "ncmb_block_attention";
    BlockArgs a;
    if (cache_check(who, c, a.c)) return -1;
    if (act_type != NCMB_F32 && !(act_type == NCMB_BF16 && c->type == NCMB_BF16)) return cache_refuse(who, "activations of type %d with a cache of type %d", act_type, c->type);
    if (n_head < 1 || n_head % c->n_kv) return cache_refuse(who, "%d heads over %d kv heads", n_head, c->n_kv);
    if (T < 1 || T > NCMB_MAX_NODES || T > c->capacity) return cache_refuse(who, "%d new tokens: 1 to %d, and no more than the capacity", T, NCMB_MAX_NODES);
    if (block != 16 && block != 32 && block != 64 && block != 128) return cache_refuse(who, "blocks of %d: 16, 32, 64 or 128", block);
    if (n_first < 0 || n_last < 1 || n_sel > 1024 || (int64_t)n_first + n_last > n_sel) return cache_refuse(who, "%d blocks, the first %d and the last %d among them", n_sel, n_first, n_last);
    const int64_t es = act_type == NCMB_BF16 ? 2 : 4;
    if (!q || !out || ((uintptr_t)q | (uintptr_t)out) % 16 || (ldq * es) % 16 || (ldo * es) % 16 || ldq < (int64_t)n_head * c->hd || ldo < (int64_t)n_head * c->hd)
        return cache_refuse(who, "q and out have to be 16-byte aligned, with rows of n_head * hd at multiples of 16 bytes");
    if (!codes || !scales || (uintptr_t)codes % 16) return cache_refuse(who, "codes and scales: not null, codes 16-byte aligned");
    if (!(fabsf(scale) < INFINITY)) return cache_refuse(who, "scale %g", scale);
    if (c->rows == 0) return 0;
    ensure_device();
    a.q = (const char *)q; a.out = (char *)out; a.ldq = ldq * es; a.ldo = ldo * es;
    a.H = n_head; a.G = n_head / c->n_kv; a.T = T; a.block = block; a.nb = (int)cdiv(c->capacity, block);
    a.n_sel = n_sel; a.n_first = n_first; a.n_last = n_last; a.codes = codes; a.scales = scales;
    a.scale = scale == 0.f ? 1.0f / sqrtf((float)c->hd) : scale;
    const int64_t units = (int64_t)c->rows * T * c->n_kv;
    const size_t need_picks = picks ? 0 : (size_t)units * n_sel * 4, need_keys = a.nb > BP_KEYS ? (size_t)units * a.nb * 4 : 0;
    char *scratch = need_picks + need_keys ? (char *)cache_scratch(who, need_picks + need_keys, SCRATCH_PICKS) : nullptr;
    if (need_picks + need_keys && !scratch) return -1;
    a.picks = picks ? picks : (int *)(scratch + need_keys);
    a.keys = need_keys ? (uint32_t *)scratch : nullptr;
    const size_t smem = (size_t)((a.G + 3) & ~3) * 4 + (((size_t)a.G * c->hd + 15) & ~(size_t)15) + (need_keys ? 0 : (size_t)a.nb * 4);
    if (smem > 150000) return cache_refuse(who, "%d query heads a kv head", a.G);
    const dim3 gp(T, c->n_kv, c->rows);
    if (act_type == NCMB_F32) {
        CUDA_CHECK(cudaFuncSetAttribute(k_block_pick<float>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        LAUNCH(k_block_pick<float>, gp, BP_THREADS, smem, a);
    } else {
        CUDA_CHECK(cudaFuncSetAttribute(k_block_pick<__nv_bfloat16>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        LAUNCH(k_block_pick<__nv_bfloat16>, gp, BP_THREADS, smem, a);
    }
    CmArgs m = {};
    m.c = a.c; m.q = a.q; m.out = a.out; m.ldq = a.ldq; m.ldo = a.ldo; m.H = a.H; m.G = a.G; m.T = T; m.M = a.G;
    m.c2 = a.scale * 1.44269504f; m.block_log = block == 16 ? 4 : block == 32 ? 5 : block == 64 ? 6 : 7; m.n_sel = n_sel; m.picks = a.picks;
    if (max_len <= 0 || max_len > c->capacity - T) max_len = c->capacity - T;
    const int keys = (int)std::min<int64_t>(max_len + T, (int64_t)n_sel * block);
    if (c->type == NCMB_F32) return cm_run<float, float, true>(who, m, keys);
    if (act_type == NCMB_F32) return cm_run<__nv_bfloat16, float, true>(who, m, keys);
    return cm_run<__nv_bfloat16, __nv_bfloat16, true>(who, m, keys);
}
