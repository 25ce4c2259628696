// Shared by the operators on long key/value caches (cache_attention.cu, cache_evict.cu, cache_blocks.cu): the cache as
// kernels see it, argument checks, and the scratch memory of a call.
#pragma once
#include "common.cuh"

#include <cooperative_groups.h>
#include <cuda_bf16.h>

namespace ncmb {

struct CacheDev {
    const char *k, *v;               // bytes
    int64_t rs, hs, ts;              // strides in bytes
    int rows, nkv, hd, cap;
    const int *len;
};

// One line to stderr and -1: what an entry point returns for arguments it refuses.
int cache_refuse(const char *who, const char *fmt, ...);
// 0 when the cache's description is one the kernels take (see ncm_b200.h), else -1 with a message
int cache_check(const char *who, const NcmbCache *c, CacheDev &d);
inline int cache_elem(const NcmbCache *c) { return c->type == NCMB_BF16 ? 2 : 4; }
// Scratch of at least `bytes` of the library's stream, kept and grown; null with a message when the device has no room for it, or when it
// would have to grow while the stream is captured. Calls on a stream are ordered, so all of them share it; within a call, what one kernel
// leaves for another that has scratch of its own stands in another area.
// SCRATCH_DONE holds zeros when it is given out, and whoever uses it leaves zeros.
enum { SCRATCH_MAIN = 0, SCRATCH_PICKS = 1, SCRATCH_DONE = 2, SCRATCH_AREAS = 3 };
void *cache_scratch(const char *who, size_t bytes, int area = SCRATCH_MAIN);

// order of floats as unsigned: larger is larger, -0 is 0, a NaN below everything
__host__ __device__ __forceinline__ uint32_t float_key(float x) {
    if (!(x == x)) return 0u;
    if (x == 0.f) return 0x80000000u;
    uint32_t u;
#ifdef __CUDA_ARCH__
    u = __float_as_uint(x);
#else
    memcpy(&u, &x, 4);
#endif
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

#ifdef __CUDACC__
__device__ __forceinline__ int cache_len(const CacheDev &c, int row, int n_new) {   // cached tokens, made to fit
    return max(0, min(c.len[row], c.cap - n_new));
}

// a launch in clusters of nc CTAs along x, started under its predecessor
template <typename... KArgs, typename... Args>
void cache_launch(void (*kernel)(KArgs...), dim3 grid, int threads, size_t smem, int nc, Args... args) {
    static const bool off = getenv("NCM_B200_NO_PDL") != nullptr;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid; cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = smem; cfg.stream = stream();
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = off ? 0 : 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = nc; at[1].val.clusterDim.y = 1; at[1].val.clusterDim.z = 1;
    cfg.attrs = at; cfg.numAttrs = nc > 1 ? 2 : 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, KArgs(args)...);
    if (e != cudaSuccess) fatal("cache operators: launch failed: %s", cudaGetErrorString(e));
    ctx().launches++;
}

// ---- the k-th largest of many 32-bit keys, by a cluster of CTAs that each hold a part of them ----
constexpr int SEL_BINS = 2048;
struct SelShared {
    alignas(16) uint32_t hist[3][SEL_BINS];      // one per pass, so that one cluster barrier a pass is enough
    uint32_t wsum[32];
    uint32_t bin, left;
};
// Digits of 11, 11 and 10 bits from the top: each pass counts the keys that agree with what is settled so far by their next
// digit, adds the CTAs' counts up and settles the digit at which the count from above reaches k. key(i), i in [0, n): this
// CTA's keys. Returns a bound: the keys above it and `ties` of the keys equal to it are the k largest (1 <= k <= their
// number). Where all keys with the digits settled so far are among them, the rest is left open: the bound is the smallest
// key with these digits, and ties says all. All threads of all CTAs of the cluster call it; NT threads a CTA, CL: more than one CTA. Nothing is unrolled on
// purpose: code that runs once a call is paced by instruction fetches (unrolled, a pass took 5000 cycles).
__device__ __forceinline__ uint32_t hist_of(const uint4 &c, uint32_t i) { return i & 2u ? (i & 1u ? c.w : c.z) : (i & 1u ? c.y : c.x); }
template <int NT, bool CL, class KEY>
__device__ uint32_t select_kth(SelShared &s, int n, uint32_t k, uint32_t &ties, KEY key) {
    namespace cg = cooperative_groups;
    static_assert(SEL_BINS % (4 * NT) == 0 && NT % 32 == 0, "whole groups of four bins a thread");
    constexpr int BPT = SEL_BINS / NT;
    static_assert(BPT == 4, "a thread has four bins");
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    for (int i = tid; i < 3 * SEL_BINS / 4; i += NT) ((uint4 *)&s.hist[0][0])[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    uint32_t prefix = 0, settled = 0;            // settled: mask of the bits that prefix states
#pragma unroll 1
    for (int pass = 0; pass < 3; pass++) {
        const int sh = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const uint32_t dm = pass == 2 ? 1023u : 2047u;
        uint32_t *hist = s.hist[pass];
#pragma unroll 1
        for (int i0 = 0; i0 < n; i0 += NT) {     // lanes that agree with the first of their warp add once: equal keys are common
            const int i = i0 + tid;
            const uint32_t u = i < n ? key(i) : 0u;
            const bool in = i < n && (u & settled) == prefix;
            const uint32_t d = (u >> sh) & dm, m = __ballot_sync(0xffffffffu, in);
            if (m == 0) continue;
            const int lead = __ffs(m) - 1;
            const uint32_t d0 = __shfl_sync(0xffffffffu, d, lead), same = __ballot_sync(0xffffffffu, in && d == d0);
            if (in && (d != d0 || lane == lead)) atomicAdd(&hist[d], d == d0 ? (uint32_t)__popc(same) : 1u);
        }
        const int b = SEL_BINS - 4 - 4 * tid;    // thread t has bins b + 3 ... b
        uint4 c;
        if constexpr (CL) {
            cg::cluster_group cl = cg::this_cluster();
            cl.sync();
            c = make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int r = 0; r < 8; r++) {            // loads from the other CTAs all at once: each takes some 600 cycles
                if (r >= (int)cl.num_blocks()) break;
                const uint4 v = *(const uint4 *)(cl.map_shared_rank(hist, r) + b);
                c.x += v.x; c.y += v.y; c.z += v.z; c.w += v.w;
            }
        } else {
            __syncthreads();
            c = *(const uint4 *)(hist + b);
        }
        const uint32_t sum = c.x + c.y + c.z + c.w;
        uint32_t inc = sum;
#pragma unroll 1
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += v;
        }
        if (lane == 31) s.wsum[warp] = inc;
        __syncthreads();
        const uint32_t others = __reduce_add_sync(0xffffffffu, lane < warp ? s.wsum[lane] : 0u);
        uint32_t above = others + inc - sum;
        if (above < k && above + sum >= k) {
            uint32_t bin = b + 3;
            if (above + c.w < k) { above += c.w; bin--; if (above + c.z < k) { above += c.z; bin--; if (above + c.y < k) { above += c.y; bin--; } } }
            s.bin = bin;
            s.left = k - above == hist_of(c, bin & 3u) ? 0xffffffffu : k - above;
        }
        __syncthreads();
        prefix |= s.bin << sh;
        settled |= dm << sh;
        k = s.left;
        if (k == 0xffffffffu) break;             // all of them
    }
    if constexpr (CL) cg::this_cluster().sync();     // the others have read this CTA's counts
    ties = k;
    return prefix;
}
#endif

} // namespace ncmb
