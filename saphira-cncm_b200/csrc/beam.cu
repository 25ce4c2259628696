// The best continuations of groups of beams over beams and vocabulary (ncmb_beam_select, include/ncm_b200.h).
//
// score(k, w) = s_k + x_kw - log sum_w exp x_kw, s_k the beam's score so far; the n best of a group, in order. One pass over the logits: a CTA has a
// part of a row, in tiles of 16 values a thread; it keeps a running maximum and sum a thread and the part's n largest logits -- within a beam
// the order is that of its logits, so no more of them can be wanted. The last CTA of a group joins the parts.
//
// n largest: of the maxima of 2 n or more groups of threads the n-th largest is a bound that n values reach, and few values more; what
// reaches it goes to a list in shared memory. Later tiles have to beat the n-th of the list, which most do not: they cost a comparison a value.
// Keys are unique -- value, then lower index -- so equal values are no case of their own, and no order of arrival shows in the result. A bound is reached
// by at most n groups, so a tile adds at most half of its values to the list, whatever the values are.
//
// Rounding: exponentials in fp32 against the thread's maximum, 16 of them summed in fp32, everything after in 64 bits; scores in 64 bits, so that
// their order does not depend on the rounding of a score near 100 (2^-18 in fp32). All rows of a call are split alike: equal rows have equal sums.
#include "cache.cuh"

#include <algorithm>

namespace ncmb {
namespace {

constexpr int BM_THREADS = 256, BM_WARPS = BM_THREADS / 32;
constexpr int BM_EPT = 16, BM_TILE = BM_THREADS * BM_EPT;        // logits of a thread and a CTA at a time
constexpr int BM_JOIN = 4;                                       // candidates of a thread at a time where parts are joined
constexpr float BM_LOG2E = 1.44269504f;

struct BeamArgs {
    const char *x;
    int64_t ld;                      // bytes
    int groups, beams, V, n, parts, tiles;
    const float *scores; const int *done;
    int eos;
    float *scores_out; int *parents, *tokens, *done_out;
    unsigned long long *keys;        // scratch, [row][part][n]
    double2 *sums;                   // scratch, [row][part]: maximum, sum
    int *arrived;                    // scratch, [group], zero between calls
};

struct Wide { unsigned long long hi, lo; };      // score; then beam, logit, word
__device__ __forceinline__ bool operator>(const Wide &a, const Wide &b) { return a.hi > b.hi || (a.hi == b.hi && a.lo > b.lo); }
__device__ __forceinline__ bool bm_there(unsigned long long k) { return k != 0; }
__device__ __forceinline__ bool bm_there(const Wide &k) { return k.hi != 0; }
__device__ __forceinline__ unsigned long long bm_xor(unsigned long long k, int o) { return __shfl_xor_sync(0xffffffffu, k, o); }
__device__ __forceinline__ Wide bm_xor(const Wide &k, int o) { return Wide{__shfl_xor_sync(0xffffffffu, k.hi, o), __shfl_xor_sync(0xffffffffu, k.lo, o)}; }

// the n largest keys of tiles of EPT a thread
template <class K, int EPT> struct TopN {
    static constexpr int CAP = BM_THREADS * EPT / 2 + NCMB_MAX_BEAMS;            // n, and what a tile adds at most
    static constexpr int PER = (CAP + BM_THREADS - 1) / BM_THREADS;
    K list[CAP], few[NCMB_MAX_BEAMS * PER], groups[BM_THREADS], bound;
    int count, n_few, sums[BM_WARPS];

    __device__ void clear() {
        if (threadIdx.x == 0) { count = 0; bound = K{}; }
        __syncthreads();
    }
    // the n-th largest of the maxima of 2 n groups of threads or more; no key where fewer than n have one
    __device__ K nth(K best, int n) {
        int size = 8;
        while (size > 1 && BM_THREADS / size < 2 * n) size >>= 1;
        for (int o = 1; o < size; o <<= 1) { const K other = bm_xor(best, o); if (other > best) best = other; }
        const int tid = threadIdx.x, G = BM_THREADS / size;
        __syncthreads();
        if (tid % size == 0) groups[tid / size] = best;
        if (tid == 0) bound = K{};
        __syncthreads();
        if (tid < G) {
            const K mine = groups[tid];
            int rank = 0;
            for (int j = 0; j < G; j++) rank += groups[j] > mine;
            if (rank == n - 1 && bm_there(mine)) bound = mine;
        }
        __syncthreads();
        return bound;
    }
    // the list becomes its n largest, in order; returns the n-th, no key where there are fewer
    __device__ K settle(int n) {
        const int tid = threadIdx.x, c = count;
        int m = c;
        if (c > 128) {
            K best = K{};
            for (int i = tid; i < c; i += BM_THREADS) if (list[i] > best) best = list[i];
            const K least = nth(best, n);
            if (tid == 0) n_few = 0;
            __syncthreads();
            for (int i = tid; i < c; i += BM_THREADS) if (!(least > list[i])) few[atomicAdd(&n_few, 1)] = list[i];
        } else if (tid < c) {
            few[tid] = list[tid];
        }
        __syncthreads();
        if (c > 128) m = n_few;
        for (int i = tid; i < m; i += BM_THREADS) {
            const K mine = few[i];
            int rank = 0;
            for (int j = 0; j < m; j++) rank += few[j] > mine;
            if (rank < n) list[rank] = mine;
        }
        if (tid == 0) count = min(n, m);
        __syncthreads();
        return m >= n ? list[n - 1] : K{};
    }
    // the tile's keys that reach `least` (the n-th largest so far, or none) join the list; all threads call it. least is raised where the tile shows how far
    __device__ void add(const K (&key)[EPT], int n, K &least) {
        const int tid = threadIdx.x;
        auto joins = [&](int e) { return bm_there(key[e]) && !(least > key[e]); };
        for (int round = 0;; round++) {
            int c = 0;
#pragma unroll
            for (int e = 0; e < EPT; e++) c += joins(e);
            c = __reduce_add_sync(0xffffffffu, c);
            if ((tid & 31) == 0) sums[tid >> 5] = c;
            const int have = count;                              // before the barrier: after it others add to it
            __syncthreads();
            int total = 0;
#pragma unroll
            for (int w = 0; w < BM_WARPS; w++) total += sums[w];
            if ((bm_there(least) && have + total <= CAP) || round > 1) break;
            __syncthreads();
            if (round == 0 && have > n) {
                const K x = settle(n);
                if (x > least) least = x;
                continue;
            }
            K best = K{};
#pragma unroll
            for (int e = 0; e < EPT; e++) if (key[e] > best) best = key[e];
            const K x = nth(best, n);
            if (x > least) least = x;
            round = 1;
        }
#pragma unroll
        for (int e = 0; e < EPT; e++) if (joins(e)) list[atomicAdd(&count, 1)] = key[e];
        __syncthreads();
    }
};

__device__ __forceinline__ float bm_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t bm_order(float x) {          // larger is larger; no NaN, no -0
    const uint32_t u = __float_as_uint(x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float bm_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }
__device__ __forceinline__ unsigned long long bm_order(double x) {
    const unsigned long long u = __double_as_longlong(x);
    return u >> 63 ? ~u : u | 1ull << 63;
}
__device__ __forceinline__ double bm_value(unsigned long long k) { return __longlong_as_double(k >> 63 ? k ^ 1ull << 63 : ~k); }

union BeamShared {
    TopN<unsigned long long, BM_EPT> part;
    TopN<Wide, BM_JOIN> join;
};

// ---- a group's parts, by the last CTA that has one ----
__device__ void beam_join(const BeamArgs &a, int g, TopN<Wide, BM_JOIN> &top) {
    __shared__ double lse[NCMB_MAX_BEAMS], score[NCMB_MAX_BEAMS];
    __shared__ int over[NCMB_MAX_BEAMS];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, n = a.n;
    const int64_t row0 = (int64_t)g * a.beams;
    for (int k = warp; k < a.beams; k += BM_WARPS) {
        const double2 *s = a.sums + (row0 + k) * a.parts;
        const bool ended = a.done && a.done[row0 + k];
        double m = -INFINITY, t = 0;
        if (!ended) {
            for (int p = lane; p < a.parts; p += 32) m = fmax(m, __ldcg(&s[p].x));
            for (int o = 16; o; o >>= 1) m = fmax(m, __shfl_xor_sync(0xffffffffu, m, o));
            for (int p = lane; p < a.parts; p += 32) t += __ldcg(&s[p].y) * bm_exp2((float)(__ldcg(&s[p].x) - (m == -INFINITY ? 0 : m)) * BM_LOG2E);
            for (int o = 16; o; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
        }
        if (lane == 0) {
            const float sc = a.scores[row0 + k];
            lse[k] = ended || m == -INFINITY ? 0.0 : m + log(t);
            score[k] = sc == sc ? (double)sc : -INFINITY;
            over[k] = ended;
        }
    }
    top.clear();
    const unsigned long long *keys = a.keys + row0 * a.parts * n;
    const int total = a.beams * a.parts * n;
    Wide least = {};
    for (int i0 = 0; i0 < total; i0 += BM_THREADS * BM_JOIN) {
        Wide key[BM_JOIN];
#pragma unroll
        for (int e = 0; e < BM_JOIN; e++) {
            const int i = i0 + e * BM_THREADS + tid;
            key[e] = Wide{};
            if (i >= total) continue;
            const int k = i / (a.parts * n), j = i - k * (a.parts * n);
            uint32_t w;
            float x;
            if (over[k]) {                                       // its end, then the other words, which have nothing
                if (j >= min(n, a.V)) continue;
                w = j == 0 ? a.eos : j - 1 + (j - 1 >= a.eos);
                x = j == 0 ? 0.f : -INFINITY;
            } else {
                const unsigned long long u = __ldcg(keys + i);
                if (!u) continue;
                w = 0xffffffffu - (uint32_t)u;
                x = bm_value((uint32_t)(u >> 32));
            }
            const double sc = x == -INFINITY ? -INFINITY : score[k] + ((double)x - lse[k]) + 0.0;
            key[e] = Wide{bm_order(sc), (unsigned long long)(NCMB_MAX_BEAMS - 1 - k) << 56 | (unsigned long long)bm_order(x) << 24 | (0xffffffu - w)};
        }
        top.add(key, n, least);
    }
    top.settle(n);
    for (int i = tid; i < n; i += BM_THREADS) {
        const Wide x = top.list[i];
        const int k = NCMB_MAX_BEAMS - 1 - (int)(x.lo >> 56), w = 0xffffff - (int)(x.lo & 0xffffffu);
        const int64_t at = (int64_t)g * n + i;
        a.scores_out[at] = (float)bm_value(x.hi);
        a.parents[at] = k;
        a.tokens[at] = w;
        if (a.done_out) a.done_out[at] = over[k] || w == a.eos;
    }
}

// CTA (row, part). VEC: rows of whole 16 bytes
template <class E, bool VEC>
__global__ void __launch_bounds__(BM_THREADS) k_beam_select(const __grid_constant__ BeamArgs a) {
    __shared__ BeamShared sh;
    __shared__ double reduce[BM_WARPS];
    __shared__ float rmax[BM_WARPS];
    __shared__ int last;
    constexpr int VE = 16 / sizeof(E), NV = BM_EPT / VE;         // elements of 16 bytes, vectors of a thread
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int64_t row = blockIdx.x / a.parts;
    const int part = (int)(blockIdx.x - row * a.parts), g = (int)(row / a.beams);
    pdl_wait();
    pdl_launch_dependents();
    if (!(a.done && a.done[row])) {
        const int t0 = (int)((int64_t)part * a.tiles / a.parts), t1 = (int)((int64_t)(part + 1) * a.tiles / a.parts);
        const E *x0 = (const E *)(a.x + row * a.ld);
        auto word = [&](int t, int e) { return t * BM_TILE + (VEC ? (e / VE * BM_THREADS + tid) * VE + e % VE : e * BM_THREADS + tid); };
        auto load = [&](int t, float (&x)[BM_EPT]) {
            if constexpr (VEC) {
#pragma unroll
                for (int i = 0; i < NV; i++) {
                    const int w = word(t, i * VE);
                    if (w + VE > a.V) {                          // the row's end
#pragma unroll
                        for (int e = 0; e < VE; e++) x[i * VE + e] = w + e < a.V ? (float)x0[w + e] : -INFINITY;
                        continue;
                    }
                    const uint4 u = __ldcs((const uint4 *)(x0 + w));
                    const uint32_t uu[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                    for (int e = 0; e < VE; e++) {
                        if constexpr (sizeof(E) == 4) x[i * VE + e] = __uint_as_float(uu[e]);
                        else x[i * VE + e] = __uint_as_float(e & 1 ? uu[e / 2] & 0xffff0000u : uu[e / 2] << 16);
                    }
                }
            } else {
#pragma unroll
                for (int e = 0; e < BM_EPT; e++) {
                    const int w = word(t, e);
                    x[e] = w < a.V ? (float)x0[w] : -INFINITY;
                }
            }
        };
        sh.part.clear();
        unsigned long long least = 0;
        float m = -INFINITY, beat = -INFINITY;                   // beat: what a logit has to exceed, once the list is full
        double s = 0;
        float ahead[BM_EPT];
        load(t0, ahead);
        for (int t = t0; t < t1; t++) {
            float x[BM_EPT];
#pragma unroll
            for (int e = 0; e < BM_EPT; e++) x[e] = fminf(fmaxf(ahead[e], -INFINITY), 3.402823466e38f);     // a NaN is -infinity
            if (t + 1 < t1) load(t + 1, ahead);
            float tm = x[0];
#pragma unroll
            for (int e = 1; e < BM_EPT; e++) tm = fmaxf(tm, x[e]);
            if (tm > m) {
                s *= bm_exp2((m - tm) * BM_LOG2E);
                m = tm;
            }
            const float base = m == -INFINITY ? 0.f : m;
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int e = 0; e < BM_EPT; e++) sum[e & 3] += bm_exp2((x[e] - base) * BM_LOG2E);
            s += (double)((sum[0] + sum[1]) + (sum[2] + sum[3]));
            if (!__syncthreads_or(least == 0 || tm > beat)) continue;
            unsigned long long key[BM_EPT];
#pragma unroll
            for (int e = 0; e < BM_EPT; e++) {
                const int w = word(t, e);
                key[e] = w < a.V ? (unsigned long long)bm_order(x[e] + 0.f) << 32 | (0xffffffffu - w) : 0ull;
            }
            sh.part.add(key, a.n, least);
            beat = bm_value((uint32_t)(least >> 32));
        }
        sh.part.settle(a.n);
        // the part's list, maximum and sum
        for (int i = tid; i < a.n; i += BM_THREADS) a.keys[(row * a.parts + part) * a.n + i] = i < sh.part.count ? sh.part.list[i] : 0ull;
        float top = m;
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (lane == 0) rmax[warp] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < BM_WARPS; w++) top = fmaxf(top, rmax[w]);
        s *= m == -INFINITY ? 0.f : bm_exp2((m - top) * BM_LOG2E);
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0) reduce[warp] = s;
        __syncthreads();
        if (tid == 0) {
            s = 0;
            for (int w = 0; w < BM_WARPS; w++) s += reduce[w];
            a.sums[row * a.parts + part] = make_double2(top, s);
        }
    }
    __threadfence();
    __syncthreads();
    if (tid == 0) last = atomicAdd(&a.arrived[g], 1) == a.beams * a.parts - 1;
    __syncthreads();
    if (!last) return;
    if (tid == 0) a.arrived[g] = 0;                              // for the next call
    __threadfence();
    beam_join(a, g, sh.join);
}

} // namespace
} // namespace ncmb

using namespace ncmb;

extern "C" int ncmb_beam_select(const void *logits, int64_t ldl, int type, int groups, int beams, int V, const float *scores, const int *done, int eos,
                                int n_out, float *scores_out, int *parents, int *tokens, int *done_out) {
    const char *who = "ncmb_beam_select";
    if (type != NCMB_F32 && type != NCMB_BF16) return cache_refuse(who, "logits of type %d", type);
    if (groups < 0 || beams < 1 || beams > NCMB_MAX_BEAMS || V < 1 || V > 1 << 24) return cache_refuse(who, "%d groups of %d beams (at most %d), %d words (at most 2^24)", groups, beams, NCMB_MAX_BEAMS, V);
    if (n_out < 1 || n_out > NCMB_MAX_BEAMS || n_out > (int64_t)beams * V) return cache_refuse(who, "%d continuations of %d x %d: at most %d", n_out, beams, V, NCMB_MAX_BEAMS);
    if (done ? eos < 0 || eos >= V : eos >= V) return cache_refuse(who, "word %d of %d ends a beam", eos, V);
    if (groups == 0) return 0;
    const int64_t es = type == NCMB_BF16 ? 2 : 4, rows = (int64_t)groups * beams;
    if (ldl < V) return cache_refuse(who, "rows of %lld logits, %d words", (long long)ldl, V);
    if (!logits || !scores || !scores_out || !parents || !tokens) return cache_refuse(who, "a null pointer");
    if ((uintptr_t)logits % es || ((uintptr_t)scores | (uintptr_t)done | (uintptr_t)scores_out | (uintptr_t)parents | (uintptr_t)tokens | (uintptr_t)done_out) % 4)
        return cache_refuse(who, "arrays have to be aligned to their elements");
    if (rows > 1 << 24) return cache_refuse(who, "%lld rows", (long long)rows);
    if (cache_device(who)) return -1;
    BeamArgs a = {};
    a.x = (const char *)logits; a.ld = ldl * es; a.groups = groups; a.beams = beams; a.V = V; a.n = n_out;
    a.tiles = (int)cdiv(V, BM_TILE);
    a.scores = scores; a.done = done; a.eos = eos; a.scores_out = scores_out; a.parents = parents; a.tokens = tokens; a.done_out = done_out;
    // parts of a row: three rounds of the CTAs that fit the GPU, so that its last round is nearly full, but no more candidates than one CTA joins quickly
    const int64_t slots = 4LL * ctx().sm_count;
    a.parts = (int)std::max<int64_t>(1, std::min<int64_t>({a.tiles, cdiv(3 * slots, rows), 16384 / ((int64_t)beams * n_out)}));
    const size_t kb = (size_t)rows * a.parts * n_out * 8, sb = (size_t)rows * a.parts * sizeof(double2);
    char *scratch = (char *)cache_scratch(who, sb + kb);
    if (!scratch) return -1;
    a.sums = (double2 *)scratch;
    a.keys = (unsigned long long *)(scratch + sb);
    if (!(a.arrived = (int *)cache_scratch(who, (size_t)groups * 4, SCRATCH_DONE))) return -1;
    ProfScope prof(NCMB_K_SAMPLE, 4.0 * rows * V, (double)rows * V * es);
    const bool vec = (uintptr_t)logits % 16 == 0 && a.ld % 16 == 0;
    const unsigned grid = (unsigned)(rows * a.parts);
    if (type == NCMB_F32) { if (vec) LAUNCH_PDL((k_beam_select<float, true>), grid, BM_THREADS, 0, a); else LAUNCH_PDL((k_beam_select<float, false>), grid, BM_THREADS, 0, a); }
    else if (vec) LAUNCH_PDL((k_beam_select<__nv_bfloat16, true>), grid, BM_THREADS, 0, a);
    else LAUNCH_PDL((k_beam_select<__nv_bfloat16, false>), grid, BM_THREADS, 0, a);
    return 0;
}
