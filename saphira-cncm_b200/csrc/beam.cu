// The best continuations of groups of beams over beams and vocabulary (ncmb_beam_select, include/ncm_b200.h).
//
// score(k, w) = s_k + x_kw - log sum_w exp x_kw, s_k the beam's score so far; the n best of a group, in order. One pass over the logits: a CTA has a
// part of a row, in tiles of 32 values a thread; it keeps a running maximum and sum a thread and the part's n largest logits -- within a beam
// the order is that of its logits, so no more of them can be wanted. The last CTA of a group joins the parts.
//
// n largest: of the maxima of 2 n or more groups of threads the n-th largest is a bound that n values reach, and few values more; what
// reaches it goes to a list in shared memory, as does what beats the bound in later tiles; a list that fills up is cut to its n largest, and the
// bound is theirs. So a value costs a comparison, and few more. Keys are unique -- value, then lower index -- so equal values are no case of
// their own, and no order of arrival shows in the result. However the values lie, a bound is reached by n groups at most, so a few values a thread
// at a time always fit the list; tiles of which more beat an older bound than there is room for are gone through once more that way.
//
// Rounding: exponentials in fp32 against the thread's maximum, 32 of them summed in fp32 -- 64 bits from a value on would be several instructions more for
// each --, everything after in 64 bits: log sum exp within 5e-7 where roundings do not average, 2e-8 where they do. Scores in 64 bits, so that
// their order does not depend on the rounding of a score near 100 (2^-18 in fp32). All rows of a call are split alike: equal rows have equal sums.
//
// Bound: with many rows by the SMs that have most of them -- 256 rows of 151936 in fp32: 37 us (4.2 TB/s), of which an SM that has two of them
// streams 27 at 48 GB/s; in bf16 33: an SM is active in 46 000 of 70 000 cycles on the average and issues in 38% of those, its warps wait for fixed
// latencies and for one another. With few by latency: 4 rows of 50257, 9.4 us, 40% of it the join.
#include "paged.cuh"

#include <algorithm>

namespace ncmb {
namespace {

constexpr int BM_THREADS = 256, BM_WARPS = BM_THREADS / 32;
constexpr int BM_EPT = 32, BM_TILE = BM_THREADS * BM_EPT;        // logits of a thread and a CTA at a time
constexpr int BM_CHUNK = 8;                                      // logits of a thread whose keys fit the list whatever they are, once they are bounded
constexpr int BM_JOIN = 2;                                       // candidates of a thread at a time where parts are joined
constexpr int BM_BATCH = 4;                                      // tiles from one meeting of the warps to the next
constexpr int BM_START = 2, BM_ROUNDS = 4, BM_CTAS = 2;          // BM_CTAS: of an SM; with three, 80 registers a thread leave less to overlap (then 39 -> 47 us)
constexpr int BM_FEW = 16;                                       // continuations that most calls want
constexpr float BM_LOG2E = 1.44269504f;

struct alignas(16) PartSum { double sum; float top, unused; };     // of exponentials against the part's maximum
struct BeamArgs {
    const char *x;
    int64_t ld;                      // bytes
    int groups, beams, V, n, parts, tiles;
    int slots;                       // keys that a part leaves: 2 n in any order where one tile joins them all, so that most need not settle which; else n in order
    const float *scores; const int *done;
    int eos;
    float *scores_out; int *parents, *tokens, *done_out;
    unsigned long long *keys;        // scratch, [group][slot][beam][part]
    PartSum *sums;                   // scratch, [row][part]
    int *arrived;                    // scratch, [group], zero between calls
};

struct Wide { unsigned long long hi, lo; };      // score; then beam, logit, word
__device__ __forceinline__ bool operator>(const Wide &a, const Wide &b) { return (a.hi > b.hi) | ((a.hi == b.hi) & (a.lo > b.lo)); }       // without branches: many of them are in a row
__device__ __forceinline__ bool bm_there(unsigned long long k) { return k != 0; }
__device__ __forceinline__ bool bm_there(const Wide &k) { return k.hi != 0; }
__device__ __forceinline__ unsigned long long bm_xor(unsigned long long k, int o) { return __shfl_xor_sync(0xffffffffu, k, o); }
__device__ __forceinline__ Wide bm_xor(const Wide &k, int o) { return Wide{__shfl_xor_sync(0xffffffffu, k.hi, o), __shfl_xor_sync(0xffffffffu, k.lo, o)}; }

// The n-th largest of the maxima of 2 n groups of threads or more (of 8 threads at most); no key where fewer than n have one. One copy of the code for
// whoever wants it: a part's first tile, lists that are cut, the join. Code that runs once is paced by instruction fetches.
template <class K> __device__ __noinline__ K bm_nth(K best, int n, K *groups, K *bound) {
    const int lg = min(3, __clz(2 * n - 1) - 24), size = 1 << lg;           // BM_THREADS >> lg is 2 n or more
#pragma unroll 1
    for (int o = 1; o < size; o <<= 1) { const K other = bm_xor(best, o); if (other > best) best = other; }
    const int tid = threadIdx.x, G = BM_THREADS >> lg, mine = tid >> lg;
    __syncthreads();
    if ((tid & (size - 1)) == 0) groups[mine] = best;
    if (tid == 0) *bound = K{};
    __syncthreads();
    int rank = 0;                        // a group's threads share the comparisons with the others; of equal keys the lower group is first
#pragma unroll 4
    for (int j = tid & (size - 1); j < G; j += size) { const K other = groups[j]; rank += (other > best) | ((j < mine) & !(best > other)); }
#pragma unroll 1
    for (int o = 1; o < size; o <<= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
    if ((tid & (size - 1)) == 0 && rank == n - 1 && bm_there(best)) *bound = best;
    __syncthreads();
    return *bound;
}

// The n largest keys of tiles of EPT a thread; n up to MOST, BM_FEW or NCMB_MAX_BEAMS: the fewer, the less room the lists take.
// ROOM: keys that the list holds beside 2 n; 0: what a tile adds at most, once it has a bound.
template <class K, int EPT, int MOST, int ROOM = 0> struct TopN {
    static constexpr int REACH = BM_THREADS / 2;                 // threads whose groups reach a bound, at most: n groups of 2 n or more
    static constexpr int CAP = (ROOM ? ROOM : REACH * EPT) + 2 * MOST;
    static constexpr int PER = (CAP + BM_THREADS - 1) / BM_THREADS;
    K list[CAP], few[REACH * PER > BM_THREADS / 2 ? REACH * PER : BM_THREADS / 2], groups[BM_THREADS], bound;
    int count, n_few, sums[BM_WARPS];

    __device__ void clear() {
        if (threadIdx.x == 0) { count = 0; bound = K{}; }
        __syncthreads();
    }
    __device__ K nth(K best, int n) { return bm_nth(best, n, groups, &bound); }
    // use(key, rank) for each of m keys
    template <class USE> __device__ void ranks(const K *keys, int m, USE use) {
        const int lg = m <= BM_THREADS / 8 ? 3 : m <= BM_THREADS / 4 ? 2 : m <= BM_THREADS / 2 ? 1 : 0, ways = 1 << lg, tid = threadIdx.x;      // threads that share a key's comparisons
#pragma unroll 1
        for (int i0 = 0; i0 < m; i0 += BM_THREADS >> lg) {
            const int i = i0 + (tid >> lg);
            const K mine = keys[min(i, m - 1)];
            int rank = 0;
#pragma unroll 4
            for (int j = tid & (ways - 1); j < m; j += ways) rank += keys[j] > mine;
#pragma unroll 1
            for (int o = 1; o < ways; o <<= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
            if (i < m && (tid & (ways - 1)) == 0) use(mine, rank);
        }
    }
    // the list becomes its n largest, in order; returns the n-th, no key where there are fewer
    __device__ K settle(int n) {
        const int tid = threadIdx.x, c = count;
        int m = c;
        if (c > BM_THREADS / 2) {
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
        if (c > BM_THREADS / 2) m = n_few;
        ranks(few, m, [&](const K &key, int rank) { if (rank < n) list[rank] = key; });
        if (tid == 0) count = min(n, m);
        __syncthreads();
        return m >= n ? list[n - 1] : K{};
    }
    // the tile's keys -- key(e), e < EPT, of this thread -- that reach `least` (a bound that n keys reach, or none) join the list; all threads call it.
    // least is raised where the tile shows how far
    template <class KEY> __device__ void add(int n, K &least, KEY key) {
        const int tid = threadIdx.x;
        auto joins = [&](const K &k) { return bm_there(k) && !(least > k); };
        if (!bm_there(least)) raise(n, least, key);
        for (int round = 0;; round++) {
            int c = 0;
#pragma unroll 4
            for (int e = 0; e < EPT; e++) c += joins(key(e));
            c = __reduce_add_sync(0xffffffffu, c);
            if ((tid & 31) == 0) sums[tid >> 5] = c;
            const int have = count;      // before the barrier: after it others add to it
            __syncthreads();
            int total = 0;
#pragma unroll
            for (int w = 0; w < BM_WARPS; w++) total += sums[w];
            if (have + total <= CAP || round == 2) break;
            __syncthreads();
            if (round == 0) {
                const K x = settle(n);
                if (x > least) least = x;
            } else {
                raise(n, least, key);
            }
        }
#pragma unroll 4
        for (int e = 0; e < EPT; e++) {
            const K k = key(e);
            if (joins(k)) list[atomicAdd(&count, 1)] = k;
        }
        __syncthreads();
    }
    // of a settled list, the keys whose lower half is at most `low`
    __device__ void drop(uint32_t low) {
        const int tid = threadIdx.x;
        const bool stays = tid < count && (uint32_t)list[min(tid, CAP - 1)] > low;
        const K mine = list[min(tid, CAP - 1)];
        __syncthreads();
        if (tid == 0) count = 0;
        __syncthreads();
        if (stays) list[atomicAdd(&count, 1)] = mine;
        __syncthreads();
    }
    // least: up to what n keys of the tile reach
    template <class KEY> __device__ void raise(int n, K &least, KEY key) {
        K best = K{};
#pragma unroll
        for (int e = 0; e < EPT; e++) { const K k = key(e); if (k > best) best = k; }
        const K x = nth(best, n);
        if (x > least) least = x;
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
__device__ __forceinline__ float bm_clamp(float x) { return fminf(fmaxf(x, -INFINITY), 3.402823466e38f); }      // a NaN is -infinity
__device__ __forceinline__ unsigned long long bm_key(float x, int w) {       // of a logit; -0 is 0. Bits 24 ... 31 are free
    return (unsigned long long)bm_order(x + 0.f) << 32 | (0xffffffu - (uint32_t)w);
}
__device__ __forceinline__ float bm_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }
__device__ __forceinline__ unsigned long long bm_order(double x) {
    const unsigned long long u = __double_as_longlong(x);
    return u >> 63 ? ~u : u | 1ull << 63;
}
__device__ __forceinline__ double bm_value(unsigned long long k) { return __longlong_as_double(k >> 63 ? k ^ 1ull << 63 : ~k); }

// ---- a group's parts, by the last CTA that has one ----
template <int MOST> struct JoinShared {
    TopN<Wide, BM_JOIN, MOST, BM_JOIN * BM_THREADS> top;         // a whole tile fits
    unsigned long long bound;
    double lse[NCMB_MAX_BEAMS], score[NCMB_MAX_BEAMS];
    int over[NCMB_MAX_BEAMS];
};
// score, ended: of beam threadIdx.x, read when the kernel began
template <int MOST> __device__ __noinline__ void beam_join(const BeamArgs &a, int g, float score, bool ended, JoinShared<MOST> &sh) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, n = a.n, slots = a.slots;
    const int64_t row0 = (int64_t)g * a.beams;
    const int lists = a.beams * a.parts, total = lists * slots;
    const unsigned long long *keys = a.keys + (int64_t)g * total;
    unsigned long long u[BM_JOIN];
    auto load = [&](int i0) {
#pragma unroll
        for (int e = 0; e < BM_JOIN; e++) {
            const int i = i0 + e * BM_THREADS + tid;
            u[e] = i < total ? __ldcg(keys + i) : 0;
        }
    };
    load(0);                                                     // on their way while the sums meet
    if (tid < a.beams) {
        sh.score[tid] = score == score ? (double)score : -INFINITY;
        sh.over[tid] = ended;
    }
    __syncthreads();
    for (int k = warp; k < a.beams; k += BM_WARPS) {
        const PartSum *s = a.sums + (row0 + k) * a.parts;
        float m = -INFINITY;
        double t = 0;
        if (!sh.over[k]) {
#pragma unroll 1
            for (int p = lane; p < a.parts; p += 32) {
                const float4 x = __ldcg((const float4 *)(s + p));
                const float top = fmaxf(m, x.z), base = top == -INFINITY ? 0.f : top;
                t = t * bm_exp2((m - base) * BM_LOG2E) + __hiloint2double(__float_as_int(x.y), __float_as_int(x.x)) * bm_exp2((x.z - base) * BM_LOG2E);
                m = top;
            }
            float top = m;
#pragma unroll 1
            for (int o = 1; o < min(32, a.parts); o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            t *= bm_exp2((m - (top == -INFINITY ? 0.f : top)) * BM_LOG2E);
#pragma unroll 1
            for (int o = 1; o < min(32, a.parts); o <<= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
            m = top;
        }
        if (lane == 0) sh.lse[k] = m == -INFINITY ? 0.0 : m + log(t);
    }
    sh.top.clear();
    unsigned long long least = 0;
    const int limit = min(3 * n + 8, 2 * MOST);                  // fewer are in the list when a tile begins, so the tile fits
#pragma unroll 1
    for (int i0 = 0; i0 < total; i0 += BM_THREADS * BM_JOIN) {
        Wide key[BM_JOIN];
#pragma unroll
        for (int e = 0; e < BM_JOIN; e++) {
            const int k = NCMB_MAX_BEAMS - 1 - (int)(u[e] >> 24 & 0x7f);
            const float x = bm_value((uint32_t)(u[e] >> 32));
            const double sc = x == -INFINITY ? -INFINITY : sh.score[k] + ((double)x - sh.lse[k]) + 0.0;
            key[e] = u[e] ? Wide{bm_order(sc), (u[e] >> 24 & 0x7f) << 56 | u[e] >> 32 << 24 | (u[e] & 0xffffff)} : Wide{};
        }
        load(i0 + BM_THREADS * BM_JOIN);
        if (least == 0) {                                        // by the scores alone: those that are equal to the n-th join too
            unsigned long long most = 0;
#pragma unroll
            for (int e = 0; e < BM_JOIN; e++) most = max(most, key[e].hi);
            least = bm_nth(most, n, (unsigned long long *)sh.top.groups, &sh.bound);
        }
        bool full = false, any = false;
#pragma unroll
        for (int e = 0; e < BM_JOIN; e++) {
            if (!bm_there(key[e]) || key[e].hi < least) continue;
            const int at = atomicAdd(&sh.top.count, 1);
            sh.top.list[at] = key[e];
            full |= at >= limit;
            any = true;
        }
        // in order, and none of the next of each list is among the best: nor are those behind
        if (slots == n && lists <= BM_THREADS * BM_JOIN && !__syncthreads_or(any)) break;
        if (__syncthreads_or(full)) {
            const Wide nth = sh.top.settle(n);
            least = max(least, nth.hi);
        }
    }
    // the n best to where their ranks say
    if (sh.top.count > BM_THREADS / 2) sh.top.settle(n);
    sh.top.ranks(sh.top.list, sh.top.count, [&](const Wide &x, int rank) {
        if (rank >= n) return;
        const int k = NCMB_MAX_BEAMS - 1 - (int)(x.lo >> 56), w = 0xffffff - (int)(x.lo & 0xffffffu);
        const int64_t at = (int64_t)g * n + rank;
        a.scores_out[at] = (float)bm_value(x.hi);
        a.parents[at] = k;
        a.tokens[at] = w;
        if (a.done_out) a.done_out[at] = sh.over[k] || w == a.eos;
    });
}

// ---- CTA (row, part) ----
// One tile of fp32 is on its way while another is worked on, or two of bf16
template <class E, int MOST> struct PartShared {
    static constexpr int STAGES = sizeof(E) == 4 ? 2 : 3;
    E ring[STAGES][BM_TILE];
    TopN<unsigned long long, BM_CHUNK, MOST> top;
    double sums[BM_WARPS];
    float maxima[BM_WARPS];
};
template <class E, int MOST> constexpr size_t beam_smem() { return std::max(sizeof(PartShared<E, MOST>), sizeof(JoinShared<MOST>)); }

template <int VE> __device__ __forceinline__ int bm_place(int e) { return (e / VE * BM_THREADS + (int)threadIdx.x) * VE + e % VE; }     // of a thread's e-th value in a tile
// Tiles [t0, t1), of whose keys some found no room in the list: once more, a few values a thread at a time, each time bounded by what these show.
// Rare: their values rise from tile to tile, or most of the large ones lie with few threads.
template <class E, bool VEC, int MOST>
__device__ __noinline__ void beam_again(const E *x0, int t0, int t1, int V, int n, TopN<unsigned long long, BM_CHUNK, MOST> &top, unsigned long long &least) {
    constexpr int VE = VEC ? 16 / (int)sizeof(E) : 1;
    top.drop(0xffffffu - t0 * BM_TILE);
    for (int t = t0; t < t1; t++)
        for (int e0 = 0; e0 < BM_EPT; e0 += BM_CHUNK)
            top.add(n, least, [&](int e) {
                const int w = t * BM_TILE + bm_place<VE>(e0 + e);
                return w < V ? bm_key(bm_clamp((float)x0[w]), w) : 0ull;
            });
}

// Tiles come through a ring in shared memory; a thread reads what it has copied itself, so no barrier is in between. VEC: rows of whole 16 bytes. Else a
// thread's values are a CTA's width apart: 4 bytes a copy, and through registers those of 2 bytes.
template <class E, bool VEC, int MOST>
__global__ void __launch_bounds__(BM_THREADS, BM_CTAS) k_beam_select(const __grid_constant__ BeamArgs a) {
    extern __shared__ __align__(16) char smem[];
    __shared__ int last;
    using Shared = PartShared<E, MOST>;
    Shared &sh = *(Shared *)smem;
    constexpr int STAGES = Shared::STAGES, VE = VEC ? 16 / (int)sizeof(E) : 1, NV = BM_EPT / VE;      // elements together, how many of them
    constexpr bool ASYNC = VEC || sizeof(E) == 4;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int64_t row = blockIdx.x / a.parts;
    const int part = (int)(blockIdx.x - row * a.parts), g = (int)(row / a.beams);
    pdl_wait();
    pdl_launch_dependents();
    const int lists = a.beams * a.parts, beam = (int)(row - (int64_t)g * a.beams);
    auto leave = [&](int i, unsigned long long key) {            // as slot i of the part, with its beam
        a.keys[((int64_t)g * a.slots + i) * lists + beam * a.parts + part] = key ? key | (unsigned long long)(NCMB_MAX_BEAMS - 1 - beam) << 24 : 0ull;
    };
    const bool mine = tid < a.beams;
    const float score = mine ? a.scores[(int64_t)g * a.beams + tid] : 0.f;       // for the join, should this CTA do it
    const bool ended = mine && a.done && a.done[(int64_t)g * a.beams + tid];
    if (a.done && a.done[row]) {                                 // its end, then the other words, which have nothing
        for (int i = tid; i < a.slots; i += BM_THREADS)
            leave(i, part > 0 || i >= min(a.n, a.V) ? 0ull : i == 0 ? bm_key(0.f, a.eos) : bm_key(-INFINITY, i - 1 + (i - 1 >= a.eos)));
    } else {
        const int t0 = (int)((int64_t)part * a.tiles / a.parts), t1 = (int)((int64_t)(part + 1) * a.tiles / a.parts);
        const E *x0 = (const E *)(a.x + row * a.ld);
        auto place = [&](int e) { return bm_place<VE>(e); };
        E wait[ASYNC ? 1 : BM_EPT];
        auto load = [&](int t, int stage) {
            if (t < t1) {
                const int left = a.V - t * BM_TILE;
                const E *from = x0 + (int64_t)t * BM_TILE + place(0);
                if constexpr (ASYNC) {
                    const uint32_t to = (uint32_t)__cvta_generic_to_shared(&sh.ring[stage][place(0)]);
                    constexpr int STEP = BM_THREADS * VE;                    // from one copy of a thread to its next
                    if (left >= BM_TILE) {
#pragma unroll
                        for (int i = 0; i < NV; i++) {
                            const uint32_t dst = to + i * STEP * (int)sizeof(E);
                            if constexpr (VEC) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(from + i * STEP) : "memory");
                            else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(from + i * STEP) : "memory");
                        }
                    } else {                                     // the row's end: a loop, so that whole tiles do not go through its instructions
#pragma unroll 2
                        for (int i = 0; i < NV; i++) {
                            const uint32_t dst = to + i * STEP * (int)sizeof(E);
                            const int bytes = max(0, min(VE, left - place(i * VE))) * (int)sizeof(E);
                            if constexpr (VEC) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(bytes ? from + i * STEP : x0), "r"(bytes) : "memory");
                            else asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(bytes ? from + i * STEP : x0), "r"(bytes) : "memory");
                        }
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < BM_EPT; e++) wait[e] = place(e) < left ? from[e * BM_THREADS] : E(0.f);
                }
            }
            if constexpr (ASYNC) asm volatile("cp.async.commit_group;" ::: "memory");
        };
        constexpr int AHEAD = ASYNC ? STAGES - 1 : 1;
#pragma unroll
        for (int i = 0; i < AHEAD; i++) load(t0 + i, i);
        sh.top.clear();
        unsigned long long least = 0;
        float m = -INFINITY, beat = -INFINITY;                   // beat: what a logit has to exceed, once there is a bound
        double s = 0;
        const int limit = min(3 * a.n + 8, sh.top.CAP / 2);      // a list of so many is cut: the bound that gives spares more than it costs
        bool full = false;
        int since = t0;                                          // the tile after the last at which all warps met
#pragma unroll 1
        for (int t = t0, stage = 0; t < t1; t++) {
            E *mine = sh.ring[stage];
            if constexpr (!ASYNC) {
#pragma unroll
                for (int e = 0; e < BM_EPT; e++) mine[place(e)] = wait[e];
            }
            load(t + AHEAD, stage + AHEAD < STAGES ? stage + AHEAD : stage + AHEAD - STAGES);
            if constexpr (ASYNC) asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD) : "memory");
            const int end = a.V - t * BM_TILE;                   // words of the row from this tile on
            if (end < BM_TILE) {
#pragma unroll 4
                for (int e = 0; e < BM_EPT; e++) if (place(e) >= end) mine[place(e)] = E(-INFINITY);
            }
            float x[BM_EPT];
#pragma unroll
            for (int i = 0; i < NV; i++) {
                if constexpr (VEC) {
                    const uint4 u = *(const uint4 *)(mine + place(i * VE));
                    const uint32_t uu[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                    for (int e = 0; e < VE; e++) {
                        if constexpr (sizeof(E) == 4) x[i * VE + e] = __uint_as_float(uu[e]);
                        else x[i * VE + e] = __uint_as_float(e & 1 ? uu[e / 2] & 0xffff0000u : uu[e / 2] << 16);
                    }
                } else x[i] = (float)mine[place(i)];
            }
            float tm, sum, top;                                  // sum: of exponentials against the new maximum
#pragma unroll 1
            for (;;) {
#pragma unroll
                for (int i = 0; i < BM_EPT / 4; i++) {
                    const float quad = fmaxf(fmaxf(x[4 * i], x[4 * i + 1]), fmaxf(x[4 * i + 2], x[4 * i + 3]));
                    tm = i ? fmaxf(tm, quad) : quad;
                }
                top = fmaxf(m, tm);
                const float base = top == -INFINITY ? 0.f : -top;
                float2 part[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                for (int i = 0; i < BM_EPT / 2; i++) {
                    const float2 d = __fmul2_rn(__fadd2_rn(make_float2(x[2 * i], x[2 * i + 1]), make_float2(base, base)), make_float2(BM_LOG2E, BM_LOG2E));
                    part[i & 1] = __fadd2_rn(part[i & 1], make_float2(bm_exp2(d.x), bm_exp2(d.y)));
                }
                sum = (part[0].x + part[0].y) + (part[1].x + part[1].y);
                if (sum < INFINITY) break;
#pragma unroll
                for (int e = 0; e < BM_EPT; e++) x[e] = bm_clamp(x[e]);              // a NaN or +infinity among them
            }
            if (top > m) {
                s *= bm_exp2((m - top) * BM_LOG2E);
                m = top;
            }
            s += (double)sum;
            if (least == 0) {                                    // the first tile
                float most = tm;
                asm volatile("" : "+f"(most));                   // not formed ahead of the branch, where every tile would pay for it
                uint32_t which = 0;
#pragma unroll
                for (int e = 0; e < BM_EPT; e++) if (x[e] == most) which |= 1u << e;
                const int at = place(__ffs(which) - 1);          // of the thread's largest, of equal ones the first
                least = sh.top.nth(at < end ? bm_key(most, t * BM_TILE + at) : 0ull, a.n);
                if (least) beat = bm_value((uint32_t)(least >> 32));
            }
            if (tm >= beat) {
                uint32_t hits = 0;
#pragma unroll
                for (int e = 0; e < BM_EPT; e++) if (x[e] >= beat) hits |= 1u << e;
#pragma unroll 1
                for (; hits; hits &= hits - 1) {
                    const int e = place(__ffs(hits) - 1);
                    const unsigned long long key = bm_key(bm_clamp((float)mine[e]), t * BM_TILE + e);
                    if (key < least || e >= end) continue;
                    const int at = atomicAdd(&sh.top.count, 1);
                    if (at < sh.top.CAP) sh.top.list[at] = key;
                    full |= at >= limit;
                }
            }
            // warps meet every few tiles only: the one with most hits is not waited for
            if (t + 1 - since == BM_BATCH || t + 1 == t1) {
                if (__syncthreads_or(full)) {
                    const bool lost = sh.top.count > sh.top.CAP; // keys that found no room
                    __syncthreads();
                    if (lost && tid == 0) sh.top.count = sh.top.CAP;
                    __syncthreads();
                    const unsigned long long nth = sh.top.settle(a.n);
                    if (nth > least) least = nth;
                    if (lost) beam_again<E, VEC, MOST>(x0, since, t + 1, a.V, a.n, sh.top, least);
                    if (least) beat = bm_value((uint32_t)(least >> 32));
                }
                full = false;
                since = t + 1;
            }
            if (++stage == STAGES) stage = 0;
        }
        // what may be among the n best, and the part's maximum and sum
        if (sh.top.count > a.slots || a.slots == a.n) sh.top.settle(a.n);
        for (int i = tid; i < a.slots; i += BM_THREADS) leave(i, i < sh.top.count ? sh.top.list[i] : 0ull);
        float top = m;
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (lane == 0) sh.maxima[warp] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < BM_WARPS; w++) top = fmaxf(top, sh.maxima[w]);
        s *= m == -INFINITY ? 0.f : bm_exp2((m - top) * BM_LOG2E);
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0) sh.sums[warp] = s;
        __syncthreads();
        if (tid == 0) {
            s = 0;
            for (int w = 0; w < BM_WARPS; w++) s += sh.sums[w];
            a.sums[row * a.parts + part] = PartSum{s, top, 0.f};
        }
    }
    __syncthreads();
    if (tid == 0) {                                              // what the CTA wrote is there before its arrival counts, and what the others wrote is read after theirs
        __threadfence();
        last = atomicAdd(&a.arrived[g], 1) == a.beams * a.parts - 1;
        __threadfence();
        if (last) a.arrived[g] = 0;                              // for the next call
    }
    __syncthreads();
    if (!last) return;
    beam_join<MOST>(a, g, score, ended, *(JoinShared<MOST> *)smem);
}

template <class E, bool VEC, int MOST> void run_select_of(const BeamArgs &a, unsigned grid) {
    static bool set = false;
    if (!set) {
        CUDA_CHECK(cudaFuncSetAttribute(k_beam_select<E, VEC, MOST>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)beam_smem<E, MOST>()));
        set = true;
    }
    LAUNCH_PDL((k_beam_select<E, VEC, MOST>), grid, BM_THREADS, (beam_smem<E, MOST>()), a);
}
template <class E, bool VEC> void run_select(const BeamArgs &a, unsigned grid) {
    if (a.n <= BM_FEW) run_select_of<E, VEC, BM_FEW>(a, grid);
    else run_select_of<E, VEC, NCMB_MAX_BEAMS>(a, grid);
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
    // a group's results are there before other groups have read what they need; in place each group has its own words
    const size_t gb = (size_t)groups * n_out * 4, ib = (size_t)rows * 4, xb = ((size_t)(rows - 1) * ldl + V) * es;
    const void *in[2] = {scores, done}, *out[4] = {scores_out, done_out, parents, tokens};
    for (int i = 0; i < 4; i++) {
        for (int j = 0; j < 2; j++)
            if (paged_overlap(out[i], gb, in[j], ib) && !(i == j && out[i] == in[j] && n_out == beams)) return cache_refuse(who, "results in the memory of scores or done, other than in place with as many as there are beams");
        for (int j = 0; j < i; j++) if (paged_overlap(out[i], gb, out[j], gb)) return cache_refuse(who, "two results in the same memory");
        if (paged_overlap(out[i], gb, logits, xb)) return cache_refuse(who, "results in the memory of the logits");
    }
    if (cache_device(who)) return -1;
    BeamArgs a = {};
    a.x = (const char *)logits; a.ld = ldl * es; a.groups = groups; a.beams = beams; a.V = V; a.n = n_out;
    a.tiles = (int)cdiv(V, BM_TILE);
    a.scores = scores; a.done = done; a.eos = eos; a.scores_out = scores_out; a.parents = parents; a.tokens = tokens; a.done_out = done_out;
    // Parts of a row: as many as fill one to BM_ROUNDS rounds of the CTAs that fit the GPU, whichever takes least where a CTA's start and end take as long as
    // BM_START tiles (256 rows of 151936 in fp32, 1 / 2 / 3 / 5 parts: 37 / 42 / 46 / 53 us, in bf16 33 / 39 / 43 / 50; 32 rows, 4 / 5 / 9 parts: 15.0 / 16.3 / 15.0; 1 and 9 are taken).
    const int64_t resident = BM_CTAS * ctx().sm_count, most = std::max<int64_t>(1, std::min<int64_t>(a.tiles, 65536 / ((int64_t)beams * n_out)));
    int64_t best = INT64_MAX;
    for (int r = 1; r <= BM_ROUNDS; r++) {
        const int64_t p = std::max<int64_t>(1, std::min(most, r * resident / rows)), cost = cdiv(rows * p, resident) * (cdiv(a.tiles, p) + BM_START);
        if (cost < best) { best = cost; a.parts = (int)p; }
    }
    a.slots = (int64_t)beams * a.parts * 2 * n_out <= BM_THREADS * BM_JOIN ? 2 * n_out : n_out;
    const size_t kb = (size_t)rows * a.parts * a.slots * 8, sb = (size_t)rows * a.parts * sizeof(PartSum);
    char *scratch = (char *)cache_scratch(who, sb + kb);
    if (!scratch) return -1;
    a.sums = (PartSum *)scratch;
    a.keys = (unsigned long long *)(scratch + sb);
    if (!(a.arrived = (int *)cache_scratch(who, (size_t)groups * 4, SCRATCH_DONE))) return -1;
    ProfScope prof(NCMB_K_SAMPLE, 4.0 * rows * V, (double)rows * V * es);
    const bool vec = (uintptr_t)logits % 16 == 0 && a.ld % 16 == 0;
    const unsigned grid = (unsigned)(rows * a.parts);
    if (type == NCMB_F32) { if (vec) run_select<float, true>(a, grid); else run_select<float, false>(a, grid); }
    else if (vec) run_select<__nv_bfloat16, true>(a, grid);
    else run_select<__nv_bfloat16, false>(a, grid);
    return 0;
}
