// A cache held to a budget of tokens by the attention each has received (ncmb_cache_evict, include/ncm_b200.h).
//
// Per (row, kv head) of n tokens, n2 = min(n, budget) are kept: key = the weight as an ordered integer, the min(recent, budget)
// latest tokens above all; the n2-th largest key by three counting passes; of the tokens that tie with it those in the
// lower slots. Kept tokens below slot n2 stay where they are and the others take the freed slots in order, so a step that
// is one token over budget moves one token, and in place no source is a target.
//
// Bound by latency -- barriers and dependent reads of the selection, 22 us for 16 x 8 heads of up to 8192 slots -- and then by the
// moves, a kernel of its own where many tokens move: 28 us for 134 MB (4.8 TB/s).
#include "cache.cuh"

#include <type_traits>

namespace ncmb {
namespace {

namespace cg = cooperative_groups;

constexpr int EV_THREADS = 512, EV_WARPS = EV_THREADS / 32, EV_MAXC = 8;
constexpr int EV_KEYS = 24576;       // keys a CTA holds in shared memory; beyond, they are read again
constexpr int EV_FEW = 8;
constexpr int EV_MOST = 393216;      // slots of a row: a bit for each and EV_KEYS keys fit one CTA

struct EvictArgs {
    CacheDev c;
    char *k2, *v2;
    int64_t rs2, hs2, ts2;
    int cap2, inplace, budget, recent, es, kcap;
    const float *w; float *w2;
    const int *pos; int *pos2;
    const int *known, *seen;
    int *len2;
    int *from, *to;                  // scratch, [rows][nkv][min(budget, capacity)] each
    int *pairs;                      // scratch, [rows][nkv]: how many of them
    int room;
    int move_here;                   // few tokens move: the kernel that picks moves them too
};

// CL: a cluster of CTAs a (row, kv head), each with a part of the slots; else one CTA.
template <bool CL>
__global__ void __launch_bounds__(EV_THREADS) k_cache_evict(EvictArgs a) {
    extern __shared__ uint32_t dyn[];
    __shared__ SelShared sel;
    __shared__ int maxpos, wcount[4][EV_WARPS];
    __shared__ int share[4];         // ties, freed slots, kept tokens from beyond, kept in place: of this CTA
    cg::cluster_group cl = cg::this_cluster();
    const int rank = CL ? (int)cl.block_rank() : 0, nc = CL ? (int)cl.num_blocks() : 1;
    auto sync = [&] { if constexpr (CL) cl.sync(); else __syncthreads(); };
    const int kvh = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint32_t *keys = dyn, *kept = dyn + a.kcap;          // keys, then one bit a slot
    pdl_wait();
    pdl_launch_dependents();
    const int n = cache_len(a.c, b, 0), n2 = min(n, a.budget);
    const int64_t u = (int64_t)b * a.c.nkv + kvh;
    const int seen = a.seen[b], known = a.known ? max(0, min(a.known[b], n)) : 0;
    const float *w = a.w + u * a.c.cap;
    const int *pos = a.pos + u * a.c.cap;
    if (rank == 0 && kvh == 0 && tid == 0) a.len2[b] = n2;
    if (n == 0) {
        if (rank == 0 && tid == 0) a.pairs[u] = 0;
        return;
    }
    // slots [lo, hi) are this CTA's; a warp's part of them is a whole number of 32
    const int per_warp = ((n + nc * EV_WARPS - 1) / (nc * EV_WARPS) + 31) & ~31;
    const int per = per_warp * EV_WARPS, lo = min(n, rank * per), hi = min(n, lo + per);
    auto place = [&](int s) { return s < known ? pos[s] : seen - n + s; };
    // the latest place in the text: of the tokens since the last eviction it is seen - 1
    int last = known < n ? seen - 1 : INT_MIN;
    auto latest = [&](int s) { return (int64_t)place(s) > (int64_t)last - a.recent; };
    if (known == 0) {
        for (int s = lo + tid; s < min(hi, lo + a.kcap); s += EV_THREADS) keys[s - lo] = latest(s) ? 0xffffffffu : float_key(w[s]);
    } else {
        if (tid == 0) maxpos = INT_MIN;
        __syncthreads();
        for (int s = lo + tid; s < min(hi, lo + a.kcap); s += EV_THREADS) keys[s - lo] = float_key(w[s]);
        for (int s = lo + tid; s < min(hi, known); s += EV_THREADS) last = max(last, pos[s]);
        last = __reduce_max_sync(0xffffffffu, last);
        if (lane == 0) atomicMax(&maxpos, last);
        sync();
        if constexpr (CL) { for (int r = 0; r < nc; r++) last = max(last, *cl.map_shared_rank(&maxpos, r)); }
        else last = maxpos;
#pragma unroll 1
        for (int s = lo + tid; s < min(hi, lo + a.kcap); s += EV_THREADS) if (latest(s)) keys[s - lo] = 0xffffffffu;
    }
    __syncthreads();
    const char *k = a.c.k + b * a.c.rs + kvh * a.c.hs, *v = a.c.v + b * a.c.rs + kvh * a.c.hs;
    char *k2 = a.k2 + b * a.rs2 + kvh * a.hs2, *v2 = a.v2 + b * a.rs2 + kvh * a.hs2;
    const int units = a.c.hd * a.es / 16;                // of 16 bytes in a token's keys
    auto move = [&](int64_t f, int64_t t) {              // a warp
        if (lane < units) {
            const int4 kx = *(const int4 *)(k + f * a.c.ts + lane * 16), vx = *(const int4 *)(v + f * a.c.ts + lane * 16);
            *(int4 *)(k2 + t * a.ts2 + lane * 16) = kx;
            *(int4 *)(v2 + t * a.ts2 + lane * 16) = vx;
        }
    };
    if (!CL && a.inplace && n - n2 <= EV_FEW && n <= a.kcap) {
        // A few tokens over budget, as after a decode step: the lowest keys one after another (of equal ones the highest slot goes)
        // instead of a selection among all. One over 2048, 64 rows: 4.3 us a call, by selection 9.6.
        __shared__ unsigned long long low[2];
        __shared__ int gone[EV_FEW], from[EV_FEW], to[EV_FEW], moves;
#pragma unroll 1
        for (int d = 0; d < n - n2; d++) {
            if (tid == 0) low[d & 1] = ~0ull;
            __syncthreads();
            uint32_t best = 0xffffffffu, at = 0;         // smallest key, then largest slot
            bool any = false;
#pragma unroll 4
            for (int s = tid; s < n; s += EV_THREADS) {
                bool out = false;
                for (int x = 0; x < d; x++) out |= gone[x] == s;
                if (!out && (!any || keys[s] <= best)) { best = keys[s]; at = s; any = true; }
            }
            const uint32_t wmin = __reduce_min_sync(0xffffffffu, best);
            const uint32_t wat = __reduce_max_sync(0xffffffffu, any && best == wmin ? at + 1 : 0u);      // 0: no slot in this warp
            if (lane == 0 && wat) atomicMin(&low[d & 1], (unsigned long long)wmin << 32 | (0xffffffffu - wat));
            __syncthreads();
            if (tid == 0) gone[d] = (int)(0xffffffffu - (uint32_t)low[d & 1]) - 1;
            __syncthreads();
        }
        if (tid == 0) {
            int m = 0;
            for (int s = n2; s < n; s++) {               // kept ones from beyond, ascending
                bool out = false;
                for (int x = 0; x < n - n2; x++) out |= gone[x] == s;
                if (!out) from[m++] = s;
            }
            for (int i = 0, last = -1; i < m; i++) {     // freed slots, ascending
                int next = n2;
                for (int x = 0; x < n - n2; x++) if (gone[x] > last && gone[x] < next) next = gone[x];
                to[i] = last = next;
            }
            moves = m;
            a.pairs[u] = 0;                              // nothing is left for k_cache_move
        }
        __syncthreads();
        for (int s = known + tid; s < n2; s += EV_THREADS) a.pos2[u * a.cap2 + s] = seen - n + s;
        __syncthreads();                                 // a freed slot's place is written last
        for (int i = warp; i < moves; i += EV_WARPS) {
            if (lane == 0) { a.w2[u * a.cap2 + to[i]] = w[from[i]]; a.pos2[u * a.cap2 + to[i]] = place(from[i]); }
            move(from[i], to[i]);
        }
        return;
    }
    auto key = [&](int i) { return i < a.kcap ? keys[i] : latest(lo + i) ? 0xffffffffu : float_key(w[lo + i]); };
    uint32_t bound = 0, ties = 0xffffffffu;              // all are kept where there is room for all
    if (n2 < n) bound = select_kth<EV_THREADS, CL>(sel, hi - lo, (uint32_t)n2, ties, key);

    // how many of something (of N things) the slots before this warp's hold, given its own counts; total: all CTAs'
    const int w0 = lo + warp * per_warp, w1 = min(hi, w0 + per_warp);
    auto before = [&](auto first, int *mine, int *total) {
        constexpr int N = decltype(first)::value == 0 ? 1 : 3, AT = decltype(first)::value;
#pragma unroll
        for (int i = 0; i < N; i++) if (lane == 0) wcount[AT + i][warp] = mine[i];
        __syncthreads();
        int v[N];
#pragma unroll
        for (int i = 0; i < N; i++) {
            v[i] = lane < EV_WARPS ? wcount[AT + i][lane] : 0;
            mine[i] = __reduce_add_sync(0xffffffffu, lane < warp ? v[i] : 0);
            total[i] = __reduce_add_sync(0xffffffffu, v[i]);
        }
        if constexpr (CL) {
#pragma unroll
            for (int i = 0; i < N; i++) if (tid == 0) share[AT + i] = total[i];
            cl.sync();
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int o = lane < nc ? *cl.map_shared_rank(&share[AT + i], lane) : 0;
                mine[i] += __reduce_add_sync(0xffffffffu, lane < rank ? o : 0);
                total[i] = __reduce_add_sync(0xffffffffu, o);
            }
        }
    };
    int all;
    uint32_t tied = 0;                                   // ties before, of which the lower ones are kept
    if (ties != 0xffffffffu) {
        int mine = 0;
#pragma unroll 1
        for (int s = w0; s < w1; s += 32) mine += __popc(__ballot_sync(0xffffffffu, s + lane < w1 && key(s + lane - lo) == bound));
        before(std::integral_constant<int, 0>(), &mine, &all);
        tied = (uint32_t)mine;
    }
    int freed = 0, beyond = 0, stay = 0;
#pragma unroll 1
    for (int s = w0; s < w1; s += 32) {
        const bool in = s + lane < w1;
        const uint32_t x = in ? key(s + lane - lo) : 0;
        const uint32_t tm = __ballot_sync(0xffffffffu, in && x == bound);
        const bool keep = in && (x > bound || (x == bound && tied + (uint32_t)__popc(tm & ((1u << lane) - 1)) < ties));
        tied += (uint32_t)__popc(tm);
        const uint32_t km = __ballot_sync(0xffffffffu, keep);
        const uint32_t below = n2 - s >= 32 ? 0xffffffffu : n2 > s ? (1u << (n2 - s)) - 1 : 0u;      // slots below n2
        if (lane == 0) kept[(s - lo) >> 5] = km;
        freed += __popc(~km & below);
        beyond += __popc(km & ~below);
        stay += __popc(km & below);
    }
    int count[3] = {freed, beyond, stay}, totals[3];
    before(std::integral_constant<int, 1>(), count, totals);
    const int moves = totals[0];
    freed = count[0]; beyond = count[1]; stay = moves + count[2];
    // pairs (from, to): moves, then -- to another cache -- the tokens that keep their slot
    int *from = a.from + u * a.room, *to = a.to + u * a.room;
    __syncwarp();
#pragma unroll 1
    for (int s = w0; s < w1; s += 32) {
        const uint32_t km = kept[(s - lo) >> 5], lt = (1u << lane) - 1, me = 1u << lane;
        const uint32_t below = n2 - s >= 32 ? 0xffffffffu : n2 > s ? (1u << (n2 - s)) - 1 : 0u;
        if (~km & below & me) to[freed + __popc(~km & below & lt)] = s + lane;
        if (km & ~below & me) from[beyond + __popc(km & ~below & lt)] = s + lane;
        if (km & below & me) {
            if (!a.inplace) {
                const int i = stay + __popc(km & below & lt);
                from[i] = to[i] = s + lane;
            } else if (s + lane >= known) a.pos2[u * a.cap2 + s + lane] = seen - n + s + lane;
        }
        freed += __popc(~km & below);
        beyond += __popc(km & ~below);
        stay += __popc(km & below);
    }
    sync();                                              // also: no key is read from w / pos any more
    const int pairs = a.inplace ? moves : n2;
    for (int i = rank * EV_THREADS + tid; i < pairs; i += nc * EV_THREADS) {
        const int f = from[i], t = to[i];
        a.w2[u * a.cap2 + t] = w[f];
        a.pos2[u * a.cap2 + t] = place(f);
    }
    if (rank == 0 && tid == 0) a.pairs[u] = pairs;
    if (!a.move_here) return;
    for (int p = rank * EV_WARPS + warp; p < pairs; p += nc * EV_WARPS) move(from[p], to[p]);
}

// The tokens that move, over the whole GPU. A thread has 16 bytes of a token's keys or values, of EV_AHEAD tokens.
constexpr int EV_MTHREADS = 256, EV_AHEAD = 4;       // 8 ahead: 38 us where 4 take 28
__global__ void __launch_bounds__(EV_MTHREADS) k_cache_move(EvictArgs a, int ul) {
    const int kvh = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
    const int x = tid & ((1 << ul) - 1), is_v = (tid >> ul) & 1, tok = tid >> (ul + 1), tpc = EV_MTHREADS >> (ul + 1);
    const int64_t u = (int64_t)b * a.c.nkv + kvh;
    pdl_wait();
    pdl_launch_dependents();
    const int pairs = a.pairs[u], p0 = (int)blockIdx.x * tpc * EV_AHEAD + tok;
    if (x * 16 >= a.c.hd * a.es) return;
    const int *from = a.from + u * a.room, *to = a.to + u * a.room;
    const char *src = (is_v ? a.c.v : a.c.k) + b * a.c.rs + kvh * a.c.hs + x * 16;
    char *dst = (is_v ? a.v2 : a.k2) + b * a.rs2 + kvh * a.hs2 + x * 16;
    int4 r[EV_AHEAD];
    int64_t t[EV_AHEAD];
#pragma unroll
    for (int i = 0; i < EV_AHEAD; i++) {
        const int p = p0 + i * tpc;
        t[i] = p < pairs ? to[p] : -1;
        if (t[i] >= 0) r[i] = *(const int4 *)(src + from[p] * a.c.ts);
    }
#pragma unroll
    for (int i = 0; i < EV_AHEAD; i++) if (t[i] >= 0) *(int4 *)(dst + t[i] * a.ts2) = r[i];
}

bool overlaps(const CacheDev &a, const CacheDev &b, int es) {
    auto reach = [&](const CacheDev &c) { return (int64_t)(c.rows - 1) * c.rs + (int64_t)(c.nkv - 1) * c.hs + (int64_t)(c.cap - 1) * c.ts + (int64_t)c.hd * es; };
    const int64_t ra = reach(a), rb = reach(b);
    for (const char *x : {a.k, a.v})
        for (const char *y : {b.k, b.v})
            if (x < y + rb && y < x + ra) return true;
    return false;
}

} // namespace
} // namespace ncmb

using namespace ncmb;

extern "C" int ncmb_cache_evict(const NcmbCache *src, const NcmbCache *dst, const float *weights, float *weights_dst, const int *pos,
                                int *pos_dst, const int *known, const int *seen, int budget, int recent, int max_len, int *len_dst) {
    const char *who = "ncmb_cache_evict";
    EvictArgs a;
    CacheDev d;
    if (cache_check(who, src, a.c) || cache_check(who, dst, d)) return -1;
    if (src->type != dst->type || src->rows != dst->rows || src->n_kv != dst->n_kv || src->hd != dst->hd) return cache_refuse(who, "the two caches differ in type, rows, kv heads or head dim");
    if (budget < 1 || recent < 0) return cache_refuse(who, "budget %d, recent %d", budget, recent);
    if (src->capacity > EV_MOST) return cache_refuse(who, "capacity %d: at most %d slots", src->capacity, EV_MOST);
    if (!weights || !weights_dst || !pos || !pos_dst || !seen || !len_dst) return cache_refuse(who, "a null pointer");
    if (src->rows == 0) return 0;
    const int64_t rows = src->rows;
    auto with_len_dst = [&](const int *p) { return p < len_dst + rows && len_dst < p + rows; };
    if (with_len_dst(src->len)) return cache_refuse(who, "len_dst has to be another array than the lengths of the cache");
    a.inplace = src->k == dst->k && src->v == dst->v;
    if (a.inplace && (src->capacity != dst->capacity || src->row_stride != dst->row_stride || src->head_stride != dst->head_stride || src->token_stride != dst->token_stride))
        return cache_refuse(who, "one cache with two layouts");
    if (a.inplace && (weights != weights_dst || pos != pos_dst)) return cache_refuse(who, "in place weights and places have to be in place too");
    if (!a.inplace && (weights == weights_dst || pos == pos_dst)) return cache_refuse(who, "another cache needs weights and places of its own");
    a.room = budget < src->capacity ? budget : src->capacity;
    if (dst->capacity < a.room) return cache_refuse(who, "capacity %d for a budget of %d", dst->capacity, budget);
    const int es = cache_elem(src);
    if (!a.inplace && overlaps(a.c, d, es)) return cache_refuse(who, "the two caches overlap");
    ensure_device();
    a.k2 = (char *)dst->k; a.v2 = (char *)dst->v; a.rs2 = d.rs; a.hs2 = d.hs; a.ts2 = d.ts; a.cap2 = d.cap;
    // The latest tokens rank alike, so no more of them than the budget holds may count as such: else the lower slots stay, the oldest.
    a.budget = budget; a.recent = recent < budget ? recent : budget; a.es = es;
    a.w = weights; a.w2 = weights_dst; a.pos = pos; a.pos2 = pos_dst; a.known = known; a.seen = seen; a.len2 = len_dst;
    if (max_len <= 0 || max_len > src->capacity) max_len = src->capacity;
    const int64_t units = (int64_t)src->rows * src->n_kv;
    a.from = (int *)cache_scratch(who, units * a.room * 8 + units * 4 + rows * 8);
    if (!a.from) return -1;
    a.to = a.from + units * a.room;
    a.pairs = a.to + units * a.room;
    // A row's new length is stored by its first CTA when others may not have read `known` or `seen` yet: where these are the array of the
    // lengths -- the last call's len_dst is this one's known -- the kernel reads copies.
    int *copy = a.pairs + units;
    for (const int **x : {&a.known, &a.seen}) {
        if (!*x || !with_len_dst(*x)) continue;
        CUDA_CHECK(cudaMemcpyAsync(copy, *x, rows * 4, cudaMemcpyDeviceToDevice, stream()));
        *x = copy;
        copy += rows;
    }
    // CTAs a (row, head): as many as keep the GPU busy, with 4096 slots each at least
    int nc = 1;
    while (nc < EV_MAXC && units * nc * 2 <= 2 * ctx().sm_count && cdiv(max_len, nc) > 4096) nc *= 2;
    a.move_here = a.inplace && max_len - a.room <= 64;   // that many tokens move at most, by what the host knows
    if (a.inplace && max_len - a.room <= EV_FEW && max_len <= EV_KEYS) nc = 1;       // no selection: one CTA is enough
    // slots of a CTA when the row is as long as the cache can hold: bits for all, keys for as many as shared memory takes
    const int64_t most = cdiv(cdiv(src->capacity, nc * EV_WARPS), 32) * 32 * EV_WARPS, hint = cdiv(cdiv(max_len, nc * EV_WARPS), 32) * 32 * EV_WARPS;
    a.kcap = (int)(hint < EV_KEYS ? hint : EV_KEYS);
    const size_t smem = (size_t)a.kcap * 4 + (size_t)most / 8;
    ProfScope prof(NCMB_K_ATTN, 0, 4.0 * units * max_len);
    auto kernel = nc > 1 ? k_cache_evict<true> : k_cache_evict<false>;
    if (smem > 20000) CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    cache_launch(kernel, dim3(nc, src->n_kv, src->rows), EV_THREADS, smem, nc, a);
    if (!a.move_here) {
        int ul = 0;
        while ((16 << ul) < src->hd * es) ul++;
        const int per = (EV_MTHREADS >> (ul + 1)) * EV_AHEAD;
        cache_launch(k_cache_move, dim3((unsigned)cdiv(a.room, per), src->n_kv, src->rows), EV_MTHREADS, 0, 1, a, ul);
    }
    return 0;
}
