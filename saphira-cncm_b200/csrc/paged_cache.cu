// Paged caches: new tokens' keys and values into their rows' pages with the rotation on the way (ncmb_paged_append), and rows that go on as
// other rows of their group (ncmb_paged_reorder); include/ncm_b200.h.
#include "paged.cuh"
#include "rope.cuh"

#include <algorithm>

namespace ncmb {

int paged_check(const char *who, const NcmbPaged *c, PagedDev &d) {
    if (!c) return cache_refuse(who, "no cache");
    if (c->type != NCMB_F32 && c->type != NCMB_BF16) return cache_refuse(who, "cache type %d", c->type);
    if (c->rows < 0 || c->n_kv < 1 || c->n_pages < 1 || c->max_pages < 1) return cache_refuse(who, "%d rows, %d kv heads, %d pages, %d a row", c->rows, c->n_kv, c->n_pages, c->max_pages);
    if (c->rows > 65535 || c->n_kv > 65535) return cache_refuse(who, "%d rows, %d kv heads: at most 65535", c->rows, c->n_kv);
    if (c->hd < 8 || c->hd > 128 || c->hd % 8) return cache_refuse(who, "head dim %d: a multiple of 8 up to 128", c->hd);
    if (c->page < 8 || c->page > 1024 || (c->page & (c->page - 1))) return cache_refuse(who, "pages of %d: a power of two, 8 to 1024", c->page);
    if ((int64_t)c->max_pages * c->page > 0x7fffff00) return cache_refuse(who, "%d pages of %d tokens a row", c->max_pages, c->page);
    if (c->table_stride < (c->rows > 1 ? c->max_pages : 0)) return cache_refuse(who, "rows of the table of %lld entries, %d used", (long long)c->table_stride, c->max_pages);
    const int64_t es = c->type == NCMB_BF16 ? 2 : 4;
    if (!c->k || !c->v || (c->rows && (!c->len || !c->table))) return cache_refuse(who, "a null pointer in the cache");
    if (((uintptr_t)c->k | (uintptr_t)c->v) % 16) return cache_refuse(who, "keys and values have to be 16-byte aligned");
    if (((uintptr_t)c->len | (uintptr_t)c->table) % 4) return cache_refuse(who, "lengths and tables have to be 4-byte aligned");
    if (c->page_stride < 0 || c->head_stride < 0 || c->token_stride < 0 || (c->page_stride * es) % 16 || (c->head_stride * es) % 16 || (c->token_stride * es) % 16)
        return cache_refuse(who, "strides have to be positive multiples of 16 bytes");
    if (c->token_stride < c->hd || (c->n_kv > 1 && c->head_stride < c->hd) || (c->n_pages > 1 && c->page_stride < c->hd)) return cache_refuse(who, "a stride is smaller than the head dim");
    int lg = 3;
    while (1 << lg < c->page) lg++;
    d = PagedDev{(char *)c->k, (char *)c->v, c->page_stride * es, c->head_stride * es, c->token_stride * es, c->rows, c->n_kv, c->hd, lg, c->n_pages, c->max_pages, (int)es,
                 c->table, c->table_stride, c->len};
    return 0;
}

namespace {

// ---- new tokens ----
constexpr int PA_THREADS = 256, PA_TOKENS = 32, PA_BATCH = 3, PA_ROWS = 1024;

struct AppendArgs {
    PagedDev c;
    const char *q, *k, *v; char *q_out;
    int64_t ldq, ldqo, ldk, ldv;     // bytes
    int H;                           // 0: no queries
    const int *start, *pos;
    int tokens, T;                   // T: of every row, where start is null
    int per;                         // tokens a CTA
    RopeShare share;
};

// the row that token i belongs to, -1 for none: the last b with start[b] <= i. s: start, in shared or global memory
__device__ int append_row(const int *s, int rows, int i) {
    if (i < s[0] || i >= s[rows]) return -1;
    int lo = 0, hi = rows;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s[mid] <= i) lo = mid; else hi = mid;
    }
    return lo;
}

// A CTA has `per` tokens: where each goes and the cosines and sines of its angles once, in shared memory, then all items of its heads -- queries, keys,
// values -- PA_BATCH of a thread on their way at a time, the first of them while places and angles are found. QE: type of the activations, KE: of the
// cache. ROPE: 0 none, 1 halves, 2 pairs. Bound by latency of its dependent steps -- starts, length, table, angles -- and DRAM: 16 rows of up to 2001 tokens, 32 over
// 8 x 128 in bf16, 375 MB: 69 us (5.4 TB/s). By instructions where halves are no whole vectors, V < 16 bytes: dims 50 199 us, dims 72 87.
template <class QE, class KE, int V, int ROPE>
__global__ void __launch_bounds__(PA_THREADS, V * sizeof(QE) == 16 ? 4 : 6) k_paged_append(const __grid_constant__ NcmbRope r, const __grid_constant__ AppendArgs a) {
    extern __shared__ __align__(16) float2 cs[];         // [per][rope_row(dims)]
    __shared__ int64_t slot[PA_TOKENS];          // bytes from the pool's start; -1: not stored, -2: nobody's
    __shared__ int place[PA_TOKENS];
    __shared__ int starts[PA_ROWS + 1];
    const int tid = threadIdx.x, cs_row = ROPE ? rope_row(r.dims) : 0;
    const int n0 = blockIdx.x * a.per, here = min(a.per, a.tokens - n0);
    const bool near = a.c.rows <= PA_ROWS;
    RopeWalk at(tid, a.share);
    const RopeItem it = rope_item<V, ROPE != 1>(at.u, a.share.items, ROPE ? r.dims : 0, a.c.hd);
    pdl_wait();
    pdl_launch_dependents();
    RopeVec<QE, V> p[PA_BATCH], q[PA_BATCH];
    RopeWalk from = at;
    auto load = [&](int x) {
        if (at.tok < here) {
            const int64_t n = n0 + at.tok;
            const int kvh = at.h - a.H;
            const char *row = kvh < 0 ? a.q + n * a.ldq : kvh < a.c.nkv ? a.k + n * a.ldk : a.v + n * a.ldv;
            const QE *f = (const QE *)row + (kvh < 0 ? at.h : kvh < a.c.nkv ? kvh : kvh - a.c.nkv) * a.c.hd;
            p[x] = *(const RopeVec<QE, V> *)(f + it.d0);
            if (it.d1 >= 0) q[x] = *(const RopeVec<QE, V> *)(f + it.d1);
        }
        at.next(a.share);
    };
#pragma unroll
    for (int x = 0; x < PA_BATCH; x++) load(x);
    if (a.start && near) for (int i = tid; i <= a.c.rows; i += PA_THREADS) starts[i] = a.start[i];
    __syncthreads();
    if (tid < here) {
        const int n = n0 + tid;
        const int row = a.start ? append_row(near ? starts : a.start, a.c.rows, n) : n / a.T;
        int64_t to = -2;
        int seq = 0;
        const int len = row >= 0 ? a.c.len[row] : -1;
        if (len >= 0) {
            const int64_t s = len + (a.start ? (int64_t)n - (near ? starts : a.start)[row] : n % a.T);
            seq = (int)min(s, (int64_t)INT_MAX);
            const int page = s < (int64_t)a.c.max_pages << a.c.page_log ? paged_entry(a.c, row, (int)(s >> a.c.page_log)) : -1;
            to = page < 0 ? -1 : page * a.c.ps + (s & ((1 << a.c.page_log) - 1)) * a.c.ts;
        }
        slot[tid] = to;
        place[tid] = ROPE && a.pos ? a.pos[n] : seq;
    }
    __syncthreads();
    if (ROPE) {
        rope_angles(tid, here, a.share, [&](int t, int i) { cs[t * cs_row + rope_place<V, ROPE == 2>(i, r.dims)] = rope_angle(r, i, place[t], false); });
        __syncthreads();
    }
    while (from.tok < here) {
#pragma unroll
        for (int x = 0; x < PA_BATCH; x++) {
            const int64_t to = from.tok < here ? slot[from.tok] : -2;
            const int kvh = from.h - a.H;
            if (to >= (kvh < 0 ? -1 : 0)) {
                float f[V], g[V];
                rope_unpack<QE, V>(p[x], f);
                if (it.d1 >= 0) rope_unpack<QE, V>(q[x], g);
                if (ROPE && kvh < a.c.nkv) rope_turn<V, ROPE == 2>(it, r.dims, cs + from.tok * cs_row, f, g);
                if (kvh < 0) {
                    QE *y = (QE *)(a.q_out + (n0 + from.tok) * a.ldqo) + from.h * a.c.hd;
                    rope_store<QE, V>(y + it.d0, f);
                    if (it.d1 >= 0) rope_store<QE, V>(y + it.d1, g);
                } else {
                    KE *y = (KE *)((kvh < a.c.nkv ? a.c.k + kvh * a.c.hs : a.c.v + (kvh - a.c.nkv) * a.c.hs) + to);
                    rope_store<KE, V>(y + it.d0, f);
                    if (it.d1 >= 0) rope_store<KE, V>(y + it.d1, g);
                }
            }
            from.next(a.share);
            load(x);
        }
    }
}

template <class QE, class KE, int V> void run_append(const NcmbRope *r, AppendArgs &a) {
    a.share = rope_share(r, rope_items(r, a.c.hd, V), a.H + 2 * a.c.nkv, PA_THREADS);
    // four items a thread (short vectors: more, which share the angles), and CTAs for all SMs (16 rows of up to 2001 tokens, 32 over 8 x 128 in bf16, 4 / 8 / 12 items a thread: 69 / 76 / 77 us)
    const int64_t per_token = (int64_t)(a.H + 2 * a.c.nkv) * a.share.items, rounds = V * sizeof(QE) == 16 ? 4 : 20;
    a.per = (int)std::max<int64_t>(1, std::min<int64_t>({PA_TOKENS, rounds * PA_THREADS / per_token, a.tokens / (4 * ctx().sm_count)}));
    const size_t smem = r ? (size_t)a.per * rope_row(r->dims) * sizeof(float2) : 0;
    const unsigned grid = (unsigned)cdiv(a.tokens, a.per);
    static const NcmbRope none = {};
    if (!r) { if constexpr (V * sizeof(QE) == 16) LAUNCH_PDL((k_paged_append<QE, KE, V, 0>), grid, PA_THREADS, smem, none, a); }
    else if (r->layout == NCMB_ROPE_HALVES) LAUNCH_PDL((k_paged_append<QE, KE, V, 1>), grid, PA_THREADS, smem, *r, a);
    else if constexpr (V * sizeof(QE) == 16) LAUNCH_PDL((k_paged_append<QE, KE, V, 2>), grid, PA_THREADS, smem, *r, a);
}
template <class QE, class KE> void run_append(const NcmbRope *r, AppendArgs &a) {
    switch (rope_vec(r, sizeof(QE))) {
        case 8: if constexpr (sizeof(QE) == 2) run_append<QE, KE, 8>(r, a); break;
        case 4: run_append<QE, KE, 4>(r, a); break;
        case 2: run_append<QE, KE, 2>(r, a); break;
        default: run_append<QE, KE, 1>(r, a); break;
    }
}

// ---- rows that go on as others ----
constexpr int PR_THREADS = NCMB_MAX_GROUP, PR_WARPS = PR_THREADS / 32, PR_BATCH = 8, PR_CTAS = 8;

struct ReorderArgs {
    PagedDev c;
    int group, n_layer;
    int64_t ls;                      // bytes from layer to layer
    const int *parents;
    int *table2, *len2, *refs;
};

// CTAs (x, group): each finds out whose row every row of the group continues and whose own pages it takes; the rows' tables are dealt to the
// CTAs, and of each begun page that is copied every CTA has a share.
// Bound by the copies: 16 groups of 8 beams, 32 layers of 8 x 128 in bf16, pages of 64: 73 us for 467 MB (6.4 TB/s).
__global__ void __launch_bounds__(PR_THREADS) k_paged_reorder(const __grid_constant__ ReorderArgs a) {
    __shared__ int heir[NCMB_MAX_GROUP];         // lowest row that continues a row; group: none
    __shared__ int taken[NCMB_MAX_GROUP];        // rows whose own pages are free, ascending
    __shared__ int owner[NCMB_MAX_GROUP], par[NCMB_MAX_GROUP], len[NCMB_MAX_GROUP];
    __shared__ int copies[NCMB_MAX_GROUP], cnt[3][PR_WARPS];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g0 = blockIdx.y * a.group, K = a.group;
    pdl_wait();
    pdl_launch_dependents();
    heir[tid] = K;
    int p = -1;
    if (tid < K) {
        len[tid] = a.c.len[g0 + tid];
        p = a.parents[g0 + tid];
        if ((unsigned)p >= (unsigned)K) p = -1;
        par[tid] = p;
    }
    __syncthreads();
    if (p >= 0) atomicMin(&heir[p], tid);
    __syncthreads();
    // the i-th row that takes free pages takes those of the i-th row without an heir
    const bool takes = tid < K && !(p >= 0 && heir[p] == tid), free_ = tid < K && heir[tid] == K;
    const uint32_t tm = __ballot_sync(0xffffffffu, takes), fm = __ballot_sync(0xffffffffu, free_), cm = __ballot_sync(0xffffffffu, takes && p >= 0), lt = (1u << lane) - 1;
    if (lane == 0) { cnt[0][warp] = __popc(tm); cnt[1][warp] = __popc(fm); cnt[2][warp] = __popc(cm); }
    __syncthreads();
    int ti = __popc(tm & lt), fi = __popc(fm & lt), ci = __popc(cm & lt), n_copies = 0;
    for (int w = 0; w < PR_WARPS; w++) {
        if (w < warp) { ti += cnt[0][w]; fi += cnt[1][w]; ci += cnt[2][w]; }
        n_copies += cnt[2][w];
    }
    if (free_) taken[fi] = tid;
    if (takes && p >= 0) copies[ci] = tid;       // the rows that get a begun page, in the same order for all CTAs
    __syncthreads();
    if (tid < K) owner[tid] = takes ? taken[ti] : p;
    __syncthreads();
    const int64_t cap = (int64_t)a.c.max_pages << a.c.page_log;
    auto used = [&](int i) { return (int)max((int64_t)0, min((int64_t)len[i], cap)); };
    for (int j = blockIdx.x; j < K; j += gridDim.x) {
        const int pj = par[j], own = owner[j], n = pj >= 0 ? used(pj) : 0, tp = n >> a.c.page_log, to = used(own) >> a.c.page_log;
        int *t2 = a.table2 + (int64_t)(g0 + j) * a.c.table_stride;
        for (int i = tid; i < a.c.max_pages; i += PR_THREADS) {
            const int e = i < tp ? paged_entry(a.c, g0 + pj, i) : i - tp + to < a.c.max_pages ? paged_entry(a.c, g0 + own, i - tp + to) : -1;
            t2[i] = e;
            if (a.refs) {
                const int before = paged_entry(a.c, g0 + j, i);
                if (before != e) {
                    if (before >= 0) atomicAdd(&a.refs[before], -1);
                    if (e >= 0) atomicAdd(&a.refs[e], 1);
                }
            }
        }
        if (tid == 0) a.len2[g0 + j] = pj >= 0 ? len[pj] : -1;
    }
    // a warp copies the begun page's keys, or values, of a row, head and layer: 16 bytes a lane, PR_BATCH of them on their way
    const uint32_t units = a.c.hd * a.c.es / 16, lg = units & (units - 1) ? 0 : __ffs(units) - 1;      // of 16 bytes in a token's keys
    const int runs = a.n_layer * 2 * a.c.nkv;
    for (int64_t x = blockIdx.x * PR_WARPS + warp; x < (int64_t)n_copies * runs; x += gridDim.x * PR_WARPS) {
        const int c = (int)(x / runs), run = (int)(x - (int64_t)c * runs), side = run / a.c.nkv, h = run - side * a.c.nkv;
        const int j = copies[c], pj = par[j], own = owner[j], n = used(pj);
        const uint32_t total = (n & ((1 << a.c.page_log) - 1)) * units;
        if (total == 0) continue;
        const int from = paged_entry(a.c, g0 + pj, n >> a.c.page_log), dst = paged_entry(a.c, g0 + own, used(own) >> a.c.page_log);
        if (from < 0 || dst < 0) continue;
        char *base = ((side & 1) ? a.c.v : a.c.k) + (side >> 1) * a.ls + h * a.c.hs;
        const char *src = base + from * a.c.ps;
        char *to_page = base + dst * a.c.ps;
        for (uint32_t i0 = lane; i0 < total; i0 += 32 * PR_BATCH) {
            int4 v[PR_BATCH];
#pragma unroll
            for (int k = 0; k < PR_BATCH; k++) {
                const uint32_t i = i0 + 32 * k, t = units == 1 || lg ? i >> lg : i / units;
                if (i < total) v[k] = *(const int4 *)(src + t * a.c.ts + (i - t * units) * 16);
            }
#pragma unroll
            for (int k = 0; k < PR_BATCH; k++) {
                const uint32_t i = i0 + 32 * k, t = units == 1 || lg ? i >> lg : i / units;
                if (i < total) *(int4 *)(to_page + t * a.c.ts + (i - t * units) * 16) = v[k];
            }
        }
    }
}

} // namespace
} // namespace ncmb

using namespace ncmb;

extern "C" int ncmb_paged_append(const NcmbPaged *c, const NcmbRope *r, const void *q, int64_t ldq, void *q_out, int64_t ldqo, int n_head,
                                 const void *k, int64_t ldk, const void *v, int64_t ldv, int act_type, int n_tokens, const int *start, const int *pos) {
    const char *who = "ncmb_paged_append";
    AppendArgs a = {};
    if (paged_check(who, c, a.c)) return -1;
    if (act_type != NCMB_F32 && !(act_type == NCMB_BF16 && c->type == NCMB_BF16)) return cache_refuse(who, "activations of type %d with a cache of type %d", act_type, c->type);
    if (r && rope_check(who, r, c->hd)) return -1;
    const int64_t es = act_type == NCMB_BF16 ? 2 : 4, kv = (int64_t)c->n_kv * c->hd, qw = (int64_t)n_head * c->hd;
    if (n_tokens < 0 || (!start && (c->rows ? n_tokens % c->rows : n_tokens))) return cache_refuse(who, "%d tokens of %d rows", n_tokens, c->rows);
    if (((uintptr_t)start | (uintptr_t)pos) % 4) return cache_refuse(who, "starts and positions have to be 4-byte aligned");
    if (n_tokens == 0 || c->rows == 0) return 0;
    if (!k || !v || ((uintptr_t)k | (uintptr_t)v) % 16 || (ldk * es) % 16 || (ldv * es) % 16 || ldk < kv || ldv < kv)
        return cache_refuse(who, "k and v have to be 16-byte aligned, with rows of n_kv * hd at multiples of 16 bytes");
    if (q && (n_head < 1 || !q_out || ((uintptr_t)q | (uintptr_t)q_out) % 16 || (ldq * es) % 16 || (ldqo * es) % 16 || ldq < qw || ldqo < qw))
        return cache_refuse(who, "q and q_out have to be 16-byte aligned, with rows of n_head * hd at multiples of 16 bytes");
    if (q && q == q_out && ldq != ldqo) return cache_refuse(who, "queries in place with another stride");
    if (kv + (q ? qw : 0) > 1 << 24) return cache_refuse(who, "%d heads over %d", n_head, c->n_kv);
    if (cache_device(who)) return -1;
    a.q = (const char *)q; a.q_out = (char *)q_out; a.k = (const char *)k; a.v = (const char *)v;
    a.ldq = ldq * es; a.ldqo = ldqo * es; a.ldk = ldk * es; a.ldv = ldv * es;
    a.H = q ? n_head : 0; a.start = start; a.pos = pos; a.tokens = n_tokens; a.T = n_tokens / c->rows;
    ProfScope prof(NCMB_K_ELEM, 3.0 * n_tokens * (a.H + c->n_kv) * c->hd, (double)n_tokens * (2.0 * a.H * c->hd * es + 2.0 * kv * (es + a.c.es)));
    if (c->type == NCMB_F32) run_append<float, float>(r, a);
    else if (act_type == NCMB_F32) run_append<float, __nv_bfloat16>(r, a);
    else run_append<__nv_bfloat16, __nv_bfloat16>(r, a);
    return 0;
}

extern "C" int ncmb_paged_reorder(const NcmbPaged *c, int group, const int *parents, int n_layer, int64_t layer_stride, int *table_dst, int *len_dst, int *refs) {
    const char *who = "ncmb_paged_reorder";
    ReorderArgs a = {};
    if (paged_check(who, c, a.c)) return -1;
    if (group < 1 || group > NCMB_MAX_GROUP || c->rows % group) return cache_refuse(who, "groups of %d in %d rows: at most %d, a divisor", group, c->rows, NCMB_MAX_GROUP);
    if (n_layer < 1 || n_layer > 65535 || layer_stride < 0 || (layer_stride * a.c.es) % 16 || (n_layer > 1 && layer_stride < c->hd))
        return cache_refuse(who, "%d layers, %lld elements apart: a multiple of 16 bytes", n_layer, (long long)layer_stride);
    const int64_t runs = (int64_t)n_layer * 2 * c->n_kv;
    if (runs > 1 << 30) return cache_refuse(who, "%d layers of %d kv heads", n_layer, c->n_kv);
    if (c->rows == 0) return 0;
    if (!parents || !table_dst || !len_dst || ((uintptr_t)parents | (uintptr_t)table_dst | (uintptr_t)len_dst | (uintptr_t)refs) % 4) return cache_refuse(who, "parents, table_dst and len_dst: not null, 4-byte aligned");
    // CTAs read what others may have written to already: nothing that is read is written
    const size_t tb = ((size_t)(c->rows - 1) * c->table_stride + c->max_pages) * 4, lb = (size_t)c->rows * 4;
    const struct { const void *p; size_t bytes; } in[3] = {{c->table, tb}, {c->len, lb}, {parents, lb}}, out[3] = {{table_dst, tb}, {len_dst, lb}, {refs, (size_t)c->n_pages * 4}};
    for (int i = 0; i < 3; i++)
        for (int j = 0; j < 3; j++)
            if (paged_overlap(out[i].p, out[i].bytes, in[j].p, in[j].bytes) || (j != i && paged_overlap(out[i].p, out[i].bytes, out[j].p, out[j].bytes)))
                return cache_refuse(who, "new tables, lengths and counts have to stand in memory of their own");
    if (cache_device(who)) return -1;
    a.group = group; a.n_layer = n_layer; a.ls = layer_stride * a.c.es; a.parents = parents; a.table2 = table_dst; a.len2 = len_dst; a.refs = refs;
    ProfScope prof(NCMB_K_ELEM, 0, (double)c->rows * runs * c->page * c->hd * a.c.es);
    // a run of half of the group a warp, but no more CTAs than keep the GPU busy: each finds the group's parents first
    const int groups = c->rows / group;
    const int64_t most = std::max<int64_t>(1, PR_CTAS * (int64_t)ctx().sm_count / groups);
    LAUNCH_PDL(k_paged_reorder, dim3((unsigned)std::min(most, cdiv(runs * cdiv(group, 2), PR_WARPS)), groups), PR_THREADS, 0, a);
    return 0;
}
