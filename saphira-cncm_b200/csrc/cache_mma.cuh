// Attention of a few query rows to many cached keys on mma.sync tiles: what ncmb_cache_attention, ncmb_block_attention and
// ncmb_paged_attention share. The query rows of a kv head -- its G query heads times the tokens that share the keys --
// are the 16-row tiles; a warp walks chunks of keys with a running maximum and sum a row.
//
// Products in fp32 grade whatever the types: a bf16 key meets an fp32 query as three bf16 terms (24 bits, exact products),
// probabilities meet bf16 values as three terms (two where the result is bf16); fp32 keys and values as TF32 pairs (22 bits),
// three products, or all four where the pairs are stacked. The leading term and the small ones have accumulators of their
// own, and a chunk's P V starts from zero and is added to the running result in fp32 by the multiply-add that rescales it: the
// tensor core truncates its accumulator after each product, which would bias a sum that runs over thousands of keys.
//
// Bound: at 8 rows by reading keys and values (64 rows of up to 16000 tokens, 14 heads over 2 x 64 in bf16: 63 us, 5.4 TB/s with start
// and end, 82 us with the weights); at 16 rows by mma.sync (about 1000 multiply-adds a cycle and SM); for a few thousand keys by
// latency, above all by instruction fetches (12 x 64 over 811 tokens in fp32: 6.6 us).
#pragma once
#include "cache.cuh"

#include <algorithm>

namespace ncmb {

constexpr int CM_LOG(int x) { return x <= 1 ? 0 : 1 + CM_LOG(x / 2); }
constexpr int CM_WARPS = 4, CM_THREADS = CM_WARPS * 32, CM_MAXC = 8;      // CM_MAXC: CTAs of a cluster
// R: query rows of a tile, 16 or 8. A tile of 8 has two terms of its queries (or probabilities) stacked in the 16 rows of the
// tensor-core tile; a lane holds rows lane / 4 and lane / 4 + 8 of a result, so it adds the two terms' products up itself.
template <class KE, class QE, int HDP_, int R_> struct CmCfg {
    static constexpr bool BF = sizeof(KE) == 2;
    static constexpr int HDP = HDP_, M = R_;
    static constexpr bool R8 = R_ == 8;
    static constexpr int NH = R8 ? 1 : 2;                        // rows a lane has
    static constexpr int ROW = HDP * (int)sizeof(KE);            // bytes of a key in shared memory
    static constexpr int UPR = ROW / 16;
    // Two stages of 8 KB a warp and three CTAs an SM. Measured at 64 x 16000 (bf16, 64) / 32 rows of picked blocks (bf16, 128) / 3 x 24
    // (fp32, 64): 87 / 82 / 66 us; four stages of 4 KB 93 / 88 / 71; three of 8 KB in two CTAs 88 / 97 / 68; three of 4 KB in four
    // CTAs 93 / 82 / 88.
    static constexpr int CM_STAGE = 8192, CM_STAGES = 2;
    static constexpr int KC = CM_STAGE / (2 * ROW);              // keys a chunk
    static constexpr int NT = KC / 8;                            // 8-key tiles a chunk
    static constexpr int NQ = !BF ? 2 : sizeof(QE) == 4 ? 3 : 1; // terms of a query
    static constexpr int NP = !BF ? 2 : sizeof(QE) == 4 ? 3 : 2; // terms of a probability
    static constexpr int QT = !BF ? 2 : R8 ? (NQ + 1) / 2 : NQ;  // tiles of 16 rows the queries take; fp32: of M rows
    static constexpr int QROWS = BF ? 16 : M;
    static constexpr int QBYTES = QT * QROWS * HDP * (BF ? 2 : 4);
    static constexpr int RING = CM_WARPS * CM_STAGES * CM_STAGE;
    // CTAs that an SM's 228 KB of shared memory hold: ring and queries, masks or picked blocks, 1 KB that each one costs. Two for 16 rows of
    // 128 dims in fp32, and for picked blocks of 128 dims with fp32 queries or of 64 in fp32 at 16 rows; else three.
    static constexpr int ctas(bool blocks) { return 3 * (RING + QBYTES + (blocks ? 4864 : 2304) + 1024) <= 228 * 1024 ? 3 : 2; }
    static constexpr int SUMS = 2 * M, CTX = M * HDP;            // floats of a partial result: maxima and sums, context
};

struct CmArgs {
    CacheDev c;
    const char *q; char *out;
    int64_t ldq, ldo;                // bytes
    int row0;                        // first row of this launch; items count from it
    int H, G, T, M;                  // M: query rows of a kv head that share keys (T * G, or G)
    int tiles;                       // tiles of CmCfg::M rows they make
    int items;                       // rows, or rows * T where every token has keys of its own
    const int *parents;
    float c2;                        // scale * log2(e)
    float *sums, *ctx;               // partial results: a slot of sums a (CTA + unit), two of contexts a CTA
    int2 *range;                     // first and last CTA of each unit
    int ctas;                        // CTAs of the attention kernel
    const int *err;                  // wide tiles: set when a wait ran out, and then the three above may be what was there before
    int *done;                       // chunks of each unit whose parts are there, zero between calls; null: k_cache_join joins
    float *scores;                   // [row][kv head][M][pitch], or null
    int64_t pitch;
    float *weights;
    // block attention
    int block_log, n_sel;
    const int *picks;
    // paged caches (c.cap: what a row's pages hold)
    const int *table;
    int64_t table_stride, ps;        // entries; bytes from page to page
    int page_log, n_pages, max_pages;
};

__device__ __forceinline__ uint32_t cm_smem(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cm_cp16(uint32_t dst, const void *src, bool ok) {       // 16 bytes, zeros where not ok
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cm_ldm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void cm_ldm4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void cm_mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void cm_mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Two TF32 terms of v, together within 2^-23 of it. BITS: by the integer and fp32 pipes instead of two conversions, which the paged kernels wait for (fp32, 16 heads
// over 4 x 64, 32 rows of up to 8000: 79 -> 69 us); contiguous caches (67 us) keep the conversions, and their results. The leading term is rounded as a
// conversion does, half of its last place added and cut off; the rest is less than 2^12 of v's last places, so a cut after 11 bits loses one of them
// at most, as rounding would. A NaN that the addition carries into the sign leaves a NaN as the rest.
template <bool BITS = false> __device__ __forceinline__ void cm_tf32(float v, uint32_t &hi, uint32_t &lo) {
    if constexpr (BITS) {
        hi = (__float_as_uint(v) + 0x1000u) & 0xffffe000u;
        lo = __float_as_uint(v - __uint_as_float(hi)) & 0xffffe000u;
    } else {
        asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(v));
        asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(lo) : "f"(v - __uint_as_float(hi)));
    }
}
__device__ __forceinline__ float cm_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t cm_pack(float a, float b) {      // two bf16, a in the low half
    const __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
    return *(const uint32_t *)&t;
}
__device__ __forceinline__ float2 cm_unpack(uint32_t u) { return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)); }
__device__ __forceinline__ void cm_put(float *p, float v) { *p = v; }
__device__ __forceinline__ void cm_put(__nv_bfloat16 *p, float v) { *p = __float2bfloat16(v); }

__device__ __forceinline__ bool cm_used(const int *par, int t) { return !par || (par[t] >= -1 && par[t] < t); }

static __device__ __noinline__ unsigned cm_div(unsigned x, unsigned d) { return x / d; }       // one copy of the code

// keys that the queries of an item see
template <bool BLOCKS> __device__ __forceinline__ int cm_keys(const CmArgs &a, int item) {
    if (!BLOCKS) return cache_len(a.c, a.row0 + item, a.T) + a.T;
    const int here = cache_len(a.c, a.row0 + item / a.T, a.T) + item % a.T, cur = here >> a.block_log;
    return ((min(cur + 1, a.n_sel) - 1) << a.block_log) + (here & ((1 << a.block_log) - 1)) + 1;
}

// ---- how the chunks of all units are dealt to CTAs ----
// The units (item, kv head, tile) in order, each with its start and its chunks in order, are one sequence, of which every CTA takes an equal
// run: rows of any lengths keep all SMs busy to the end. A unit is done by one CTA or by consecutive ones. CTA c's maxima and
// sums of unit u go to slot c + u (along the sequence one of the two grows by one at a time); its context, where it has not
// done the whole unit, to slot 2 c + 1 if it began the unit, else to 2 c: a CTA begins at most one that it does not end, its
// last, and continues at most one, its first. So the memory for contexts does not grow with the units.
// (Counts are 32-bit: the host limits the rows of a launch. Nothing here is unrolled: code that runs once is paced by
// instruction fetches, about 150 cycles for 8 instructions.)
// A unit takes places of whole rounds -- a chunk a warp -- and one round more, what its start and end cost, or the CTA that gets the units
// of a short row is the last. All begin and end at whole rounds, so none is cut inside one. Counted by chunks alone, picked blocks of 32 rows
// up to 32768 tokens (one of none) took 80 us for 65, of 6 rows of up to 17705 with 24 new tokens 151 for 37.
constexpr int CM_START = CM_WARPS;
__host__ __device__ constexpr int cm_span(int chunks) { return ((chunks + CM_WARPS - 1) & ~(CM_WARPS - 1)) + CM_START; }
struct CmPlan { int total, per; };
template <bool BLOCKS, int KC> __device__ __forceinline__ int cm_chunks(const CmArgs &a, int item) {           // of all units of an item
    return item < a.items ? cm_span((cm_keys<BLOCKS>(a, item) + KC - 1) / KC) * a.c.nkv * a.tiles : 0;
}
template <bool BLOCKS, int KC> __device__ CmPlan cm_plan(const CmArgs &a, int ctas, int *sh) {
    int t = 0;
#pragma unroll 1
    for (int i = threadIdx.x; i < a.items; i += CM_THREADS) t += cm_chunks<BLOCKS, KC>(a, i);
    t = __reduce_add_sync(0xffffffffu, t);
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = t;
    __syncthreads();
    CmPlan p;
    p.total = sh[0] + sh[1] + sh[2] + sh[3];
    p.per = ((unsigned)(p.total + ctas - 1) / (unsigned)ctas + CM_WARPS - 1) & ~(CM_WARPS - 1);
    return p;
}
// the item that holds place x of the sequence, and where that item begins
template <bool BLOCKS, int KC> __device__ int cm_find(const CmArgs &a, int x, int &start, int *sh) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int before = 0;
#pragma unroll 1
    for (int i0 = 0;; i0 += CM_THREADS) {
        const int i = i0 + threadIdx.x, mine = cm_chunks<BLOCKS, KC>(a, i);
        int inc = mine;
#pragma unroll 1
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += v;
        }
        __syncthreads();
        if (lane == 31) sh[warp] = inc;
        __syncthreads();
        const int v = lane < CM_WARPS ? sh[lane] : 0;
        const int from = before + __reduce_add_sync(0xffffffffu, lane < warp ? v : 0) + inc - mine;
        if (x >= from && x < from + mine) { sh[CM_WARPS] = i; sh[CM_WARPS + 1] = from; }
        before += __reduce_add_sync(0xffffffffu, v);
        if (x < before || i0 + CM_THREADS >= a.items) break;
    }
    __syncthreads();
    start = sh[CM_WARPS + 1];
    return sh[CM_WARPS];
}

// ---- the attention kernel ----
// Shared memory: the ring (per warp, CM_STAGES stages of keys then values), the terms of the queries, the masks of the nodes.
// bf16 rows are swizzled by 16-byte units for ldmatrix (unit ^ row & 7); fp32 keys by (row & 1) << 2 and values by
// ((row >> 1) & 3) << 1, for a lane's own 16-byte reads: a lane has the key n = lane / 4 of a score tile and of each 16 dims
// the four from 4 (lane % 4) on, which are its elements of two k-steps; of a P V tile the keys 2 (lane % 4) and the next, and
// of each 32 dims the four from 4 (lane / 4) on, which are its column of four tiles. Where a dim stands in a k-step and where a
// column in a tile is free as long as both operands, or all who read the result, agree.
// CL: a cluster of CTAs does a unit, each an equal run of its chunks, and their results meet in distributed shared memory: for
// calls that are all latency. Else the units' chunks are dealt out as above.
// PAGED: keys through the row's table of pages. A chunk's keys stand in one page or in up to four; their entries are fetched a chunk ahead of
// its copies, an entry a lane, and an entry that is no page (or a row of a negative length) leaves zeros, which no query sees.
template <class KE, class QE, int HDP, int R, bool BLOCKS, bool CL, bool PAGED = false>
__global__ void __launch_bounds__(CM_THREADS, CmCfg<KE, QE, HDP, R>::ctas(BLOCKS)) k_cache_attention(const __grid_constant__ CmArgs a) {
    using F = CmCfg<KE, QE, HDP, R>;
    constexpr int KC = F::KC, NT = F::NT, NQ = F::NQ, NP = F::NP, ROW = F::ROW, UPR = F::UPR, M = F::M, NH = F::NH;
    constexpr bool R8 = F::R8;
    constexpr int CM_STAGE = F::CM_STAGE, CM_STAGES = F::CM_STAGES;
    extern __shared__ __align__(128) char smem[];
    char *ring = smem, *qs = smem + F::RING;
    __shared__ int sh[CM_WARPS + 2], joined;
    __shared__ uint32_t node_bits[BLOCKS ? 1 : M][8];       // ancestors of the tile's nodes (from node m0 / G on)
    __shared__ uint32_t used_bits[8];
    __shared__ int spar[BLOCKS ? 1 : NCMB_MAX_NODES];
    __shared__ int spicks[BLOCKS ? 1024 : 1];
    __shared__ float most[BLOCKS ? 1 : M];                  // the largest score of a row: -infinity where no token is
    __shared__ float wm[CM_WARPS][M], wl[CM_WARPS][M], cmax[M];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c4 = lane & 3;
    const int hd = a.c.hd, G = a.G;
    pdl_wait();
    pdl_launch_dependents();           // after the wait: one kernel ahead, not a queue of them that takes the SMs' room
    namespace cg = cooperative_groups;
    cg::cluster_group cl = cg::this_cluster();
    const int rank = CL ? (int)cl.block_rank() : 0, nc = CL ? (int)cl.num_blocks() : 1;
    CmPlan plan = {};
    if constexpr (!CL) plan = cm_plan<BLOCKS, KC>(a, gridDim.x, sh);
    int at = min((int64_t)blockIdx.x * plan.per, (int64_t)plan.total);
    const int end = min((int64_t)plan.total, (int64_t)at + plan.per);
    if (!CL && at >= end) return;
    int item_at = 0, item = CL ? blockIdx.z : 0;
    if constexpr (!CL) { if (a.items > 1) item = cm_find<BLOCKS, KC>(a, at, item_at, sh); }
    char *my = ring + warp * (CM_STAGES * CM_STAGE);
    do {
        const int n = cm_keys<BLOCKS>(a, item), nch = (n + KC - 1) / KC, span = cm_span(nch);
        int sub, kvh, tile, first, stop, from = 0, take = 0;
        if constexpr (CL) {
            const int share = ((nch + nc - 1) / nc + CM_WARPS - 1) & ~(CM_WARPS - 1);
            kvh = blockIdx.y; tile = a.tiles == 1 ? 0 : blockIdx.x / nc; sub = kvh * a.tiles + tile;
            first = min(nch, rank * share); stop = min(nch, first + share);
        } else {
            sub = cm_div(at - item_at, span); kvh = a.tiles == 1 ? sub : cm_div(sub, a.tiles); tile = sub - kvh * a.tiles;
            from = item_at + sub * span;                         // where the unit begins: its start, then its chunks
            take = min(from + span, end) - at;
            first = max(0, at - from - CM_START); stop = min(nch, at + take - from - CM_START);
        }
        auto advance = [&] {
            at += take;
            if (at == item_at + span * a.c.nkv * a.tiles) { item_at = at; item++; }
        };
        if (!CL && stop <= first) { advance(); continue; }       // its start alone
        const int unit = item * a.c.nkv * a.tiles + sub;
        const int m0 = tile * M;
        const int row = a.row0 + (BLOCKS ? item / a.T : item), tok = BLOCKS ? item % a.T : 0, len = BLOCKS ? n : n - a.T;
        const bool tail = !BLOCKS && stop * KC > len;            // this run has keys of the new tokens
        const int *par = a.parents ? a.parents + (int64_t)row * a.T : nullptr;
        __syncthreads();
        if (BLOCKS) {
            const int np = ((n - 1) >> a.block_log) + 1;
            const int *picks = a.picks + ((int64_t)(a.row0 * a.T + item) * a.c.nkv + kvh) * a.n_sel;
            for (int i = tid; i < np; i += CM_THREADS) spicks[i] = picks[i];
        } else if (par) {
            for (int i = tid; i < a.T; i += CM_THREADS) spar[i] = par[i];
        }
        __syncthreads();
        if (!BLOCKS && par) {
            for (int w = warp; w < 8; w += CM_WARPS) {
                const int t = w * 32 + lane;
                const uint32_t u = __ballot_sync(0xffffffffu, t < a.T && spar[t] >= -1 && spar[t] < t);
                if (lane == 0) used_bits[w] = u;
            }
            __syncthreads();
        }
        auto used = [&](int t) { return !par || ((used_bits[t >> 5] >> (t & 31)) & 1u); };
        const char *kb = a.c.k + row * a.c.rs + kvh * a.c.hs, *vb = a.c.v + row * a.c.rs + kvh * a.c.hs;
        const int lu = lane % UPR, lr = lane / UPR;
        constexpr int RPI = 32 / UPR;                            // rows that the warp's lanes cover at once
        const bool lane_in = lu * 16 < hd * (int)sizeof(KE);
        // A lane copies 16 bytes of every RPI-th key. Its rows are lr + i RPI with lr < RPI, a power of two, so the swizzles of row i
        // differ from row 0's by a constant.
        const uint32_t to_k = cm_smem(my) + lr * ROW + (F::BF ? lu ^ lr : lu ^ ((lr & 1) << 2)) * 16, to_v = cm_smem(my) + CM_STAGE / 2 + lr * ROW + (F::BF ? lu ^ lr : lu ^ ((lr >> 1) << 1)) * 16;
        constexpr auto swz_k = [](int i) { return F::BF ? ((i * RPI) & 7) * 16 : (((i * RPI) & 1) << 2) * 16; };
        constexpr auto swz_v = [](int i) { return F::BF ? ((i * RPI) & 7) * 16 : ((((i * RPI) >> 1) & 3) << 1) * 16; };
        const int64_t step = (int64_t)RPI * a.c.ts, mine = lr * a.c.ts + lu * 16;
        const bool fast = hd == HDP && (!BLOCKS || (1 << a.block_log) >= KC);
        // paged: entries of a chunk's pages, one a lane; unseen: four bits a stage, set for pages of its chunk that are none
        constexpr int MOST_PAGES = KC / 8;
        static_assert(!PAGED || (MOST_PAGES <= 4 && CM_STAGES <= 8), "a chunk's pages fit four bits");
        const int pages_log = PAGED ? max(0, CM_LOG(KC) - a.page_log) : 0, pages = 1 << pages_log, slot_log = CM_LOG(KC) - pages_log;
        const int *entries = PAGED ? a.table + row * a.table_stride : nullptr;
        const bool has_row = !PAGED || a.c.len[row] >= 0;
        uint32_t unseen = 0;
        auto fetch = [&](int ch) {
            int e = -1;
            if (PAGED && has_row && ch < stop && lane < MOST_PAGES && lane < pages) {
                const int i = ch * KC >> a.page_log;
                if (i + lane < a.max_pages) e = __ldg(entries + i + lane);
            }
            return e;
        };
        auto load_paged = [&](int ch, int stage, int entry) {
            const bool there = (unsigned)entry < (unsigned)a.n_pages;
            const uint32_t none = ~__ballot_sync(0xffffffffu, there) & ((1u << pages) - 1);
            unseen = (unseen & ~(15u << 4 * stage)) | none << 4 * stage;
            const uint32_t ks = to_k + stage * CM_STAGE, vs = to_v + stage * CM_STAGE;
            const int64_t at = (int64_t)(ch * KC & ((1 << a.page_log) - 1)) * a.c.ts + lu * 16;
            const bool whole = fast && none == 0 && (ch + 1) * KC <= len;
#pragma unroll
            for (int i = 0; i < KC / RPI; i++) {
                const int r = lr + i * RPI, j = r >> slot_log;
                const int64_t off = (int64_t)__shfl_sync(0xffffffffu, entry, j) * a.ps + (int64_t)(r - (j << slot_log)) * a.c.ts + at;
                const uint32_t dk = (ks ^ swz_k(i)) + i * RPI * ROW, dv = (vs ^ swz_v(i)) + i * RPI * ROW;
                if (whole) {
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dk), "l"(kb + off) : "memory");
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dv), "l"(vb + off) : "memory");
                } else {
                    const int pos = ch * KC + r;
                    const bool ok = lane_in && pos < n && !((none >> j) & 1u) && !(tail && pos >= len && !used(pos - len));
                    cm_cp16(dk, kb + (ok ? off : 0), ok);
                    cm_cp16(dv, vb + (ok ? off : 0), ok);
                }
            }
        };
        auto load = [&](int ch, int stage) {
            const uint32_t ks = to_k + stage * CM_STAGE, vs = to_v + stage * CM_STAGE;
            if (fast && (ch + 1) * KC <= len) {                  // keys side by side, all there
                int64_t slot = ch * KC;
                if (BLOCKS) slot = ((int64_t)spicks[ch * KC >> a.block_log] << a.block_log) + (ch * KC & ((1 << a.block_log) - 1));
                const char *kp = kb + slot * a.c.ts + mine, *vp = vb + slot * a.c.ts + mine;
#pragma unroll
                for (int i = 0; i < KC / RPI; i++) {
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((ks ^ swz_k(i)) + i * RPI * ROW), "l"(kp) : "memory");
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((vs ^ swz_v(i)) + i * RPI * ROW), "l"(vp) : "memory");
                    kp += step; vp += step;
                }
                return;
            }
#pragma unroll 1
            for (int i = 0; i < KC / RPI; i++) {
                const int r = lr + i * RPI, pos = ch * KC + r;
                bool ok = lane_in && pos < n;
                int64_t slot = pos;
                if (BLOCKS) slot = ok ? ((int64_t)spicks[pos >> a.block_log] << a.block_log) + (pos & ((1 << a.block_log) - 1)) : 0;
                else if (tail && ok && pos >= len) ok = used(pos - len);
                const int64_t off = ok ? slot * a.c.ts + lu * 16 : 0;
                const int xk = F::BF ? ((i * RPI) & 7) * 16 : (((i * RPI) & 1) << 2) * 16, xv = F::BF ? xk : ((((i * RPI) >> 1) & 3) << 1) * 16;
                cm_cp16((ks ^ xk) + i * RPI * ROW, kb + off, ok);
                cm_cp16((vs ^ xv) + i * RPI * ROW, vb + off, ok);
            }
        };
        // the tile's queries as terms, zero where no query stands, and what each of its nodes sees; under the first loads
        auto prepare = [&] {
#pragma unroll 1
            for (int i = tid; i < M * HDP / 8; i += CM_THREADS) {
                const int m = i / (HDP / 8), d0 = i % (HDP / 8) * 8, mm = m0 + m;
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; e++) x[e] = 0.f;
                if (mm < a.M && d0 < hd) {
                    const int t = BLOCKS ? tok : mm / G, h = kvh * G + mm % G;
                    if (BLOCKS || used(t)) {
                        const char *p = a.q + ((int64_t)row * a.T + t) * a.ldq + ((int64_t)h * hd + d0) * sizeof(QE);
                        if (sizeof(QE) == 4) {
                            *(float4 *)&x[0] = *(const float4 *)p;
                            *(float4 *)&x[4] = *(const float4 *)(p + 16);
                        } else {
                            const uint4 u = *(const uint4 *)p;
                            const uint32_t uu[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                            for (int e = 0; e < 4; e++) { const float2 f = cm_unpack(uu[e]); x[2 * e] = f.x; x[2 * e + 1] = f.y; }
                        }
                    }
                }
                if constexpr (F::BF) {
#pragma unroll
                    for (int k = 0; k < (R8 ? 2 * F::QT : NQ); k++) {
                        uint32_t u[4] = {0, 0, 0, 0};
#pragma unroll
                        for (int e = 0; k < NQ && e < 4; e++) {
                            u[e] = cm_pack(x[2 * e], x[2 * e + 1]);
                            const float2 f = cm_unpack(u[e]);
                            x[2 * e] -= f.x; x[2 * e + 1] -= f.y;
                        }
                        const int r = k * M + m;                     // 8 rows: terms 0 and 1 are one tile of 16, then 2 and zeros
                        *(uint4 *)(qs + r * ROW + (((d0 / 8) ^ (r & 7)) * 16)) = make_uint4(u[0], u[1], u[2], u[3]);
                    }
                } else {
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        uint32_t hi[4], lo[4];
#pragma unroll
                        for (int e = 0; e < 4; e++) cm_tf32<PAGED>(x[4 * h + e], hi[e], lo[e]);
                        const int u = (d0 / 4 + h) ^ ((m & 1) << 2);
                        *(uint4 *)(qs + m * ROW + u * 16) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                        *(uint4 *)(qs + (M + m) * ROW + u * 16) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                    }
                }
            }
            // No token, no share: such a row's scores are zeros by keys that may hold anything. (A NaN of another row becomes an infinity,
            // which its sum, a NaN too, makes a NaN again.)
            if (!BLOCKS && a.scores && tid < M) most[tid] = m0 + tid < a.M && used((m0 + tid) / G) ? INFINITY : -INFINITY;
            if (tail) {
                const int t0 = m0 / G, nt = (min(a.M, m0 + M) + G - 1) / G - t0;   // nodes of this tile
                for (int i = tid; i < nt; i += CM_THREADS) {
                    const int t = t0 + i;
#pragma unroll 1
                    for (int w = 0; w < 8; w++) node_bits[i][w] = par ? 0u : t >= 32 * w + 31 ? 0xffffffffu : t >= 32 * w ? (2u << (t - 32 * w)) - 1 : 0u;
#pragma unroll 1
                    for (int x = par ? t : -1; x >= 0 && used(x); x = spar[x]) node_bits[i][x >> 5] |= 1u << (x & 31);
                }
            }
            __syncthreads();
        };
        float O[HDP / 8][2 * NH], mx[NH], ls[NH];                // context, maximum and sum of the lane's rows
#pragma unroll
        for (int j = 0; j < HDP / 8; j++)
#pragma unroll
            for (int e = 0; e < 2 * NH; e++) O[j][e] = 0.f;
#pragma unroll
        for (int hh = 0; hh < NH; hh++) { mx[hh] = -INFINITY; ls[hh] = 0.f; }
        int stage = 0, entry = -1;
        if constexpr (PAGED) entry = fetch(first + warp);
        // loads run CM_STAGES - 1 chunks ahead of the arithmetic
        for (int ch = first + warp - (CM_STAGES - 1) * CM_WARPS, ahead = 0; ch < stop; ch += CM_WARPS) {
            const int next = ch + (CM_STAGES - 1) * CM_WARPS;
            __syncwarp();                                        // the stage it goes to has been read
            if constexpr (PAGED) {
                if (next < stop) load_paged(next, ahead, entry);
                entry = fetch(next + CM_WARPS);
            } else {
                if (next < stop) load(next, ahead);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            if (++ahead == CM_STAGES) ahead = 0;
            if (ch < first) {
                if (next == first + warp) prepare();
                continue;
            }
            asm volatile("cp.async.wait_group %0;" ::"n"(CM_STAGES - 1) : "memory");
            __syncwarp();
            const char *kt = my + stage * CM_STAGE, *vt = kt + CM_STAGE / 2;
            const uint32_t none = PAGED ? (unseen >> 4 * stage) & 15u : 0u;
            const bool masked = (ch + 1) * KC > len || none != 0;
            float S[NT][4];
#pragma unroll
            for (int j = 0; j < NT; j++) S[j][0] = S[j][1] = S[j][2] = S[j][3] = 0.f;
            if constexpr (F::BF) {
                float L[NT][4];                                  // 16 rows: the smaller terms
#pragma unroll
                for (int j = 0; j < NT; j++) L[j][0] = L[j][1] = L[j][2] = L[j][3] = 0.f;
#pragma unroll 1
                for (int kp = 0; kp < HDP / 32; kp++) {          // two k-steps at a time
                    uint32_t kf[NT][4];
#pragma unroll
                    for (int j = 0; j < NT; j++)
                        cm_ldm4(kf[j], cm_smem(kt) + (8 * j + (lane & 7)) * ROW + (((4 * kp + (lane >> 3)) ^ (lane & 7)) * 16));
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const int qr = lane & 15, qu = 4 * kp + 2 * e + (lane >> 4);
#pragma unroll
                        for (int k = F::QT - 1; k >= 0; k--) {
                            uint32_t qf[4];
                            cm_ldm4(qf, cm_smem(qs) + (16 * k + qr) * ROW + ((qu ^ (qr & 7)) * 16));
#pragma unroll
                            for (int j = 0; j < NT; j++) cm_mma_bf16(k && !R8 ? L[j] : S[j], qf, kf[j][2 * e], kf[j][2 * e + 1]);
                        }
                    }
                }
#pragma unroll
                for (int j = 0; j < NT; j++)
#pragma unroll
                    for (int e = 0; e < 4; e++) S[j][e] += L[j][e];
            } else {
                // paged: leading products of even and of odd k-steps apart, half as many cuts of an accumulator (8 x 128, 3000 tokens: errors of 8e-7 -> 5e-7, 1% of the time)
                float L[NT][4], S2[NT][4];
#pragma unroll
                for (int j = 0; j < NT; j++) S2[j][0] = S2[j][1] = S2[j][2] = S2[j][3] = 0.f;
#pragma unroll
                for (int j = 0; j < NT; j++) L[j][0] = L[j][1] = L[j][2] = L[j][3] = 0.f;
#pragma unroll 1
                for (int i = 0; i < HDP / 16; i++) {             // two k-steps at a time
                    const int u0 = (4 * i + c4) ^ ((g & 1) << 2);       // rows g and g + 8: the same parity
                    uint32_t ah[2][4], al[2][4];
                    {
                        const uint4 h0 = *(const uint4 *)(qs + g * ROW + u0 * 16), l0 = *(const uint4 *)(qs + (M + g) * ROW + u0 * 16);
                        if constexpr (R8) {                      // leading terms in rows 0 ... 7, remainders in 8 ... 15
                            ah[0][0] = h0.x; ah[0][1] = l0.x; ah[0][2] = h0.y; ah[0][3] = l0.y;
                            ah[1][0] = h0.z; ah[1][1] = l0.z; ah[1][2] = h0.w; ah[1][3] = l0.w;
                        } else {
                            const uint4 h1 = *(const uint4 *)(qs + (g + 8) * ROW + u0 * 16), l1 = *(const uint4 *)(qs + (M + g + 8) * ROW + u0 * 16);
                            ah[0][0] = h0.x; ah[0][1] = h1.x; ah[0][2] = h0.y; ah[0][3] = h1.y;
                            ah[1][0] = h0.z; ah[1][1] = h1.z; ah[1][2] = h0.w; ah[1][3] = h1.w;
                            al[0][0] = l0.x; al[0][1] = l1.x; al[0][2] = l0.y; al[0][3] = l1.y;
                            al[1][0] = l0.z; al[1][1] = l1.z; al[1][2] = l0.w; al[1][3] = l1.w;
                        }
                    }
#pragma unroll
                    for (int j = 0; j < NT; j++) {
                        const float4 kx = *(const float4 *)(kt + (8 * j + g) * ROW + u0 * 16);
                        const float kv[4] = {kx.x, kx.y, kx.z, kx.w};
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            uint32_t bh[2], bl[2];
                            cm_tf32<PAGED>(kv[2 * e], bh[0], bl[0]);
                            cm_tf32<PAGED>(kv[2 * e + 1], bh[1], bl[1]);
                            if constexpr (!R8) cm_mma_tf32(L[j], al[e], bh[0], bh[1]);
                            cm_mma_tf32(L[j], ah[e], bl[0], bl[1]);
                            cm_mma_tf32(PAGED && e ? S2[j] : S[j], ah[e], bh[0], bh[1]);
                        }
                    }
                }
#pragma unroll
                for (int j = 0; j < NT; j++)
#pragma unroll
                    for (int e = 0; e < 4; e++) S[j][e] += PAGED ? S2[j][e] + L[j][e] : L[j][e];
            }
#pragma unroll
            for (int j = 0; j < NT; j++)
#pragma unroll
                for (int e = 0; e < 2 * NH; e++) S[j][e] = (R8 ? S[j][e] + S[j][2 + e] : S[j][e]) * a.c2;
            if (masked) {
#pragma unroll
                for (int hh = 0; hh < NH; hh++) {
                    const int mm = min(m0 + g + 8 * hh, a.M - 1);
                    const uint32_t *bits = node_bits[BLOCKS ? 0 : mm / G - m0 / G];
#pragma unroll
                    for (int j = 0; j < NT; j++)
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const int pos = ch * KC + 8 * j + 2 * c4 + e;
                            bool see = pos < len;
                            if (!BLOCKS && !see && pos < n) see = (bits[(pos - len) >> 5] >> ((pos - len) & 31)) & 1u;
                            if (PAGED && ((none >> ((pos & (KC - 1)) >> slot_log)) & 1u)) see = false;
                            if (!see) S[j][2 * hh + e] = -INFINITY;
                        }
                }
            }
            if (!BLOCKS && a.scores) {
                float *sp = a.scores + ((int64_t)item * a.c.nkv + kvh) * a.M * a.pitch + ch * KC + 2 * c4;
#pragma unroll
                for (int hh = 0; hh < NH; hh++) {
                    const int mm = m0 + g + 8 * hh;
                    if (mm < a.M) {
                        const float top = most[g + 8 * hh];
#pragma unroll
                        for (int j = 0; j < NT; j++) *(float2 *)(sp + mm * a.pitch + 8 * j) = make_float2(fminf(S[j][2 * hh], top), fminf(S[j][2 * hh + 1], top));
                    }
                }
            }
            float al[NH];
#pragma unroll
            for (int hh = 0; hh < NH; hh++) {
                float t = mx[hh];
#pragma unroll
                for (int j = 0; j < NT; j++) t = fmaxf(t, fmaxf(S[j][2 * hh], S[j][2 * hh + 1]));
                t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 1));
                t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 2));
                const float base = t == -INFINITY ? 0.f : t;
                al[hh] = cm_exp2(mx[hh] - base);
                mx[hh] = t;
                float sum = 0.f;
#pragma unroll
                for (int j = 0; j < NT; j++)
#pragma unroll
                    for (int e = 0; e < 2; e++) { S[j][2 * hh + e] = cm_exp2(S[j][2 * hh + e] - base); sum += S[j][2 * hh + e]; }
                ls[hh] = ls[hh] * al[hh] + sum;
            }
            if (++stage == CM_STAGES) stage = 0;
            bool odd = false;                                    // an infinity or NaN among values that not every row sees
            if (masked && !BLOCKS) {
                for (int i = lane; i < KC * HDP; i += 32) {
                    const float x = (float)((const KE *)vt)[i];
                    odd |= !(fabsf(x) < INFINITY);
                }
                odd = __any_sync(0xffffffffu, odd);
            }
            if (odd) {
                // rows that do not see such a value must not multiply it by zero: one key at a time
#pragma unroll
                for (int j = 0; j < HDP / 8; j++)
#pragma unroll
                    for (int e = 0; e < 2 * NH; e++) O[j][e] *= al[e >> 1];
#pragma unroll
                for (int jj = 0; jj < NT; jj++)
#pragma unroll 1
                    for (int r = 0; r < 8; r++) {
                        const int src = (lane & ~3) | (r >> 1), kr = 8 * jj + r;
                        float p[NH];
#pragma unroll
                        for (int hh = 0; hh < NH; hh++) p[hh] = __shfl_sync(0xffffffffu, (r & 1) ? S[jj][2 * hh + 1] : S[jj][2 * hh], src);
#pragma unroll
                        for (int j = 0; j < HDP / 8; j++)
#pragma unroll
                            for (int e = 0; e < 2; e++) {
                                const int d = F::BF ? 8 * j + 2 * c4 + e : 32 * (j / 4) + 8 * c4 + 4 * e + j % 4;
                                const int u = d * (int)sizeof(KE) / 16, us = F::BF ? u ^ (kr & 7) : u ^ (((kr >> 1) & 3) << 1);
                                const float x = (float)*(const KE *)(vt + kr * ROW + us * 16 + d * sizeof(KE) % 16);
#pragma unroll
                                for (int hh = 0; hh < NH; hh++) if (p[hh] != 0.f) O[j][2 * hh + e] = fmaf(p[hh], x, O[j][2 * hh + e]);
                            }
                    }
                continue;
            }
            auto add = [&](int j, const float (&c)[4]) {         // a chunk's part of tile j
#pragma unroll
                for (int e = 0; e < 2 * NH; e++) O[j][e] = fmaf(O[j][e], al[e >> 1], R8 ? c[e] + c[(2 + e) & 3] : c[e]);
            };
            if constexpr (F::BF) {
                constexpr int PT = R8 ? (NP + 1) / 2 : NP;       // tiles the probabilities take
                uint32_t pf[KC / 16][PT][4];
#pragma unroll
                for (int k2 = 0; k2 < KC / 16; k2++)
#pragma unroll
                    for (int e = 0; e < 2 * NH; e++) {           // 16 rows: e & 1 is the row, e >> 1 the half of the keys; 8: e the half
                        float *s = R8 ? &S[2 * k2 + e][0] : &S[2 * k2 + (e >> 1)][2 * (e & 1)];
#pragma unroll
                        for (int k = 0; k < (R8 ? 2 * PT : NP); k++) {
                            uint32_t u = 0;
                            if (k < NP) {
                                u = cm_pack(s[0], s[1]);
                                const float2 f = cm_unpack(u);
                                s[0] -= f.x; s[1] -= f.y;
                            }
                            if (R8) pf[k2][k / 2][2 * e + (k & 1)] = u; else pf[k2][k][e] = u;
                        }
                    }
#pragma unroll
                for (int jp = 0; jp < HDP / 16; jp++) {          // two tiles of 8 dims at a time
                    float c0[4] = {0.f, 0.f, 0.f, 0.f}, c1[4] = {0.f, 0.f, 0.f, 0.f};
                    uint32_t vf[KC / 16][4];
#pragma unroll
                    for (int k2 = 0; k2 < KC / 16; k2++) {
                        const int vr = 16 * k2 + (lane & 15);
                        cm_ldm4t(vf[k2], cm_smem(vt) + vr * ROW + (((2 * jp + (lane >> 4)) ^ (vr & 7)) * 16));
                    }
#pragma unroll
                    for (int k = PT - 1; k >= 0; k--)            // small terms first
#pragma unroll
                        for (int k2 = 0; k2 < KC / 16; k2++) {
                            cm_mma_bf16(c0, pf[k2][k], vf[k2][0], vf[k2][1]);
                            cm_mma_bf16(c1, pf[k2][k], vf[k2][2], vf[k2][3]);
                        }
                    add(2 * jp, c0);
                    add(2 * jp + 1, c1);
                }
            } else {
                uint32_t ph[NT][4], pl[NT][4];
#pragma unroll
                for (int j = 0; j < NT; j++) {                   // k position c: key 2 c, position c + 4: key 2 c + 1
                    if constexpr (R8) {
                        cm_tf32<PAGED>(S[j][0], ph[j][0], ph[j][1]);
                        cm_tf32<PAGED>(S[j][1], ph[j][2], ph[j][3]);
                    } else {
                        cm_tf32<PAGED>(S[j][0], ph[j][0], pl[j][0]); cm_tf32<PAGED>(S[j][2], ph[j][1], pl[j][1]);
                        cm_tf32<PAGED>(S[j][1], ph[j][2], pl[j][2]); cm_tf32<PAGED>(S[j][3], ph[j][3], pl[j][3]);
                    }
                }
#pragma unroll
                for (int jj = 0; jj < HDP / 32; jj++) {          // four tiles of 8 dims at a time
                    float cc[4][4];
#pragma unroll
                    for (int x = 0; x < 4; x++)
#pragma unroll
                        for (int e = 0; e < 4; e++) cc[x][e] = 0.f;
#pragma unroll
                    for (int j = 0; j < NT; j++) {
                        const int r0 = 8 * j + 2 * c4, u = (8 * jj + g) ^ (c4 << 1);        // (row >> 1) & 3 = c4 for both rows
                        const float4 v0 = *(const float4 *)(vt + r0 * ROW + u * 16), v1 = *(const float4 *)(vt + (r0 + 1) * ROW + u * 16);
                        const float va[4] = {v0.x, v0.y, v0.z, v0.w}, vv[4] = {v1.x, v1.y, v1.z, v1.w};
#pragma unroll
                        for (int x = 0; x < 4; x++) {
                            uint32_t bh[2], bl[2];
                            cm_tf32<PAGED>(va[x], bh[0], bl[0]);
                            cm_tf32<PAGED>(vv[x], bh[1], bl[1]);
                            if constexpr (!R8) cm_mma_tf32(cc[x], pl[j], bh[0], bh[1]);
                            cm_mma_tf32(cc[x], ph[j], bl[0], bl[1]);
                            cm_mma_tf32(cc[x], ph[j], bh[0], bh[1]);
                        }
                    }
#pragma unroll
                    for (int x = 0; x < 4; x++) add(4 * jj + x, cc[x]);
                }
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        // the warps' results meet in shared memory: every warp's maxima first, then scaled contexts where the ring was
#pragma unroll
        for (int hh = 0; hh < NH; hh++) {
            float l = ls[hh];
            l += __shfl_xor_sync(0xffffffffu, l, 1);
            l += __shfl_xor_sync(0xffffffffu, l, 2);
            if (c4 == 0) { wm[warp][g + 8 * hh] = mx[hh]; wl[warp][g + 8 * hh] = l; }
        }
        __syncthreads();
        float *ctx_sh = (float *)ring;                           // [warp][M][HDP]
        static_assert(CM_WARPS * M * HDP * 4 <= F::RING, "contexts of the warps fit the ring");
#pragma unroll
        for (int hh = 0; hh < NH; hh++) {
            const int m = g + 8 * hh;
            float top = wm[0][m];
#pragma unroll
            for (int w = 1; w < CM_WARPS; w++) top = fmaxf(top, wm[w][m]);
            const float f = mx[hh] == -INFINITY ? 0.f : cm_exp2(mx[hh] - top);
            float *o = ctx_sh + (warp * M + m) * HDP;
#pragma unroll
            for (int j = 0; j < HDP / 8; j++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int d = F::BF ? 8 * j + 2 * c4 + e : 32 * (j / 4) + 8 * c4 + 4 * e + j % 4;
                    o[d] = O[j][2 * hh + e] * f;
                }
        }
        __syncthreads();
        const bool whole = first == 0 && stop == nch;
        float *sums = CL ? nullptr : a.sums + ((int64_t)blockIdx.x + unit) * F::SUMS;
        float *part = CL ? nullptr : a.ctx + (2 * (int64_t)blockIdx.x + (first == 0)) * F::CTX;
        if constexpr (!CL) {
            if (tid == 0 && first == 0) a.range[unit].x = blockIdx.x;
            if (tid == 0 && stop == nch) a.range[unit].y = blockIdx.x;
        }
        if (tid < M) {
            const int m = tid;
            float top = wm[0][m], l = 0.f;
#pragma unroll
            for (int w = 1; w < CM_WARPS; w++) top = fmaxf(top, wm[w][m]);
#pragma unroll
            for (int w = 0; w < CM_WARPS; w++) l += wm[w][m] == -INFINITY ? 0.f : wl[w][m] * cm_exp2(wm[w][m] - top);
            if constexpr (CL) cmax[m] = top;
            else { sums[m] = top; sums[M + m] = l; }
            wl[0][m] = l;                                        // read by the owner of this m alone until the barrier
        }
        if constexpr (!CL) __syncthreads();
        const int nm = min(M, a.M - m0);                         // rows that hold a query
        auto write = [&](int m, int d, float4 o, float l) {      // a result, four dims of a row
            const int mm = m0 + m, t = BLOCKS ? tok : mm / G, h = kvh * G + mm % G;
            const float r = l > 0.f ? 1.f / l : 0.f;
            if (!BLOCKS && !used(t)) o = make_float4(0.f, 0.f, 0.f, 0.f);        // not by r = 0: values may hold infinities
            QE *p = (QE *)(a.out + ((int64_t)row * a.T + t) * a.ldo) + (int64_t)h * hd + d;
            if constexpr (sizeof(QE) == 4) *(float4 *)p = make_float4(o.x * r, o.y * r, o.z * r, o.w * r);
            else *(uint2 *)p = make_uint2(cm_pack(o.x * r, o.y * r), cm_pack(o.z * r, o.w * r));
        };
        if constexpr (CL) {
            // the warps' contexts first, then the CTAs': a thread has the same four dims of a row in every CTA, scaled by that CTA's
            // maximum against the cluster's. Loads from the others all at once: each takes some 600 cycles.
#pragma unroll 1
            for (int i = tid; i < nm * (HDP / 4); i += CM_THREADS) {
                float4 *p = (float4 *)ctx_sh + i;
                float4 o = *p;
#pragma unroll
                for (int w = 1; w < CM_WARPS; w++) {
                    const float4 x = p[w * M * HDP / 4];
                    o.x += x.x; o.y += x.y; o.z += x.z; o.w += x.w;
                }
                *p = o;
            }
            cl.sync();
#pragma unroll 1
            for (int i = rank * CM_THREADS + tid; i < nm * (HDP / 4); i += nc * CM_THREADS) {
                const int m = i / (HDP / 4), d = i % (HDP / 4) * 4;
                float cm[CM_MAXC], cw[CM_MAXC], top = -INFINITY, l = 0.f;
                float4 x[CM_MAXC], o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int r = 0; r < CM_MAXC; r++) {
                    const int rr = min(r, nc - 1);
                    cm[r] = *cl.map_shared_rank(&cmax[m], rr);
                    cw[r] = *cl.map_shared_rank(&wl[0][m], rr);
                    x[r] = *((const float4 *)cl.map_shared_rank(ctx_sh, rr) + i);
                    if (r >= nc) cm[r] = -INFINITY;
                    top = fmaxf(top, cm[r]);
                }
                const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
                for (int r = 0; r < CM_MAXC; r++) {
                    const float f = cm_exp2(cm[r] - base);
                    l = fmaf(cw[r], f, l);
                    o.x = fmaf(x[r].x, f, o.x); o.y = fmaf(x[r].y, f, o.y); o.z = fmaf(x[r].z, f, o.z); o.w = fmaf(x[r].w, f, o.w);
                }
                if (d < hd) write(m, d, o, l);
            }
            if (!BLOCKS && a.weights) {                          // one tile a kv head: this CTA's slots, from its own scores
                if (tid < M) {
                    float top = -INFINITY, l = 0.f;
                    for (int r = 0; r < nc; r++) top = fmaxf(top, *cl.map_shared_rank(&cmax[tid], r));
                    const float base = top == -INFINITY ? 0.f : top;
                    for (int r = 0; r < nc; r++) l = fmaf(*cl.map_shared_rank(&wl[0][tid], r), cm_exp2(*cl.map_shared_rank(&cmax[tid], r) - base), l);
                    wm[0][tid] = tid < a.M && l > 0.f && used(tid / G) ? top + log2f(l) : INFINITY;
                }
                __syncthreads();
                const float *sp = a.scores + ((int64_t)item * a.c.nkv + kvh) * a.M * a.pitch;
                float *wp = a.weights + ((int64_t)row * a.c.nkv + kvh) * a.c.cap;
#pragma unroll 1
                for (int key = first * KC + tid; key < min(n, stop * KC); key += CM_THREADS) {
                    float w = 0.f;
#pragma unroll 4
                    for (int m = 0; m < a.M; m++) w += cm_exp2(sp[m * a.pitch + key] - wm[0][m]);
                    wp[key] = key < len ? wp[key] + w : w;
                }
            }
            cl.sync();                                           // the others have read this CTA's results
        }
#pragma unroll 1
        for (int i = tid; !CL && i < nm * (HDP / 4); i += CM_THREADS) {
            const int m = i / (HDP / 4), d = i % (HDP / 4) * 4;
            if (d >= hd) continue;
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < CM_WARPS; w++) {
                const float4 x = *(const float4 *)(ctx_sh + (w * M + m) * HDP + d);
                o.x += x.x; o.y += x.y; o.z += x.z; o.w += x.w;
            }
            if (whole) write(m, d, o, wl[0][m]);
            else *(float4 *)(part + m * HDP + d) = o;
        }
        if (!CL && a.done && !whole) {
            // the CTA that brings the unit's last chunks joins its parts
            __threadfence();
            __syncthreads();
            if (tid == 0) joined = atomicAdd(&a.done[unit], stop - first) + stop - first;
            __syncthreads();
            if (joined == nch) {
                if (tid == 0) a.done[unit] = 0;                  // for the next call
                __threadfence();
                const int c0 = (from + CM_START) / plan.per, parts = (from + span - 1) / plan.per - c0 + 1;
                const float *s0 = a.sums + ((int64_t)c0 + unit) * F::SUMS, *p0 = a.ctx + 2 * (int64_t)c0 * F::CTX;
                constexpr int D4 = HDP / 4;
                int ways = 1;                                    // threads that share the parts of four dims of a row
                while (ways * 2 * nm * D4 <= CM_THREADS) ways *= 2;
                const int way = tid & (ways - 1);
#pragma unroll 1
                for (int i0 = 0; i0 < nm * D4; i0 += CM_THREADS / ways) {
                    const int i = i0 + tid / ways, m = min(i / D4, nm - 1), d = i % D4 * 4;
                    float top = -INFINITY, l = 0.f;
                    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
                    auto add = [&](float x, float xl, float4 p) {
                        const float t = fmaxf(top, x), base = t == -INFINITY ? 0.f : t, fo = cm_exp2(top - base), fp = cm_exp2(x - base);
                        top = t;
                        l = l * fo + xl * fp;
                        o.x = o.x * fo + p.x * fp; o.y = o.y * fo + p.y * fp; o.z = o.z * fo + p.z * fp; o.w = o.w * fo + p.w * fp;
                    };
#pragma unroll 4
                    for (int c = way; c < parts; c += ways) {
                        const float *s = s0 + c * F::SUMS, *p = p0 + (int64_t)(2 * c + (c == 0)) * F::CTX;
                        add(__ldcg(s + m), __ldcg(s + M + m), __ldcg((const float4 *)(p + m * HDP + d)));
                    }
#pragma unroll 1
                    for (int w = 1; w < ways; w <<= 1) {
                        const float x = __shfl_xor_sync(0xffffffffu, top, w), xl = __shfl_xor_sync(0xffffffffu, l, w);
                        float4 p;
                        p.x = __shfl_xor_sync(0xffffffffu, o.x, w); p.y = __shfl_xor_sync(0xffffffffu, o.y, w);
                        p.z = __shfl_xor_sync(0xffffffffu, o.z, w); p.w = __shfl_xor_sync(0xffffffffu, o.w, w);
                        add(x, xl, p);
                    }
                    if (way == 0 && i < nm * D4 && d < hd) write(m, d, o, l);
                }
            }
        }
        if (CL) break;
        advance();
    } while (at < end);
}

// ---- units that several CTAs share are joined; weights are added up ----
// CTAs [0, joins): rows of one unit each. A thread has four dims of a row; of the CTA's groups of HDP / 4 threads either each
// has a row, or (`split`: few units, each in many parts) all have the same row and every one a share of its parts.
// The others: `wkeys` slots of one (row, kv head) each, from the scores that the kernel above left.
constexpr int CM_PITCH = 128;        // scores of a query: whole tiles of keys
// The CTAs that have a part of a unit; none (0, -1) for a range that the attention kernel cannot have written: no part is read by it
__device__ __forceinline__ int2 cm_range(const CmArgs &a, int64_t unit) {
    const int2 r = a.range[unit];
    return r.x >= 0 && r.x <= r.y && r.y < a.ctas ? r : make_int2(0, -1);
}
template <class KE, class QE, int HDP, int R, bool BLOCKS, bool PAGED = false>       // PAGED: each instance is in one file
__global__ void __launch_bounds__(CM_THREADS) k_cache_join(const __grid_constant__ CmArgs a, int joins, int split, int wkeys) {
    using F = CmCfg<KE, QE, HDP, R>;
    constexpr int M = F::M, D4 = HDP / 4, GROUPS = CM_THREADS / D4;
    __shared__ float lse[NCMB_MAX_NODES];
    __shared__ float gm[GROUPS], gl[GROUPS];
    __shared__ float4 go[GROUPS][D4];
    const int tid = threadIdx.x, G = a.G, hd = a.c.hd;
    pdl_wait();
    pdl_launch_dependents();           // after the wait: one kernel ahead, not a queue of them that takes the SMs' room
    const int gave_up = a.err ? *a.err : 0;               // CTAs that saw it set have left without a result
    const bool join = (int)blockIdx.x < joins;
    const int per_item = a.c.nkv * a.tiles, rows = split ? 1 : GROUPS, steps = M / rows;      // rows a CTA, CTAs a unit
    int item, sub, key0 = 0;
    if (join) { item = blockIdx.x / steps / per_item; sub = blockIdx.x / steps % per_item; }
    else {
        const int span = (int)((a.pitch + wkeys - 1) / wkeys), x = blockIdx.x - joins;
        key0 = x % span * wkeys;
        sub = x / span % a.c.nkv * a.tiles;
        item = x / span / a.c.nkv;
    }
    const int row = a.row0 + (BLOCKS ? item / a.T : item);
    const int *par = a.parents ? a.parents + (int64_t)row * a.T : nullptr;
    const int64_t unit0 = (int64_t)item * per_item + sub;
    if (join) {
        const int2 cr = cm_range(a, unit0);
        const int c0 = cr.x, c1 = cr.y;
        if (c0 >= c1 || gave_up) return;                         // written already
        const float *sums = a.sums + (c0 + unit0) * F::SUMS, *part = a.ctx + 2 * (int64_t)c0 * F::CTX;
        const int grp = tid / D4, d = tid % D4 * 4, kvh = sub / a.tiles;
        const int m = (int)(blockIdx.x % steps) * rows + (split ? 0 : grp), mm = sub % a.tiles * M + m;
        if (split && mm >= a.M) return;
        float top = -INFINITY, l = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        if (mm < a.M) {
#pragma unroll 4
            for (int c = split ? grp : 0; c <= c1 - c0; c += split ? GROUPS : 1) {
                const float x = sums[c * F::SUMS + m], xl = sums[c * F::SUMS + M + m];
                const float4 p = *(const float4 *)(part + (int64_t)(2 * c + (c == 0)) * F::CTX + m * HDP + d);
                const float t = fmaxf(top, x), base = t == -INFINITY ? 0.f : t, fo = cm_exp2(top - base), fp = cm_exp2(x - base);
                top = t;
                l = l * fo + xl * fp;
                o.x = o.x * fo + p.x * fp; o.y = o.y * fo + p.y * fp; o.z = o.z * fo + p.z * fp; o.w = o.w * fo + p.w * fp;
            }
        }
        if (split) {
            if (d == 0) { gm[grp] = top; gl[grp] = l; }
            go[grp][d / 4] = o;
            __syncthreads();
            if (grp > 0) return;
            for (int q = 0; q < GROUPS; q++) top = fmaxf(top, gm[q]);
            const float base = top == -INFINITY ? 0.f : top;
            l = 0.f;
            o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int q = 0; q < GROUPS; q++) {
                const float f = cm_exp2(gm[q] - base);
                const float4 p = go[q][d / 4];
                l = fmaf(gl[q], f, l);
                o.x = fmaf(p.x, f, o.x); o.y = fmaf(p.y, f, o.y); o.z = fmaf(p.z, f, o.z); o.w = fmaf(p.w, f, o.w);
            }
        }
        if (mm >= a.M || d >= hd) return;
        const int t = BLOCKS ? item % a.T : mm / G, h = kvh * G + mm % G;
        const float r = l > 0.f ? 1.f / l : 0.f;
        if (!BLOCKS && !cm_used(par, t)) o = make_float4(0.f, 0.f, 0.f, 0.f);
        QE *out = (QE *)(a.out + ((int64_t)row * a.T + t) * a.ldo) + (int64_t)h * hd + d;
        cm_put(out, o.x * r); cm_put(out + 1, o.y * r); cm_put(out + 2, o.z * r); cm_put(out + 3, o.w * r);
        return;
    }
    const int kvh = sub / a.tiles, n = cm_keys<BLOCKS>(a, item), len = n - a.T;
    if (key0 >= n || gave_up) return;
    const float *sc = a.scores + ((int64_t)item * a.c.nkv + kvh) * a.M * a.pitch;
    float *wp = a.weights + ((int64_t)row * a.c.nkv + kvh) * a.c.cap;
    const int stop = min(n, key0 + wkeys);
    float early[R == 8 ? 8 : 1][4], old[4];                      // few rows: scores and weights are on their way while the sums are formed
    if constexpr (R == 8) {
#pragma unroll
        for (int x = 0; x < 4; x++) old[x] = key0 + tid + x * CM_THREADS < min(stop, len) ? wp[key0 + tid + x * CM_THREADS] : 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
            for (int x = 0; x < 4; x++) {
                const int key = key0 + tid + x * CM_THREADS;
                early[i][x] = i < a.M && key < stop ? sc[i * a.pitch + key] : -INFINITY;
            }
    }
    for (int mb = 0; mb < a.M; mb += NCMB_MAX_NODES) {
        const int nm = min(NCMB_MAX_NODES, a.M - mb);
        __syncthreads();
        for (int i = tid; i < nm; i += CM_THREADS) {
            const int mm = mb + i, m = mm % M;
            const int64_t u = unit0 + mm / M;
            const int2 cr = cm_range(a, u);
            const float *sums = a.sums + (cr.x + u) * F::SUMS;
            float top = -INFINITY, l = 0.f;
#pragma unroll 4
            for (int c = 0; c <= cr.y - cr.x; c++) {
                const float x = sums[c * F::SUMS + m], xl = sums[c * F::SUMS + M + m];
                const float t = fmaxf(top, x), base = t == -INFINITY ? 0.f : t;
                l = l * cm_exp2(top - base) + xl * cm_exp2(x - base);
                top = t;
            }
            lse[i] = l > 0.f && cm_used(par, mm / G) ? top + log2f(l) : INFINITY;
        }
        __syncthreads();
        if (wkeys > CM_THREADS) {
            // few rows: four slots a thread, so that as many loads are under way
            float w[4] = {0.f, 0.f, 0.f, 0.f};
            if constexpr (R == 8) {
#pragma unroll
                for (int i = 0; i < 8; i++)
#pragma unroll
                    for (int x = 0; x < 4; x++) if (i < nm) w[x] += cm_exp2(early[i][x] - lse[i]);
            }
            for (int i = R == 8 ? nm : 0; i < nm; i++) {
                const float *s = sc + (int64_t)(mb + i) * a.pitch + key0 + tid;
                const float e = lse[i];
#pragma unroll
                for (int x = 0; x < 4; x++) if (key0 + tid + x * CM_THREADS < stop) w[x] += cm_exp2(s[x * CM_THREADS] - e);
            }
#pragma unroll
            for (int x = 0; x < 4; x++) {
                const int key = key0 + tid + x * CM_THREADS;
                if (key >= stop) continue;                       // the new tokens' slots are stored to, the others added to
                wp[key] = R == 8 ? old[x] + w[x] : mb || key < len ? wp[key] + w[x] : w[x];
            }
        } else if (key0 + tid < stop) {
            const int key = key0 + tid;
            float w = 0.f;
#pragma unroll 8
            for (int i = 0; i < nm; i++) w += cm_exp2(sc[(int64_t)(mb + i) * a.pitch + key] - lse[i]);
            wp[key] = mb || key < len ? wp[key] + w : w;
        }
    }
}

// ---- launches ----
// slots of a CTA that adds up weights: it finds the sums of M queries first, then goes over M scores a slot
inline int cm_wkeys(int M) { return M <= 32 ? 4 * CM_THREADS : CM_THREADS; }
constexpr int CM_ROUNDS = 8, CM_FUSED = 24;
// scratch of a launch: scores where weights are wanted, then what the join reads; false (said) when there is no room
template <class F> bool cm_parts(const char *who, CmArgs &a, int rows, int64_t units, int ctas) {
    auto whole = [](size_t bytes) { return (bytes + 255) & ~(size_t)255; };
    const size_t sc = a.weights ? (size_t)rows * a.c.nkv * a.M * a.pitch * 4 : 0, ranges = whole((size_t)units * 8);
    const size_t sums = whole((size_t)(units + ctas) * F::SUMS * 4), ctx = (size_t)ctas * 2 * F::CTX * 4;
    char *scratch = (char *)cache_scratch(who, sc + ranges + sums + ctx);
    if (!scratch) return false;
    a.scores = a.weights ? (float *)scratch : nullptr;
    a.range = (int2 *)(scratch + sc);
    a.sums = (float *)(scratch + sc + ranges);
    a.ctx = (float *)(scratch + sc + ranges + sums);
    a.ctas = ctas;
    return true;
}
// first(): launches what has to run before; only once nothing can be refused any more
template <class KE, class QE, int HDP, int R, bool BLOCKS, bool PAGED = false, class FIRST>
int cm_run_as(const char *who, CmArgs a, int max_keys, FIRST first) {
    using F = CmCfg<KE, QE, HDP, R>;
    a.tiles = (int)cdiv(a.M, F::M);
    const int smem = F::RING + F::QBYTES;
    static bool set = false;
    if (!set) {
        CUDA_CHECK(cudaFuncSetAttribute(k_cache_attention<KE, QE, HDP, R, BLOCKS, false, PAGED>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        CUDA_CHECK(cudaFuncSetAttribute(k_cache_attention<KE, QE, HDP, R, BLOCKS, true, PAGED>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        set = true;
    }
    // rows of a launch: as many as leave the scores some GB at most, and the count of chunks in 31 bits
    const int rows = a.c.rows, per_row = BLOCKS ? a.T : 1;
    const int64_t row_units = (int64_t)per_row * a.c.nkv * a.tiles;
    const int64_t row_chunks = row_units * (cdiv(BLOCKS ? (int64_t)a.n_sel << a.block_log : a.c.cap, F::KC) + CM_WARPS + CM_START);
    int64_t most = 0x70000000 / row_chunks;
    if (a.weights) {
        a.pitch = cdiv((int64_t)a.c.cap, CM_PITCH) * CM_PITCH;
        most = std::min(most, std::max<int64_t>(1, ((int64_t)2 << 30) / (a.c.nkv * a.M * a.pitch * 4)));
    }
    if (most < 1) return cache_refuse(who, "%lld pieces of keys in a row", (long long)row_chunks);
    const int step = (int)std::min<int64_t>(rows, most);
    const int64_t units = step * row_units, spans = a.weights ? cdiv(a.pitch, cm_wkeys(a.M)) * step * a.c.nkv : 0;
    if (units * F::M + spans > 0x7fffffff) return cache_refuse(who, "%lld query tiles", (long long)units);
    // Clusters: where one, of as many CTAs as give a warp two chunks and fit the GPU, does a unit in a few rounds. Single CTAs where they fit
    // in one and a half waves: a second launch costs more (picked blocks, fp32, 128 dims, 384 units of 3 keys: 12.7 us, dealt out 20.2).
    const int64_t chunks = cdiv(max_keys, F::KC);
    const int resident = F::ctas(BLOCKS) * ctx().sm_count;
    int nc = 1;
    while (nc < CM_MAXC && nc * 2 * CM_WARPS <= chunks && units * nc * 2 <= resident) nc *= 2;
    if (step == rows && units * nc <= 3 * ctx().sm_count && chunks <= (int64_t)CM_ROUNDS * nc * CM_WARPS && (!a.weights || a.tiles == 1)) {
        if (a.weights && !(a.scores = (float *)cache_scratch(who, (size_t)rows * a.c.nkv * a.M * a.pitch * 4))) return -1;
        a.items = rows * per_row;
        first();
        cache_launch(k_cache_attention<KE, QE, HDP, R, BLOCKS, true, PAGED>, dim3(nc * a.tiles, a.c.nkv, a.items), CM_THREADS, smem, nc, a);
        return 0;
    }
    const int ctas = (int)std::max<int64_t>(1, std::min<int64_t>(resident, cdiv(units * chunks, CM_WARPS)));
    if (!cm_parts<F>(who, a, step, units, ctas)) return -1;
    // Few parts a unit: the CTA that finishes it joins them. Many: a kernel of its own, which has a CTA for each row of a
    // unit; it also adds up weights.
    const bool fused = !a.weights && ctas <= CM_FUSED * units;
    if (fused && !(a.done = (int *)cache_scratch(who, (size_t)units * 4, SCRATCH_DONE))) return -1;
    const int split = ctas > 4 * units;
    first();
    for (int r = 0; r < rows; r += step) {
        const int nr = std::min(step, rows - r);
        a.row0 = r;
        a.items = nr * per_row;
        LAUNCH_PDL((k_cache_attention<KE, QE, HDP, R, BLOCKS, false, PAGED>), ctas, CM_THREADS, smem, a);
        if (fused) continue;
        const int64_t joins = nr * row_units * (F::M / (split ? 1 : CM_THREADS / (HDP / 4)));
        LAUNCH_PDL((k_cache_join<KE, QE, HDP, R, BLOCKS, PAGED>), (unsigned)(joins + spans / step * nr), CM_THREADS, 0, a, (int)joins, split, cm_wkeys(a.M));
    }
    return 0;
}

} // namespace ncmb
