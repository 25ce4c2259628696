// Attention over blocks of the cache that a cheap score picks for each query (ncmb_block_summaries and
// ncmb_block_attention, include/ncm_b200.h).
#include "cache_mma.cuh"

namespace ncmb {
namespace {

template <class E> __device__ __forceinline__ float get(const char *p, int d) { return (float)((const E *)p)[d]; }

// ---- mean keys ----
// One warp a block. A lane has 16 bytes of the dims of every R-th slot (R: rows of slots that the warp's lanes cover), CNT
// slots in all; sums by halves of the block are sums by halves of a lane's own slots first, then of the lanes' rows.
// Bound by reading the keys: 8 loads of 16 bytes a lane are in flight. 4 rows of 32768 tokens, 8 x 128 in bf16: 55 us (4.9 TB/s).
template <class KE> struct BsVec { static constexpr int N = 16 / sizeof(KE); };
template <class KE, int CNT>
__device__ __forceinline__ void bs_sum(float (&r)[16 / sizeof(KE)], const char *p, int64_t ts, int i, int step, int cnt) {
    constexpr int VE = BsVec<KE>::N;
    if constexpr (CNT <= 8) {
        uint4 raw[CNT];
#pragma unroll
        for (int j = 0; j < CNT; j++) raw[j] = i + step * j < cnt ? *(const uint4 *)(p + (i + step * j) * ts) : make_uint4(0, 0, 0, 0);
        float x[CNT][VE];
#pragma unroll
        for (int j = 0; j < CNT; j++) {
            const uint32_t u[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if constexpr (VE == 4) x[j][e] = __uint_as_float(u[e]);
                else { x[j][2 * e] = __uint_as_float(u[e] << 16); x[j][2 * e + 1] = __uint_as_float(u[e] & 0xffff0000u); }
            }
        }
#pragma unroll
        for (int h = CNT / 2; h > 0; h >>= 1)
#pragma unroll
            for (int j = 0; j < h; j++)
#pragma unroll
                for (int e = 0; e < VE; e++) x[j][e] = __fadd_rn(x[j][e], x[j + h][e]);
#pragma unroll
        for (int e = 0; e < VE; e++) r[e] = x[0][e];
    } else {
        float b[VE];
        bs_sum<KE, CNT / 2>(r, p, ts, i, 2 * step, cnt);
        bs_sum<KE, CNT / 2>(b, p, ts, i + step, 2 * step, cnt);
#pragma unroll
        for (int e = 0; e < VE; e++) r[e] = __fadd_rn(r[e], b[e]);
    }
}

template <class KE, int CNT>
__global__ void __launch_bounds__(256, CNT <= 16 ? 4 : CNT <= 32 ? 3 : 2) k_block_summaries(CacheDev c, int n_new, const int *first, int block, int nb, int upr_log, signed char *codes, float *scales) {
    constexpr int VE = BsVec<KE>::N;
    const int lane = threadIdx.x & 31, kvh = blockIdx.y, b = blockIdx.z;
    const int u = lane & ((1 << upr_log) - 1), tr = lane >> upr_log, R = block / CNT;
    pdl_wait();
    pdl_launch_dependents();
    const int n = cache_len(c, b, n_new) + n_new, f = first ? max(0, first[b]) : 0;
    const bool in = u * VE < c.hd && tr < R;
    const char *kb = c.k + b * c.rs + kvh * c.hs + u * 16;
    for (int64_t i = f / block + (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i * block < n; i += (int64_t)gridDim.x * 8) {
        const int s0 = (int)i * block, cnt = min(block, n - s0);
        float m[VE];
        bs_sum<KE, CNT>(m, kb + s0 * c.ts, c.ts, tr, R, in ? cnt : 0);
        for (int o = (R >> 1) << upr_log; o >= (1 << upr_log); o >>= 1)
#pragma unroll
            for (int e = 0; e < VE; e++) m[e] = __fadd_rn(m[e], __shfl_xor_sync(0xffffffffu, m[e], o));
        float top = 0.f;
#pragma unroll
        for (int e = 0; e < VE; e++) { m[e] = __fdiv_rn(m[e], (float)cnt); top = fmaxf(top, fabsf(m[e])); }
        if (!in) top = 0.f;
        for (int o = 1; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float sc = __fdiv_rn(top, 127.f);
        const int64_t at = ((int64_t)b * c.nkv + kvh) * nb + i;
        if (in && tr == 0) {
            uint32_t w[VE / 4];
#pragma unroll
            for (int x = 0; x < VE / 4; x++) {
                w[x] = 0;
#pragma unroll
                for (int e = 0; e < 4; e++) w[x] |= (sc > 0.f ? (uint32_t)(int)rintf(__fdiv_rn(m[4 * x + e], sc)) & 255u : 0u) << (8 * e);
            }
            uint32_t *p = (uint32_t *)(codes + at * c.hd + u * VE);
#pragma unroll
            for (int x = 0; x < VE / 4; x++) p[x] = w[x];
        }
        if (lane == 0) scales[at] = sc;
    }
}

template <class KE>
void run_summaries(const CacheDev &d, int n_new, const int *first, int block, int nb, int hint, signed char *codes, float *scales) {
    const int units = d.hd * (int)sizeof(KE) / 16;
    int ul = 0;
    while ((1 << ul) < units) ul++;
    const int rows = 32 >> ul, cnt = block / (rows < block ? rows : block);
    const dim3 grid((unsigned)std::max<int64_t>(1, cdiv(hint, 8)), d.nkv, d.rows);
    switch (cnt) {
#define BS_CASE(N) case N: LAUNCH_PDL((k_block_summaries<KE, N>), grid, 256, 0, d, n_new, first, block, nb, ul, codes, scales); break
        BS_CASE(1); BS_CASE(2); BS_CASE(4); BS_CASE(8); BS_CASE(16); BS_CASE(32); BS_CASE(64); BS_CASE(128);
#undef BS_CASE
    }
}

// ---- picks ----
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

constexpr int BP_THREADS = 512, BP_WARPS = BP_THREADS / 32, BP_MAXC = 8;
constexpr int BP_KEYS = 32768;       // keys a CTA holds in shared memory

__device__ __forceinline__ void mma_s8(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Picks of one (row, token, kv head), by a cluster of CTAs that each score a part of the blocks. Scores are integer products on
// m16n8k32 tiles -- 16 heads of the group against 8 blocks -- with the dims of a tile's k positions chosen so that a lane's
// codes are 8 bytes in a row (any order of the dims gives the same whole numbers). Bound by latency: the codes of 128K
// tokens in blocks of 64 are 128 KB a kv head.
template <class QE, bool CL>
__global__ void __launch_bounds__(BP_THREADS) k_block_pick(BlockArgs a) {
    namespace cg = cooperative_groups;
    extern __shared__ __align__(16) char dyn[];
    __shared__ SelShared sel;
    __shared__ int wtie[BP_WARPS], wkeep[BP_WARPS], share[2];
    cg::cluster_group cl = cg::this_cluster();
    const int rank = CL ? (int)cl.block_rank() : 0, nc = CL ? (int)cl.num_blocks() : 1;
    const int t = blockIdx.x / nc, kvh = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, hd = a.c.hd;
    pdl_wait();
    pdl_launch_dependents();
    const int cur = (cache_len(a.c, b, a.T) + t) / a.block, n = cur + 1, k = min(n, a.n_sel);
    const int64_t u = ((int64_t)b * a.T + t) * a.c.nkv + kvh;
    int *picks = a.picks + u * a.n_sel;
    if (rank == 0) for (int i = k + tid; i < a.n_sel; i += BP_THREADS) picks[i] = -1;
    if (n <= a.n_sel) {
        if (rank == 0) for (int i = tid; i < n; i += BP_THREADS) picks[i] = i;
        return;                                                              // all CTAs of the cluster
    }
    // queries in 8 bits, heads in whole tiles of 16, dims in whole 32
    const int gt = (a.G + 15) / 16, hp = (hd + 31) & ~31;
    float *qs = (float *)dyn;                                                // [16 gt]
    signed char *q8 = (signed char *)(qs + 16 * gt);                         // [16 gt][hp + 8]: rows 8 bytes apart in banks
    const int qrow = hp + 8;
    for (int g = warp; g < 16 * gt; g += BP_WARPS) {
        const char *q = a.q + ((int64_t)b * a.T + t) * a.ldq + (int64_t)(kvh * a.G + g) * hd * sizeof(QE);
        float v[4], top = 0.f;
#pragma unroll
        for (int x = 0; x < 4; x++) { v[x] = g < a.G && lane + 32 * x < hd ? get<QE>(q, lane + 32 * x) : 0.f; top = fmaxf(top, fabsf(v[x])); }
#pragma unroll
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float sc = __fdiv_rn(top, 127.f);
        if (lane == 0) qs[g] = sc;
#pragma unroll
        for (int x = 0; x < 4; x++)
            if (32 * x < hp) q8[g * qrow + lane + 32 * x] = sc > 0.f ? (signed char)(int)rintf(__fdiv_rn(v[x], sc)) : 0;
    }
    __syncthreads();
    const int per = ((n + nc - 1) / nc + 31) & ~31, lo = min(n, rank * per), hi = min(n, lo + per);
    uint32_t *keys = a.keys ? a.keys + u * a.nb + lo : (uint32_t *)(q8 + 16 * gt * qrow);
    const signed char *codes = a.codes + ((int64_t)b * a.c.nkv + kvh) * a.nb * hd;
    const float *scales = a.scales + ((int64_t)b * a.c.nkv + kvh) * a.nb;
    const int g4 = lane >> 2, c4 = lane & 3;
    // A tile of 8 blocks a warp at a time, the next one's codes on their way. Not unrolled: the whole of it runs a few times only, and
    // code that runs once is paced by instruction fetches (four tiles at once: 13000 cycles for 512 blocks of 128 dims).
    int2 ahead[4];
    float scale_ahead;
    auto fetch = [&](int i0) {
        const int i = i0 + g4, j = i0 + 2 * c4 + (g4 & 1);
#pragma unroll
        for (int s = 0; s < 4; s++) {
            ahead[s] = make_int2(0, 0);
            if (32 * s + 8 * c4 < hd && i < hi) ahead[s] = *(const int2 *)(codes + (int64_t)i * hd + 32 * s + 8 * c4);
        }
        scale_ahead = j < hi ? scales[j] : 0.f;
    };
    fetch(lo + warp * 8);
#pragma unroll 1
    for (int i0 = lo + warp * 8; i0 < hi; i0 += BP_WARPS * 8) {
        int2 cd[4];
#pragma unroll
        for (int s = 0; s < 4; s++) cd[s] = ahead[s];
        const float block_scale = scale_ahead;
        fetch(i0 + BP_WARPS * 8);
        float best[2] = {-INFINITY, -INFINITY};
#pragma unroll 1
        for (int tt = 0; tt < gt; tt++) {
            int dot[4] = {0, 0, 0, 0};
            const signed char *q = q8 + (16 * tt + g4) * qrow + 8 * c4;
#pragma unroll
            for (int s = 0; s < 4; s++) {
                if (32 * s >= hd) break;
                const uint2 q0 = *(const uint2 *)(q + 32 * s), q1 = *(const uint2 *)(q + 8 * qrow + 32 * s);
                const uint32_t qa[4] = {q0.x, q1.x, q0.y, q1.y};
                mma_s8(dot, qa, (uint32_t)cd[s].x, (uint32_t)cd[s].y);
            }
#pragma unroll
            for (int hh = 0; hh < 2; hh++) {
                const int g = 16 * tt + g4 + 8 * hh;
                const float sc = qs[g];
#pragma unroll
                for (int e = 0; e < 2; e++) if (g < a.G) best[e] = fmaxf(best[e], __fmul_rn((float)dot[2 * hh + e], sc));
            }
        }
#pragma unroll
        for (int o = 4; o < 32; o <<= 1)
#pragma unroll
            for (int e = 0; e < 2; e++) best[e] = fmaxf(best[e], __shfl_xor_sync(0xffffffffu, best[e], o));
        const int i = i0 + 2 * c4 + (g4 & 1);                                // lanes with g4 = 0, 1 have a block each
        if (g4 < 2 && i < hi) {
            const bool always = i < a.n_first || i > cur - a.n_last;
            keys[i - lo] = always ? 0xffffffffu : float_key(__fmul_rn(g4 ? best[1] : best[0], block_scale));
        }
    }
    __syncthreads();
    uint32_t ties;
    const uint32_t bound = select_kth<BP_THREADS, CL>(sel, hi - lo, (uint32_t)k, ties, [&](int i) { return keys[i]; });
    const int part = ((hi - lo + BP_THREADS - 1) / BP_THREADS) * 32, w0 = min(hi - lo, warp * part), w1 = min(hi - lo, w0 + part);
    int nt = 0, above = 0;
#pragma unroll 1
    for (int s = w0; s < w1; s += 32) {
        const uint32_t x = s + lane < w1 ? keys[s + lane] : 0;
        nt += __popc(__ballot_sync(0xffffffffu, s + lane < w1 && x == bound));
        above += __popc(__ballot_sync(0xffffffffu, s + lane < w1 && x > bound));
    }
    if (lane == 0) { wtie[warp] = nt; wkeep[warp] = above; }
    __syncthreads();
    const int vt = lane < BP_WARPS ? wtie[lane] : 0, vk = lane < BP_WARPS ? wkeep[lane] : 0;
    int tb = __reduce_add_sync(0xffffffffu, lane < warp ? vt : 0), at = __reduce_add_sync(0xffffffffu, lane < warp ? vk : 0);
    if constexpr (CL) {
        if (warp == 0) {
            const int x = __reduce_add_sync(0xffffffffu, vt), y = __reduce_add_sync(0xffffffffu, vk);
            if (lane == 0) { share[0] = x; share[1] = y; }
        }
        cl.sync();
        tb += __reduce_add_sync(0xffffffffu, lane < rank ? *cl.map_shared_rank(&share[0], lane) : 0);
        at += __reduce_add_sync(0xffffffffu, lane < rank ? *cl.map_shared_rank(&share[1], lane) : 0);
    }
    at += (int)min((uint32_t)tb, ties);          // ties before this warp: tb; picks before it: at
#pragma unroll 1
    for (int s = w0; s < w1; s += 32) {
        const bool in = s + lane < w1;
        const uint32_t x = in ? keys[s + lane] : 0, lt = (1u << lane) - 1;
        const uint32_t tm = __ballot_sync(0xffffffffu, in && x == bound);
        const bool keep = in && (x > bound || (x == bound && (uint32_t)(tb + __popc(tm & lt)) < ties));
        const uint32_t km = __ballot_sync(0xffffffffu, keep);
        if (keep) picks[at + __popc(km & lt)] = lo + s + lane;
        at += __popc(km);
        tb += __popc(tm);
    }
    if constexpr (CL) cl.sync();                 // the others have read this CTA's counts
}

template <class QE>
void run_pick(const BlockArgs &a, int nc, size_t smem) {
    auto kernel = nc > 1 ? k_block_pick<QE, true> : k_block_pick<QE, false>;
    if (smem > 20000) CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    cache_launch(kernel, dim3(a.T * nc, a.c.nkv, a.c.rows), BP_THREADS, smem, nc, a);
}

template <class KE, class QE>
int run_blocks(const char *who, const CmArgs &a, int max_keys, const BlockArgs &picks, int nc, size_t smem) {
    auto first = [&] { run_pick<QE>(picks, nc, smem); };
    if (a.c.hd <= 64) return a.M <= 8 ? cm_run_as<KE, QE, 64, 8, true>(who, a, max_keys, first) : cm_run_as<KE, QE, 64, 16, true>(who, a, max_keys, first);
    return a.M <= 8 ? cm_run_as<KE, QE, 128, 8, true>(who, a, max_keys, first) : cm_run_as<KE, QE, 128, 16, true>(who, a, max_keys, first);
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
    if (max_len <= 0 || max_len > c->capacity - n_new) max_len = c->capacity - n_new;
    const int hint = (int)cdiv((int64_t)max_len + n_new, block);
    ProfScope prof(NCMB_K_ATTN, 0, (double)c->rows * c->n_kv * hint * block * c->hd * cache_elem(c));
    if (c->type == NCMB_F32) run_summaries<float>(d, n_new, first, block, nb, hint, codes, scales);
    else run_summaries<__nv_bfloat16>(d, n_new, first, block, nb, hint, codes, scales);
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
    if (max_len <= 0 || max_len > c->capacity - T) max_len = c->capacity - T;
    ProfScope prof(NCMB_K_ATTN, 4.0 * units * a.G * c->hd * n_sel * block, 2.0 * units * n_sel * block * c->hd * cache_elem(c));
    // CTAs a (row, token, head): as many as keep the GPU busy, with 512 blocks each at least. One row of 2047 blocks, the whole call:
    // with 256 / 512 / 1024 / 2048 blocks a CTA 20.0 / 18.1 / 20.3 / 24.4 us.
    int nc = 1;
    while (nc < BP_MAXC && units * nc * 2 <= ctx().sm_count && cdiv(cdiv(max_len, block), nc) > 512) nc *= 2;
    const int64_t per = (cdiv(a.nb, nc) + 31) & ~31;
    const size_t need_picks = picks ? 0 : (size_t)units * n_sel * 4, need_keys = per > BP_KEYS ? (size_t)units * a.nb * 4 : 0;
    char *scratch = need_picks + need_keys ? (char *)cache_scratch(who, need_picks + need_keys, SCRATCH_PICKS) : nullptr;
    if (need_picks + need_keys && !scratch) return -1;
    a.picks = picks ? picks : (int *)(scratch + need_keys);
    a.keys = need_keys ? (uint32_t *)scratch : nullptr;
    const int gt = (a.G + 15) / 16;
    const size_t smem = (size_t)gt * 16 * (4 + ((c->hd + 31) & ~31) + 8) + (need_keys ? 0 : (size_t)per * 4);
    if (smem > 190000) return cache_refuse(who, "%d query heads a kv head", a.G);
    CmArgs m = {};
    m.c = a.c; m.q = a.q; m.out = a.out; m.ldq = a.ldq; m.ldo = a.ldo; m.H = a.H; m.G = a.G; m.T = T; m.M = a.G;
    m.c2 = a.scale * 1.44269504f; m.block_log = block == 16 ? 4 : block == 32 ? 5 : block == 64 ? 6 : 7; m.n_sel = n_sel; m.picks = a.picks;
    const int keys = (int)std::min<int64_t>(max_len + T, (int64_t)n_sel * block);
    if (c->type == NCMB_F32) return run_blocks<float, float>(who, m, keys, a, nc, smem);
    if (act_type == NCMB_F32) return run_blocks<__nv_bfloat16, float>(who, m, keys, a, nc, smem);
    return run_blocks<__nv_bfloat16, __nv_bfloat16>(who, m, keys, a, nc, smem);
}
