// Attention of many query rows (trees, runs of tokens, several heads a kv head) to cached keys on tcgen05 tiles: the wide
// variant of cache_mma.cuh, for ncmb_cache_attention.
//
// A CTA has 128 query rows of a kv head and walks tiles of 128 keys: S = Q K^T into tensor memory, softmax with a running
// maximum by 256 threads (two a row, 64 keys each), the probabilities back into tensor memory as the next product's operand,
// O = P V of the tile into tensor memory, added to the running result in registers in fp32. Operands are bf16 terms, as in
// cache_mma.cuh: a query is 3 (bf16 activations: 1), a probability 3 (2), a bf16 key or value 1, an fp32 one 3, of whose nine
// products the six largest are taken (2^-24 and more). Roles: warps 0 - 7 softmax (they also turn the queries into terms and
// write the results), warp 8 issues the MMAs, the others load: keys of the next tile, values of this one, in turn through
// one ring -- bf16 by TMA, the last tiles of a row, which end inside, by cp.async; fp32 through registers, where the terms are formed.
//
// Tiles are 128 keys wide and probabilities stand in tensor memory because MMAs are paced by operand fetch: 64-wide ones took about
// 100 cycles each with both operands in shared memory, 128-wide ones 90 with A in tensor memory (arithmetic: 16 and 32). Bound by
// the chain of a tile: products with the values, then the exponentials of the next tile, which wait for the tensor memory that
// the products read: 3900 cycles for 64 KB of keys and values at head dim 128. 16 rows of up to 8192 tokens, 32 heads over 8 x
// 128, 16 drafted tokens: 107 us, of which 51 are the time the bytes take (64-key tiles by cp.async: 179).
#pragma once
#include "cache_mma.cuh"
#include "tc_common.cuh"

namespace ncmb {

template <class KE, class QE, int HDP_> struct CtCfg {
    static constexpr bool BF = sizeof(KE) == 2;
    static constexpr int HDP = HDP_, ATOMS = HDP / 64, M = 128, KT = 128;
    static constexpr int NQ = sizeof(QE) == 4 ? 3 : 1, NP = sizeof(QE) == 4 ? 3 : 2, NK = BF ? 1 : 3;
    static constexpr int KATOM = KT * 128, QATOM = M * 128;          // bytes of 64 dims of the keys, of the queries
    static constexpr int STAGE = NK * ATOMS * KATOM, QB = NQ * ATOMS * QATOM;        // a stage: a tile's keys or its values
    static constexpr int FIT = (217 * 1024 - QB) / STAGE, NST = FIT < 8 ? FIT : 8;
    static constexpr int PG = 3, PW = BF ? PG : 2 * PG, SW = 8, THREADS = 32 * (SW + 1 + PW);    // whole warps a scheduler: registers
    static constexpr int SMEM = QB + NST * STAGE + 1024;
    // What the start of a unit costs, in tiles, for the plan: queries, the first loads and the results take about 9 us, a tile 2
    // (bf16) or 7 (fp32: forming the terms). Without it the CTA that gets a short row's heads is the last: 125 -> 100 us.
    static constexpr int START = BF ? 4 : 1;
    // columns of tensor memory: probabilities (two to a column), context, one or two score tiles
    static constexpr int PCOL = 0, OCOL = NP * 64, SCOL = OCOL + HDP, NSB = SCOL + 256 <= 512 ? 2 : 1;
};

// Query rows of a kv head that the wide tiles take: beyond some 5 million their division by the heads of a group, in fp32, is not exact.
constexpr int CT_MOST_ROWS = 1 << 20;

__host__ __device__ constexpr uint32_t umma_idesc_bf16(int M, int N) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
// Every wait is bounded. The warps of the softmax, which meet at barriers of their own, go on without waiting once one has run out;
// whoever starts copies or MMAs starts no more, and nobody leaves before those under way have ended (or a limit has passed).
struct CtWait {
    int *err, *any;                  // any: in shared memory, for the whole CTA
    bool dead;
    __device__ __forceinline__ void operator()(uint32_t bar, uint32_t parity, int code) {
        if (!dead && !mbar_wait(bar, parity, err, code)) { dead = true; *any = 1; }
    }
};
// the same MMA with A in tensor memory (16-bit elements, two to a column)
__device__ __forceinline__ void umma_f16_ta(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(tmem_d), "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&w)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"r"(taddr), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 "
                 "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\ttcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr) : "memory");
}
__device__ __forceinline__ void ct_tma(uint32_t dst, const CUtensorMap *m, int d, int slot, int head, int row, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 ::"r"(dst), "l"(m), "r"(d), "r"(slot), "r"(head), "r"(row), "r"(bar) : "memory");
}
__device__ __forceinline__ void ct_fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

template <class KE, class QE, int HDP>
__global__ void __launch_bounds__(CtCfg<KE, QE, HDP>::THREADS, 1) k_cache_attention_tc(const __grid_constant__ CmArgs a, const __grid_constant__ CUtensorMap mk,
                                                                                        const __grid_constant__ CUtensorMap mv, int *err) {
    using F = CtCfg<KE, QE, HDP>;
    constexpr int M = F::M, KT = F::KT, NST = F::NST, ATOMS = F::ATOMS;
    extern __shared__ char smem_raw[];
    char *smem = (char *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    char *qs = smem, *ring = qs + F::QB;
    __shared__ uint64_t bars[2 * 8 + 8];                             // stages full, stages free, see below
    __shared__ uint32_t tmem_at;
    __shared__ int plan[4];                                          // total, per, item, where it begins
    __shared__ float xm[2][2][M], xl[2][M];
    __shared__ uint32_t node_bits[M][8], place_bits[F::PW][8];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, hd = a.c.hd, G = a.G;
    auto full = [&](int s) { return cm_smem(&bars[s]); };
    auto empty = [&](int s) { return cm_smem(&bars[8 + s]); };
    const uint32_t bar_q = cm_smem(&bars[16]), bar_s = cm_smem(&bars[17]), bar_p = cm_smem(&bars[19]), bar_pv = cm_smem(&bars[20]);
    const uint32_t bar_sf = cm_smem(&bars[21]);                      // queries ready, scores ready (2), probabilities ready, context ready, scores read
    const uint32_t bar_done = cm_smem(&bars[22]);                    // all MMAs are done
    pdl_wait();
    pdl_launch_dependents();
    __shared__ int s_abort;
    if (tid == 0) {
        s_abort = *(volatile int *)err;                              // a wait ran out earlier: nothing more is started
        for (int s = 0; s < NST; s++) { mbar_init(full(s), F::PG); mbar_init(empty(s), 1); }
        mbar_init(bar_q, F::SW); mbar_init(bar_s, 1); mbar_init(bar_s + 8, 1); mbar_init(bar_p, F::SW); mbar_init(bar_pv, 1); mbar_init(bar_sf, F::SW); mbar_init(bar_done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        // the plan of cache_mma.cuh, by one warp; a unit counts as F::START tiles more than it has
        int t = 0;
        auto places = [&](int i) { return i < a.items ? ((cm_keys<false>(a, i) + KT - 1) / KT + F::START) * a.c.nkv * a.tiles : 0; };
        for (int i = lane; i < a.items; i += 32) t += places(i);
        t = __reduce_add_sync(0xffffffffu, t);
        const int per = (unsigned)(t + (int)gridDim.x - 1) / gridDim.x, x = (int)min((int64_t)blockIdx.x * per, (int64_t)t);
        int before = 0, item = 0, begin = 0;
        for (int i0 = 0; i0 < a.items; i0 += 32) {
            const int mine = places(i0 + lane);
            int inc = mine;
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += v;
            }
            const int from = before + inc - mine;
            const uint32_t hit = __ballot_sync(0xffffffffu, x >= from && x < from + mine);
            if (hit) { const int w = __ffs(hit) - 1; item = i0 + w; begin = __shfl_sync(0xffffffffu, from, w); break; }
            before = __shfl_sync(0xffffffffu, before + inc, 31);
        }
        if (lane == 0) { plan[0] = t; plan[1] = per; plan[2] = item; plan[3] = begin; }
    }
    __syncthreads();
    if (s_abort || (int64_t)blockIdx.x * plan[1] >= plan[0]) return;
    if (warp == F::SW) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(cm_smem(&tmem_at)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_at;
    CtWait wait{err, &s_abort, false};

    struct Unit { int item, kvh, m0, first, stop, unit, n, len, row; bool whole; };
    int at = blockIdx.x * plan[1], item = plan[2], item_at = plan[3];
    const int end = min(plan[0], at + plan[1]);
    auto next_unit = [&](Unit &u) {                                  // the run's next unit with tiles in it, or false
        while (at < end) {
            u.n = cm_keys<false>(a, item);
            const int nch = (u.n + KT - 1) / KT, span = nch + F::START, sub = cm_div(at - item_at, span), kvh = a.tiles == 1 ? sub : cm_div(sub, a.tiles);
            const int into = at - item_at - sub * span, take = min(span - into, end - at);
            u.item = item; u.kvh = kvh; u.m0 = (sub - kvh * a.tiles) * M;
            u.first = max(0, into - F::START); u.stop = into + take - F::START;
            u.unit = item * a.c.nkv * a.tiles + sub;
            u.len = u.n - a.T; u.row = a.row0 + item; u.whole = u.first == 0 && u.stop == nch;
            at += take;
            if (at == item_at + span * a.c.nkv * a.tiles) { item_at = at; item++; }
            if (u.stop > u.first) return true;
        }
        return false;
    };
    Unit u;
    uint32_t it = 0, un = 0, items = 0;                              // tiles, units, stages (two a tile) so far

    if (warp < F::SW) {
        // ================= softmax: row r of the tile, keys 64 hf ... of a key tile, half hf of the dims =================
        const int r = (warp & 3) * 32 + lane, hf = warp >> 2;
        const uint32_t tl = tmem + ((uint32_t)(warp & 3) << 21);     // this warp's 32 lanes of tensor memory
        constexpr int HC = HDP / 2;
        const float c2 = fabsf(a.c2);                                // a negative scale goes into the queries
        auto group_sync = [] { asm volatile("bar.sync 1, %0;" ::"n"(F::SW * 32) : "memory"); };
        while (next_unit(u)) {
            const int *par = a.parents ? a.parents + (int64_t)u.row * a.T : nullptr;
            // queries as terms (the MMAs that read the last unit's are done: their scores have been read)
            constexpr int QU = HDP / 8, QR = F::SW * 32 / QU, AHEAD = 4;     // units of 8 dims a row, rows a step, rows a thread loads at once
            const int d0 = tid % QU * 8;
            const float per_g = 1.0f / (float)G;
#pragma unroll 1
            for (int m1 = tid / QU; m1 < M; m1 += QR * AHEAD) {
                float4 raw[AHEAD][sizeof(QE) / 2];
#pragma unroll
                for (int i = 0; i < AHEAD; i++) {
                    const int mm = u.m0 + m1 + i * QR, t = (int)(((float)mm + 0.5f) * per_g), h = u.kvh * G + mm - t * G;     // mm / G, right below CT_MOST_ROWS + M
                    const char *p = a.q + ((int64_t)u.row * a.T + t) * a.ldq + ((int64_t)h * hd + d0) * sizeof(QE);
                    const bool ok = mm < a.M && d0 < hd && cm_used(par, t);
#pragma unroll
                    for (int x = 0; x < (int)sizeof(QE) / 2; x++) raw[i][x] = ok ? *(const float4 *)(p + 16 * x) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
#pragma unroll
                for (int i = 0; i < AHEAD; i++) {
                    const int m = m1 + i * QR;
                    float x[8];
                    if constexpr (sizeof(QE) == 4) {
                        *(float4 *)&x[0] = raw[i][0];
                        *(float4 *)&x[4] = raw[i][1];
                    } else {
                        const float w[4] = {raw[i][0].x, raw[i][0].y, raw[i][0].z, raw[i][0].w};
#pragma unroll
                        for (int e = 0; e < 4; e++) { const float2 f = cm_unpack(__float_as_uint(w[e])); x[2 * e] = f.x; x[2 * e + 1] = f.y; }
                    }
                    if (a.c2 < 0.f) {
#pragma unroll
                        for (int e = 0; e < 8; e++) x[e] = -x[e];
                    }
#pragma unroll
                    for (int k = 0; k < F::NQ; k++) {
                        uint32_t w[4];
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            w[e] = cm_pack(x[2 * e], x[2 * e + 1]);
                            const float2 f = cm_unpack(w[e]);
                            x[2 * e] -= f.x; x[2 * e + 1] -= f.y;
                        }
                        *(uint4 *)(qs + (k * ATOMS + d0 / 64) * F::QATOM + m * 128 + ((((d0 & 63) / 8) ^ (m & 7)) * 16)) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
            }
            const int mm = u.m0 + r, node = min(mm, a.M - 1) / G;
            const bool row_used = mm < a.M && cm_used(par, node);
            const bool busy = u.m0 + (warp & 3) * 32 < a.M;          // the warp has rows: else it only keeps the others' time
            const int tiles = u.stop - u.first;
            if (u.stop * KT > u.len && hf == 0) {                    // what the row's node sees of the new tokens
#pragma unroll 1
                for (int w = 0; w < 8; w++) node_bits[r][w] = par ? 0u : node >= 32 * w + 31 ? 0xffffffffu : node >= 32 * w ? (2u << (node - 32 * w)) - 1 : 0u;
#pragma unroll 1
                for (int x = par ? node : -1; x >= 0 && cm_used(par, x); x = par[x]) node_bits[r][x >> 5] |= 1u << (x & 31);
            }
            ct_fence_async();
            group_sync();
            if (lane == 0) mbar_arrive(bar_q);
            float O[HC], mx = -INFINITY, l = 0.f, al_prev = 0.f;
            bool skip = false;                                       // the last tile's context has been added already
#pragma unroll
            for (int d = 0; d < HC; d++) O[d] = 0.f;
            auto add_context = [&]() {                               // of the tile before
                wait(bar_pv, (it - 1) & 1u, 41);
                tc_fence_after();
                if (skip || !busy) { skip = false; return; }
#pragma unroll
                for (int x = 0; x < HC; x += 32) {
                    uint32_t o[32];
                    tmem_ld32(tl + (uint32_t)(F::OCOL + hf * HC + x), o);
#pragma unroll
                    for (int d = 0; d < 32; d++) O[x + d] = fmaf(O[x + d], al_prev, __uint_as_float(o[d]));
                }
            };
            for (int t = u.first; t < u.stop; t++, it++) {
                const uint32_t sb = F::NSB == 2 ? it & 1u : 0u, scol = tl + (uint32_t)F::SCOL + sb * 128u + (uint32_t)hf * 64u;
                wait(bar_s + 8 * sb, F::NSB == 2 ? (it >> 1) & 1u : it & 1u, 42);
                tc_fence_after();
                const int p0 = t * KT + 64 * hf;
                const bool masked = (t + 1) * KT > u.len;
                auto sees = [&](int from) {                          // bit j: the row sees slot from + j
                    uint32_t see = 0xffffffffu;
                    const int rel = from - u.len;                    // node of the first slot
                    if (rel > -32) {
                        uint32_t lo = 0, hi = 0;
                        const int w = rel < 0 ? -1 : rel >> 5;
                        if (w >= 0 && w < 8) lo = node_bits[r][w];
                        if (w < 0) lo = 0xffffffffu;                 // slots of the cache
                        if (w + 1 < 8) hi = node_bits[r][w + 1];
                        see = __funnelshift_r(lo, hi, rel & 31);
                    }
                    if (u.n - from < 32) see &= u.n > from ? (1u << (u.n - from)) - 1 : 0u;
                    return see;
                };
                // the maximum, then -- the scores are read again rather than kept: registers -- exponentials
                float top = -INFINITY;
                if (busy) {
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        uint32_t sr[32];
                        tmem_ld32(scol + 32u * c, sr);
                        if (masked) {
                            const uint32_t see = sees(p0 + 32 * c);
#pragma unroll
                            for (int j = 0; j < 32; j++) if (!((see >> j) & 1u)) sr[j] = 0xff800000u;
                        }
#pragma unroll
                        for (int j = 0; j < 32; j++) top = fmaxf(top, __uint_as_float(sr[j]));
                        if (a.scores && mm < a.M) {
                            float *sp = a.scores + (((int64_t)u.item * a.c.nkv + u.kvh) * a.M + mm) * a.pitch + p0 + 32 * c;
                            // No token, no share: such a row's scores are zeros by keys that may hold anything. (A NaN of another row becomes
                            // an infinity, which its sum, a NaN too, makes a NaN again.)
                            const float most = row_used ? INFINITY : -INFINITY;
                            auto score = [&](int j) { return fminf(__uint_as_float(sr[j]) * c2, most); };
#pragma unroll
                            for (int j = 0; j < 32; j += 4) *(float4 *)(sp + j) = make_float4(score(j), score(j + 1), score(j + 2), score(j + 3));
                        }
                    }
                }
                xm[it & 1u][hf][r] = top;
                group_sync();
                top = fmaxf(mx, fmaxf(top, xm[it & 1u][hf ^ 1][r]) * c2);
                const float base = top == -INFINITY ? 0.f : top, al = cm_exp2(mx - base);
                mx = top;
                if (t > u.first) add_context();                      // also: the MMAs that read the last probabilities are done
                al_prev = al;
                if (busy) {
                    float sum = 0.f;
#pragma unroll
                    for (int c = 0; c < 4; c++) {                    // 16 keys at a time (more, or some before the wait: spills, 125 -> 167 us)
                        uint32_t sr[16];
                        tmem_ld16(scol + 16u * c, sr);
                        if (masked) {
                            const uint32_t see = sees(p0 + 16 * c);
#pragma unroll
                            for (int j = 0; j < 16; j++) if (!((see >> j) & 1u)) sr[j] = 0xff800000u;
                        }
                        float s[16];
#pragma unroll
                        for (int j = 0; j < 16; j++) { s[j] = cm_exp2(fmaf(__uint_as_float(sr[j]), c2, -base)); sum += s[j]; }
#pragma unroll
                        for (int k = 0; k < F::NP; k++) {
                            uint32_t w[8];
#pragma unroll
                            for (int e = 0; e < 8; e++) {
                                w[e] = cm_pack(s[2 * e], s[2 * e + 1]);
                                if (k + 1 < F::NP) {
                                    const float2 f = cm_unpack(w[e]);
                                    s[2 * e] -= f.x; s[2 * e + 1] -= f.y;
                                }
                            }
                            tmem_st8(tl + (uint32_t)(F::PCOL + k * 64 + hf * 32 + c * 8), w);
                        }
                    }
                    l = l * al + sum;
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                }
                if (F::NSB == 1) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar_sf);
                }
                if (masked) {
                    // An infinity or NaN among values that not every row sees must not be multiplied by zero: such a tile's context is
                    // formed here, one key at a time, before the stage is given to the MMAs (whose result is then left out).
                    const uint32_t at_v = items + (t + 1 < u.stop ? 2 + 2 * (t - u.first) : 2 * tiles - 1), st = at_v % NST;
                    wait(full(st), (at_v / NST) & 1u, 43);
                    const char *vt = ring + st * F::STAGE;
                    bool odd = false;
#pragma unroll 1
                    for (int i = tid; i < F::STAGE / 4; i += F::SW * 32) {
                        const uint32_t w = ((const uint32_t *)vt)[i];
                        odd |= (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
                    }
                    uint32_t any;
                    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                                 : "=r"(any) : "r"((uint32_t)odd), "n"(F::SW * 32) : "memory");
                    if (any) {
                        tc_fence_before();
                        group_sync();                                // the other half's probabilities are in tensor memory
                        tc_fence_after();
                        if (busy) {
#pragma unroll
                            for (int d = 0; d < HC; d++) O[d] *= al;
#pragma unroll 1
                            for (int j = 0; j < KT; j += 2) {
                                float p2[2] = {0.f, 0.f};
#pragma unroll
                                for (int k = F::NP - 1; k >= 0; k--) {
                                    uint32_t w;
                                    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];\n\ttcgen05.wait::ld.sync.aligned;"
                                                 : "=r"(w) : "r"(tl + (uint32_t)(F::PCOL + k * 64 + j / 2)) : "memory");
                                    const float2 f = cm_unpack(w);
                                    p2[0] += f.x; p2[1] += f.y;
                                }
#pragma unroll 1
                                for (int e = 0; e < 2; e++) {
                                    const float p = e ? p2[1] : p2[0];
                                    if (p == 0.f) continue;
                                    const int key = j + e;
#pragma unroll
                                    for (int d = 0; d < HC; d++) {
                                        const int dd = hf * HC + d;
                                        float v = 0.f;
#pragma unroll
                                        for (int k = F::NK - 1; k >= 0; k--)
                                            v += (float)*(const __nv_bfloat16 *)(vt + (k * ATOMS + dd / 64) * F::KATOM + key * 128 + ((((dd & 63) / 8) ^ (key & 7)) * 16) + (dd & 7) * 2);
                                        O[d] = fmaf(p, v, O[d]);
                                    }
                                }
                                __syncwarp();
                            }
                        }
                        skip = true;
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar_p);
            }
            items += 2 * tiles;
            add_context();
            xl[hf][r] = l;
            if (hf == 0 && r == 0) {
                if (u.first == 0) a.range[u.unit].x = blockIdx.x;
                if (u.stop * KT >= u.n) a.range[u.unit].y = blockIdx.x;
            }
            group_sync();
            l += xl[hf ^ 1][r];
            float *sums = a.sums + ((int64_t)blockIdx.x + u.unit) * (2 * M);
            if (hf == 0) { sums[r] = mx; sums[M + r] = l; }
            if (mm < a.M) {
                if (u.whole) {
                    const float f = l > 0.f ? 1.f / l : 0.f;
                    if (!row_used) {                                 // not by f = 0: values may hold infinities
#pragma unroll
                        for (int d = 0; d < HC; d++) O[d] = 0.f;
                    }
                    QE *o = (QE *)(a.out + ((int64_t)u.row * a.T + node) * a.ldo) + (int64_t)(u.kvh * G + mm - node * G) * hd + hf * HC;
#pragma unroll
                    for (int d = 0; d < HC; d += 4) {
                        if (hf * HC + d >= hd) continue;
                        if constexpr (sizeof(QE) == 4) *(float4 *)(o + d) = make_float4(O[d] * f, O[d + 1] * f, O[d + 2] * f, O[d + 3] * f);
                        else *(uint2 *)(o + d) = make_uint2(cm_pack(O[d] * f, O[d + 1] * f), cm_pack(O[d + 2] * f, O[d + 3] * f));
                    }
                } else {
                    float *o = a.ctx + (2 * (int64_t)blockIdx.x + (u.first == 0)) * (M * HDP) + r * HDP + hf * HC;
#pragma unroll
                    for (int d = 0; d < HC; d += 4) *(float4 *)(o + d) = make_float4(O[d], O[d + 1], O[d + 2], O[d + 3]);
                }
            }
        }
    } else if (warp == F::SW) {
        // ================= MMAs =================
        if (lane == 0) {
            constexpr uint32_t ids = umma_idesc_bf16(M, KT), idv = umma_idesc_bf16(M, HDP) | (1u << 16);     // values: MN-major
            constexpr uint64_t QA = F::QATOM / 16, KA = F::KATOM / 16, ST = F::STAGE / 16;
            const uint64_t qd = umma_desc_sw128(cm_smem(qs)), rd = umma_desc_sw128(cm_smem(ring));
            const uint64_t rv = (rd & ~((uint64_t)0x3fff << 16)) | KA << 16;         // from 64 dims of the values to the next
            auto scores = [&](uint32_t i) {
                const uint32_t st = items % NST, sb = F::NSB == 2 ? i & 1u : 0u;
                wait(full(st), (items / NST) & 1u, 44);
                if (wait.dead) return;
                tc_fence_after();
                uint32_t acc = 0;
                const uint64_t kd = rd + st * ST;
#pragma unroll 1
                for (int sum = F::NQ + F::NK - 2 < 2 ? F::NQ + F::NK - 2 : 2; sum >= 0; sum--)       // small products first
#pragma unroll 1
                    for (int qk = 0; qk <= sum; qk++) {              // one term of the queries by one of the keys
                        const int kk = sum - qk;
                        if (qk >= F::NQ || kk >= F::NK) continue;
#pragma unroll
                        for (int x = 0; x < ATOMS; x++)
#pragma unroll
                            for (int k = 0; k < 4; k++) {
                                umma_f16(tmem + F::SCOL + sb * 128u, qd + (qk * ATOMS + x) * QA + k * 2, kd + (kk * ATOMS + x) * KA + k * 2, ids, acc);
                                acc = 1;
                            }
                    }
                umma_commit(bar_s + 8 * sb);
                umma_commit(empty(st));
                items++;
            };
            while (!wait.dead && next_unit(u)) {
                wait(bar_q, un & 1u, 45);
                un++;
                tc_fence_after();
                const int tiles = u.stop - u.first;
                if (!wait.dead) scores(it);
#pragma unroll 1
                for (int t = 0; t < tiles; t++, it++) {
                    if (t + 1 < tiles) {
                        if (F::NSB == 1) { wait(bar_sf, it & 1u, 48); tc_fence_after(); }
                        if (!wait.dead) scores(it + 1);
                    }
                    const uint32_t st = items % NST;
                    wait(full(st), (items / NST) & 1u, 49);
                    wait(bar_p, it & 1u, 46);
                    if (wait.dead) break;
                    tc_fence_after();
                    const uint64_t vd = rv + st * ST;
                    uint32_t acc = 0;
#pragma unroll 1
                    for (int sum = F::NP + F::NK - 2 < 2 ? F::NP + F::NK - 2 : 2; sum >= 0; sum--)
#pragma unroll 1
                        for (int pk = 0; pk <= sum; pk++) {
                            if (pk >= F::NP || sum - pk >= F::NK) continue;
#pragma unroll
                            for (int k = 0; k < KT / 16; k++) {
                                umma_f16_ta(tmem + F::OCOL, tmem + F::PCOL + pk * 64 + k * 8, vd + (sum - pk) * ATOMS * KA + k * 128, idv, acc);
                                acc = 1;
                            }
                        }
                    umma_commit(bar_pv);
                    umma_commit(empty(st));
                    items++;
                }
            }
        }
    } else {
        // ================= loads =================
        // (fp32: three warps for the keys, three for the values)
        const int grp = F::BF ? 0 : (warp - F::SW - 1) / F::PG, pt = tid - (F::SW + 1 + grp * F::PG) * 32;
        constexpr int NT = F::PG * 32;
        bool gone = false;
        while (!gone && next_unit(u)) {
            const int *par = a.parents ? a.parents + (int64_t)u.row * a.T : nullptr;
            const char *kb = a.c.k + u.row * a.c.rs + u.kvh * a.c.hs, *vb = a.c.v + u.row * a.c.rs + u.kvh * a.c.hs;
            uint32_t *bits = place_bits[warp - F::SW - 1];           // new tokens that are one, this warp's copy
            if (u.stop * KT > u.len) {
                __syncwarp();
                for (int w = 0; w * 32 < a.T; w++) {
                    const int x = w * 32 + lane;
                    const uint32_t m = __ballot_sync(0xffffffffu, x < a.T && cm_used(par, x));
                    if (lane == 0) bits[w] = m;
                }
                __syncwarp();
            }
            auto there = [&](int pos) { return pos < u.n && (pos < u.len || ((bits[(pos - u.len) >> 5] >> ((pos - u.len) & 31)) & 1u)); };
            // stage s of the unit: keys of tile 0, then in turn keys of the next tile and values of this one
            const int count = 2 * (u.stop - u.first);
            auto tile_of = [&](int s) { return s == 0 ? 0 : s == count - 1 ? (s - 1) / 2 : (s & 1) ? (s + 1) / 2 : (s - 2) / 2; };
            auto is_v = [&](int s) { return s == count - 1 || (s > 0 && !(s & 1)); };
            constexpr int UPR = HDP / 8, RPI = NT / UPR;             // units of 8 dims of a key, keys a step
            const int lu = pt % UPR, lr = pt / UPR;
            const bool in = lu * 8 < hd;
            if constexpr (F::BF) {
                // Whole tiles of cached tokens by TMA, a box of 64 dims by 128 keys at a time. The last ones, which end inside the
                // tile or have places without a token, by cp.async, which leaves zeros there.
#pragma unroll 1
                for (int s = 0; s < count; s++, it++) {
                    const uint32_t st = it % NST;
                    wait(empty(st), ((it / NST) & 1u) ^ 1u, 47);
                    if ((gone = __any_sync(0xffffffffu, wait.dead))) break;
                    const int t = u.first + tile_of(s);
                    const uint32_t to = cm_smem(ring + st * F::STAGE);
                    if ((t + 1) * KT <= u.len) {
                        if (pt == 0) {
                            mbar_expect_tx(full(st), (uint32_t)F::STAGE);
                            for (int x = 0; x < ATOMS; x++) ct_tma(to + x * F::KATOM, is_v(s) ? &mv : &mk, 64 * x, t * KT, u.kvh, u.row, full(st));
                        } else if (lane == 0) mbar_arrive(full(st));
                        continue;
                    }
                    const uint32_t mine = to + (lu / 8) * F::KATOM;
                    const char *from = (is_v(s) ? vb : kb) + lu * 16;
#pragma unroll 4
                    for (int r = lr; r < KT; r += RPI) {
                        const int pos = t * KT + r;
                        const bool ok = in && there(pos);
                        cm_cp16(mine + r * 128 + (((lu & 7) ^ (r & 7)) * 16), ok ? from + pos * a.c.ts : kb, ok);
                    }
                    asm volatile("cp.async.wait_all;" ::: "memory");
                    ct_fence_async();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(full(st));
                }
            } else {
                const char *from = (grp ? vb : kb) + lu * 32;
                const int tiles = u.stop - u.first;
#pragma unroll 1
                for (int t = 0; t < tiles; t++) {
                    const uint32_t s = it + (grp ? (t + 1 < tiles ? 2 + 2 * t : 2 * tiles - 1) : t ? 2 * t - 1 : 0), st = s % NST;
                    char *to = ring + st * F::STAGE + (lu / 8) * F::KATOM;
                    const bool tail = (u.first + t + 1) * KT > u.len;
#pragma unroll 1
                    for (int r0 = 0; r0 < KT; r0 += KT / 2) {        // half a stage: what a thread has registers for
                        constexpr int N2 = (KT / 2 + RPI - 1) / RPI;
                        float4 x[2 * N2];
#pragma unroll
                        for (int i = 0; i < N2; i++) {
                            const int rr = lr + i * RPI, pos = (u.first + t) * KT + r0 + rr;
                            const bool ok = in && rr < KT / 2 && (tail ? there(pos) : true);
                            const float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
                            x[2 * i] = ok ? *(const float4 *)(from + pos * a.c.ts) : z;
                            x[2 * i + 1] = ok ? *(const float4 *)(from + pos * a.c.ts + 16) : z;
                        }
                        if (r0 == 0) wait(empty(st), ((s / NST) & 1u) ^ 1u, 47);
#pragma unroll
                        for (int i = 0; i < N2; i++) {
                            const int r = r0 + lr + i * RPI;
                            if (lr + i * RPI >= KT / 2) continue;
                            const float4 f0 = x[2 * i], f1 = x[2 * i + 1];
                            float y[8] = {f0.x, f0.y, f0.z, f0.w, f1.x, f1.y, f1.z, f1.w};
#pragma unroll
                            for (int k = 0; k < F::NK; k++) {
                                uint32_t w[4];
#pragma unroll
                                for (int e = 0; e < 4; e++) {
                                    w[e] = cm_pack(y[2 * e], y[2 * e + 1]);
                                    const float2 f = cm_unpack(w[e]);
                                    y[2 * e] -= f.x; y[2 * e + 1] -= f.y;
                                }
                                *(uint4 *)(to + k * ATOMS * F::KATOM + r * 128 + (((lu & 7) ^ (r & 7)) * 16)) = make_uint4(w[0], w[1], w[2], w[3]);
                            }
                        }
                    }
                    ct_fence_async();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(full(st));
                }
                it += count;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (s_abort) {
        if (warp == F::SW && lane == 0) {
            umma_commit(bar_done);
            mbar_wait(bar_done, 0, err, 50);
        }
        if (F::BF && warp == F::SW + 1 && lane == 0) {               // copies into the ring's stages
            for (uint32_t x = it < NST ? 0 : it - NST; x < it; x++)
                if (!mbar_wait(full(x % NST), (x / NST) & 1u, err, 51)) break;
        }
        __syncthreads();
    }
    if (warp == F::SW) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

// a bf16 cache's keys or values as [row][head][slot][dim], boxes of 64 dims by kt slots (cache_attention.cu)
int ct_map(const char *who, const CacheDev &c, const char *p, int kt, CUtensorMap &m);

template <class KE, class QE, int HDP>
int ct_run_as(const char *who, CmArgs a, int max_keys) {
    using F = CtCfg<KE, QE, HDP>;
    using J = CmCfg<KE, QE, HDP, F::M>;
    a.tiles = (int)cdiv(a.M, F::M);
    CUtensorMap mk = {}, mv = {};
    if (F::BF && (ct_map(who, a.c, a.c.k, F::KT, mk) || ct_map(who, a.c, a.c.v, F::KT, mv))) return -1;
    static bool set = false;
    if (!set) {
        CUDA_CHECK(cudaFuncSetAttribute(k_cache_attention_tc<KE, QE, HDP>, cudaFuncAttributeMaxDynamicSharedMemorySize, F::SMEM));
        set = true;
    }
    const int rows = a.c.rows;
    const int64_t row_units = (int64_t)a.c.nkv * a.tiles, row_chunks = row_units * (cdiv(a.c.cap, F::KT) + F::START);
    int64_t most = 0x70000000 / row_chunks;
    if (a.weights) {
        a.pitch = cdiv((int64_t)a.c.cap, CM_PITCH) * CM_PITCH;
        most = std::min(most, std::max<int64_t>(1, ((int64_t)2 << 30) / (a.c.nkv * a.M * a.pitch * 4)));
    }
    if (most < 1) return cache_refuse(who, "%lld pieces of keys in a row", (long long)row_chunks);
    const int step = (int)std::min<int64_t>(rows, most);
    const int64_t units = step * row_units, spans = a.weights ? cdiv(a.pitch, cm_wkeys(a.M)) * step * a.c.nkv : 0;
    if (units * F::M + spans > 0x7fffffff) return cache_refuse(who, "%lld query tiles", (long long)units);
    const int ctas = (int)std::max<int64_t>(1, std::min<int64_t>(ctx().sm_count, units * cdiv(max_keys, F::KT)));
    if (!cm_parts<J>(who, a, step, units, ctas)) return -1;
    a.err = tc_err_flag();
    const int split = ctas > 4 * units;
    for (int r = 0; r < rows; r += step) {
        const int nr = std::min(step, rows - r);
        a.row0 = r;
        a.items = nr;
        LAUNCH_PDL((k_cache_attention_tc<KE, QE, HDP>), ctas, F::THREADS, F::SMEM, a, mk, mv, tc_err_flag());
        const int64_t joins = nr * row_units * (F::M / (split ? 1 : CM_THREADS / (HDP / 4)));
        LAUNCH_PDL((k_cache_join<KE, QE, HDP, F::M, false>), (unsigned)(joins + spans / step * nr), CM_THREADS, 0, a, (int)joins, split, cm_wkeys(a.M));
    }
    return 0;
}

} // namespace ncmb
