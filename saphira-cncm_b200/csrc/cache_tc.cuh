// Attention of many query rows (trees, runs of tokens, several heads a kv head) to cached keys on tcgen05 tiles: the wide
// variant of cache_mma.cuh, for ncmb_cache_attention.
//
// A CTA has 128 query rows of a kv head and walks tiles of 64 keys: S = Q K^T into tensor memory, softmax with a running
// maximum by 256 threads (two a row, 32 keys each), O = P V of the tile into tensor memory, added to the running result
// in registers in fp32. Operands are bf16 terms, as in cache_mma.cuh: a query is 3 (bf16 activations: 1), a probability 3
// (2), a bf16 key or value 1, an fp32 one 3, of whose nine products the six largest are taken (2^-24 and more). Roles:
// warps 0 - 7 softmax (they also turn the queries into terms and write the results), warp 8 issues the MMAs, the others load
// keys and values -- bf16 by cp.async, fp32 through registers, where the terms are formed.
//
// Bound by operand fetch from shared memory: an MMA of 128 x 64 x 16 reads 6 KB in about 48 cycles where its arithmetic
// takes 16; with one product that is below the time the keys take from HBM at 128 rows and head dim 128.
#pragma once
#include "cache_mma.cuh"
#include "tc_common.cuh"

namespace ncmb {

template <class KE, class QE, int HDP_> struct CtCfg {
    static constexpr bool BF = sizeof(KE) == 2;
    static constexpr int HDP = HDP_, ATOMS = HDP / 64, M = 128, KT = 64;
    static constexpr int NQ = sizeof(QE) == 4 ? 3 : 1, NP = sizeof(QE) == 4 ? 3 : 2, NK = BF ? 1 : 3;
    static constexpr int KATOM = KT * 128, QATOM = M * 128;          // bytes of 64 dims of the keys, of the queries
    static constexpr int STAGE = 2 * NK * ATOMS * KATOM, QB = NQ * ATOMS * QATOM, PB = NP * QATOM;
    static constexpr int FIT = (221 * 1024 - QB - PB) / STAGE, NST = FIT < 6 ? FIT : 6;
    static constexpr int PW = BF ? 3 : 7, SW = 8, THREADS = 32 * (SW + 1 + PW);      // whole warps a scheduler: registers
    static constexpr int SMEM = QB + PB + NST * STAGE + 1024;
    static constexpr int TMEM = HDP == 64 ? 256 : 256;               // columns: two score tiles of 64, the tile's context
};

__host__ __device__ constexpr uint32_t umma_idesc_bf16(int M, int N) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
struct CtWait {
    int *err; bool dead;
    __device__ __forceinline__ void operator()(uint32_t bar, uint32_t parity, int code) {
        if (!dead && !mbar_wait(bar, parity, err, code)) dead = true;
    }
};
__device__ __forceinline__ bool ct_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
__device__ __forceinline__ void ct_fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

template <class KE, class QE, int HDP>
__global__ void __launch_bounds__(CtCfg<KE, QE, HDP>::THREADS, 1) k_cache_attention_tc(const __grid_constant__ CmArgs a, int *err) {
    using F = CtCfg<KE, QE, HDP>;
    constexpr int M = F::M, KT = F::KT, NST = F::NST, ATOMS = F::ATOMS, SLOT = M * (HDP + 2);
    extern __shared__ char smem_raw[];
    char *smem = (char *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    char *qs = smem, *ps = qs + F::QB, *ring = ps + F::PB;
    __shared__ uint64_t bars[2 * 8 + 8];
    __shared__ uint32_t tmem_at;
    __shared__ int plan[4];                                          // total, per, item, where it begins
    __shared__ float xm[2][2][M], xl[2][M];
    __shared__ uint32_t node_bits[M][8];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, hd = a.c.hd, G = a.G;
    auto full = [&](int s) { return cm_smem(&bars[s]); };
    auto empty = [&](int s) { return cm_smem(&bars[8 + s]); };
    const uint32_t bar_q = cm_smem(&bars[16]), bar_s = cm_smem(&bars[17]), bar_p = cm_smem(&bars[19]), bar_pv = cm_smem(&bars[20]);
    pdl_wait();
    pdl_launch_dependents();
    __shared__ int s_abort;
    if (tid == 0) {
        s_abort = *(volatile int *)err;                              // a wait ran out earlier: nothing more is started
        for (int s = 0; s < NST; s++) { mbar_init(full(s), F::PW); mbar_init(empty(s), 1); }
        mbar_init(bar_q, F::SW); mbar_init(bar_s, 1); mbar_init(bar_s + 8, 1); mbar_init(bar_p, F::SW); mbar_init(bar_pv, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        // the plan of cache_mma.cuh, by one warp
        int t = 0;
        for (int i = lane; i < a.items; i += 32) t += cm_chunks<false, KT>(a, i);
        t = __reduce_add_sync(0xffffffffu, t);
        const int per = (unsigned)(t + (int)gridDim.x - 1) / gridDim.x, x = (int)min((int64_t)blockIdx.x * per, (int64_t)t);
        int before = 0, item = 0, begin = 0;
        for (int i0 = 0; i0 < a.items; i0 += 32) {
            const int mine = cm_chunks<false, KT>(a, i0 + lane);
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
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(cm_smem(&tmem_at)), "r"(F::TMEM) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_at;
    CtWait wait{err, false};

    struct Unit { int item, kvh, m0, first, stop, unit, n, len, row; bool whole; };
    int at = blockIdx.x * plan[1], item = plan[2], item_at = plan[3];
    const int end = min(plan[0], at + plan[1]);
    auto next_unit = [&](Unit &u) {                                  // the run's next unit, or false
        if (at >= end) return false;
        u.n = cm_keys<false>(a, item);
        const int nch = (u.n + KT - 1) / KT, sub = cm_div(at - item_at, nch), kvh = a.tiles == 1 ? sub : cm_div(sub, a.tiles);
        u.item = item; u.kvh = kvh; u.m0 = (sub - kvh * a.tiles) * M;
        u.first = at - item_at - sub * nch; u.stop = min(nch, u.first + (end - at));
        u.unit = item * a.c.nkv * a.tiles + sub;
        u.len = u.n - a.T; u.row = a.row0 + item; u.whole = u.first == 0 && u.stop == nch;
        at += u.stop - u.first;
        if (at == item_at + nch * a.c.nkv * a.tiles) { item_at = at; item++; }
        return true;
    };
    Unit u;
    uint32_t it = 0, un = 0;                                         // tiles and units so far

    if (warp < F::SW) {
        // ================= softmax: row r of the tile, keys 32 hf ... of a key tile, half hf of the dims =================
        const int r = (warp & 3) * 32 + lane, hf = warp >> 2;
        const uint32_t tl = tmem + ((uint32_t)(warp & 3) << 21);     // this warp's 32 lanes of tensor memory
        constexpr int HC = HDP / 2;
        auto group_sync = [] { asm volatile("bar.sync 1, %0;" ::"n"(F::SW * 32) : "memory"); };
        while (next_unit(u)) {
            const int *par = a.parents ? a.parents + (int64_t)u.row * a.T : nullptr;
            // queries as terms (the MMAs that read the last unit's are done: their scores have been read)
#pragma unroll 1
            for (int i = tid; i < M * HDP / 8; i += F::SW * 32) {
                const int m = i / (HDP / 8), d0 = i % (HDP / 8) * 8, mm = u.m0 + m;
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; e++) x[e] = 0.f;
                if (mm < a.M && d0 < hd) {
                    const int t = mm / G, h = u.kvh * G + mm - t * G;
                    if (cm_used(par, t)) {
                        const char *p = a.q + ((int64_t)u.row * a.T + t) * a.ldq + ((int64_t)h * hd + d0) * sizeof(QE);
                        if constexpr (sizeof(QE) == 4) {
                            *(float4 *)&x[0] = *(const float4 *)p;
                            *(float4 *)&x[4] = *(const float4 *)(p + 16);
                        } else {
                            const uint4 q = *(const uint4 *)p;
                            const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                            for (int e = 0; e < 4; e++) { const float2 f = cm_unpack(w[e]); x[2 * e] = f.x; x[2 * e + 1] = f.y; }
                        }
                    }
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
            const int mm = u.m0 + r, node = min(mm, a.M - 1) / G;
            const bool row_used = mm < a.M && cm_used(par, node);
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
                if (skip) { skip = false; return; }
#pragma unroll
                for (int x = 0; x < HC; x += 32) {
                    uint32_t o[32];
                    tmem_ld32(tl + 128u + (uint32_t)(hf * HC + x), o);
#pragma unroll
                    for (int d = 0; d < 32; d++) O[x + d] = fmaf(O[x + d], al_prev, __uint_as_float(o[d]));
                }
            };
            for (int t = u.first; t < u.stop; t++, it++) {
                wait(bar_s + 8 * (it & 1u), (it >> 1) & 1u, 42);
                tc_fence_after();
                uint32_t sr[32];
                tmem_ld32(tl + (it & 1u) * 64u + (uint32_t)hf * 32u, sr);
                float s[32];
                const int p0 = t * KT + 32 * hf;
                const bool masked = (t + 1) * KT > u.len;
                uint32_t see = 0xffffffffu;
                if (masked) {
                    // bit j: the row sees slot p0 + j
                    const int rel = p0 - u.len;                      // node of the first slot
                    if (rel > -32) {
                        uint32_t lo = 0, hi = 0;
                        const int w = rel < 0 ? -1 : rel >> 5, sh = rel & 31;
                        if (w >= 0 && w < 8) lo = node_bits[r][w];
                        if (w < 0) lo = 0xffffffffu;                 // slots of the cache
                        if (w + 1 < 8) hi = node_bits[r][w + 1];
                        see = __funnelshift_r(lo, hi, sh);
                    }
                    if (u.n - p0 < 32) see &= u.n > p0 ? (1u << (u.n - p0)) - 1 : 0u;
                }
                float top = -INFINITY;
#pragma unroll
                for (int j = 0; j < 32; j++) {
                    s[j] = __uint_as_float(sr[j]) * a.c2;
                    if (!((see >> j) & 1u)) s[j] = -INFINITY;
                    top = fmaxf(top, s[j]);
                }
                if (a.scores && mm < a.M) {
                    float *sp = a.scores + (((int64_t)u.item * a.c.nkv + u.kvh) * a.M + mm) * a.pitch + p0;
#pragma unroll
                    for (int j = 0; j < 32; j += 4) *(float4 *)(sp + j) = make_float4(s[j], s[j + 1], s[j + 2], s[j + 3]);
                }
                xm[it & 1u][hf][r] = top;
                group_sync();
                top = fmaxf(fmaxf(mx, top), xm[it & 1u][hf ^ 1][r]);
                const float base = top == -INFINITY ? 0.f : top, al = cm_exp2(mx - base);
                mx = top;
                float sum = 0.f;
#pragma unroll
                for (int j = 0; j < 32; j++) { s[j] = cm_exp2(s[j] - base); sum += s[j]; }
                l = l * al + sum;
                if (t > u.first) add_context();                      // also: the MMAs that read the last probabilities are done
                al_prev = al;
                // probabilities as terms: 4 units of 8 keys
#pragma unroll
                for (int x = 0; x < 4; x++)
#pragma unroll
                    for (int k = 0; k < F::NP; k++) {
                        uint32_t w[4];
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            float *q = &s[8 * x + 2 * e];
                            w[e] = cm_pack(q[0], q[1]);
                            const float2 f = cm_unpack(w[e]);
                            q[0] -= f.x; q[1] -= f.y;
                        }
                        *(uint4 *)(ps + k * F::QATOM + r * 128 + (((4 * hf + x) ^ (r & 7)) * 16)) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                if (masked) {
                    // An infinity or NaN among values that not every row sees must not be multiplied by zero: such a tile's context is
                    // formed here, one key at a time, before the stage is given to the MMAs (whose result is then left out).
                    const int st = it % NST;
                    wait(full(st), (it / NST) & 1u, 43);
                    const char *vt = ring + st * F::STAGE + F::STAGE / 2;
                    bool odd = false;
#pragma unroll 1
                    for (int i = tid; i < F::NK * ATOMS * F::KATOM / 4; i += F::SW * 32) {
                        const uint32_t w = ((const uint32_t *)vt)[i];
                        odd |= (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
                    }
                    uint32_t any;
                    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                                 : "=r"(any) : "r"((uint32_t)odd), "n"(F::SW * 32) : "memory");
                    if (any) {
#pragma unroll
                        for (int d = 0; d < HC; d++) O[d] *= al;
#pragma unroll 1
                        for (int j = 0; j < KT; j++) {
                            float p = 0.f;
#pragma unroll
                            for (int k = F::NP - 1; k >= 0; k--) p += (float)*(const __nv_bfloat16 *)(ps + k * F::QATOM + r * 128 + (((j / 8) ^ (r & 7)) * 16) + (j & 7) * 2);
                            if (p == 0.f) continue;
#pragma unroll
                            for (int d = 0; d < HC; d++) {
                                const int dd = hf * HC + d;
                                float v = 0.f;
#pragma unroll
                                for (int k = F::NK - 1; k >= 0; k--)
                                    v += (float)*(const __nv_bfloat16 *)(vt + (k * ATOMS + dd / 64) * F::KATOM + j * 128 + ((((dd & 63) / 8) ^ (j & 7)) * 16) + (dd & 7) * 2);
                                O[d] = fmaf(p, v, O[d]);
                            }
                        }
                        skip = true;
                    }
                }
                tc_fence_before();
                ct_fence_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar_p);
            }
            add_context();
            xl[hf][r] = l;
            if (hf == 0 && r == 0) {
                if (u.first == 0) a.range[u.unit].x = blockIdx.x;
                if (u.stop * KT >= u.n) a.range[u.unit].y = blockIdx.x;
            }
            group_sync();
            l += xl[hf ^ 1][r];
            float *slot = a.part + ((int64_t)blockIdx.x + u.unit) * SLOT;
            if (hf == 0) { slot[r] = mx; slot[M + r] = l; }
            if (mm < a.M) {
                if (u.whole) {
                    const float f = l > 0.f && row_used ? 1.f / l : 0.f;
                    QE *o = (QE *)(a.out + ((int64_t)u.row * a.T + node) * a.ldo) + (int64_t)(u.kvh * G + mm - node * G) * hd + hf * HC;
#pragma unroll
                    for (int d = 0; d < HC; d += 4) {
                        if (hf * HC + d >= hd) continue;
                        if constexpr (sizeof(QE) == 4) *(float4 *)(o + d) = make_float4(O[d] * f, O[d + 1] * f, O[d + 2] * f, O[d + 3] * f);
                        else *(uint2 *)(o + d) = make_uint2(cm_pack(O[d] * f, O[d + 1] * f), cm_pack(O[d + 2] * f, O[d + 3] * f));
                    }
                } else {
                    float *o = slot + 2 * M + r * HDP + hf * HC;
#pragma unroll
                    for (int d = 0; d < HC; d += 4) *(float4 *)(o + d) = make_float4(O[d], O[d + 1], O[d + 2], O[d + 3]);
                }
            }
        }
    } else if (warp == F::SW) {
        // ================= MMAs =================
        if (lane == 0) {
            constexpr uint32_t ids = umma_idesc_bf16(M, KT), idv = umma_idesc_bf16(M, 64) | (1u << 16);      // values: MN-major
            const uint64_t qd = umma_desc_sw128(cm_smem(qs)), pd = umma_desc_sw128(cm_smem(ps)), rd = umma_desc_sw128(cm_smem(ring));
            constexpr uint64_t QA = F::QATOM / 16, KA = F::KATOM / 16, ST = F::STAGE / 16;
            auto scores = [&](uint32_t i) {
                const uint32_t st = i % NST;
                wait(full(st), (i / NST) & 1u, 44);
                tc_fence_after();
                uint32_t acc = 0;
                const uint64_t kd = rd + st * ST;
                auto product = [&](int qk, int kk) {                 // one term of the queries by one of the keys
#pragma unroll
                    for (int x = 0; x < ATOMS; x++)
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            umma_f16(tmem + (i & 1u) * 64u, qd + (qk * ATOMS + x) * QA + k * 2, kd + (kk * ATOMS + x) * KA + k * 2, ids, acc);
                            acc = 1;
                        }
                };
#pragma unroll 1
                for (int sum = F::NQ + F::NK - 2 < 2 ? F::NQ + F::NK - 2 : 2; sum >= 0; sum--)       // small ones first
#pragma unroll 1
                    for (int qk = 0; qk <= sum; qk++) if (qk < F::NQ && sum - qk < F::NK) product(qk, sum - qk);
                umma_commit(bar_s + 8 * (i & 1u));
            };
            while (next_unit(u)) {
                wait(bar_q, un & 1u, 45);
                un++;
                tc_fence_after();
                const int tiles = u.stop - u.first;
                scores(it);
#pragma unroll 1
                for (int t = 0; t < tiles; t++, it++) {
                    if (t + 1 < tiles) scores(it + 1);
                    wait(bar_p, it & 1u, 46);
                    tc_fence_after();
                    const uint32_t st = it % NST;
                    const uint64_t vd = rd + st * ST + ST / 2;
                    uint32_t acc = 0;
#pragma unroll 1
                    for (int sum = F::NP + F::NK - 2 < 2 ? F::NP + F::NK - 2 : 2; sum >= 0; sum--)
#pragma unroll 1
                        for (int pk = 0; pk <= sum; pk++) {
                            if (pk >= F::NP || sum - pk >= F::NK) continue;
#pragma unroll
                            for (int k = 0; k < 4; k++) {
#pragma unroll
                                for (int x = 0; x < ATOMS; x++)
                                    umma_f16(tmem + 128u + 64u * x, pd + pk * QA + k * 2, vd + ((sum - pk) * ATOMS + x) * KA + k * 128, idv, acc);
                                acc = 1;
                            }
                        }
                    umma_commit(bar_pv);
                    umma_commit(empty(st));
                }
            }
        }
    } else {
        // ================= loads =================
        const int pt = tid - (F::SW + 1) * 32;
        constexpr int NT = F::PW * 32, LAG = NST - 1;
        while (next_unit(u)) {
            const int *par = a.parents ? a.parents + (int64_t)u.row * a.T : nullptr;
            const char *kb = a.c.k + u.row * a.c.rs + u.kvh * a.c.hs, *vb = a.c.v + u.row * a.c.rs + u.kvh * a.c.hs;
            auto there = [&](int pos) { return pos < u.n && (pos < u.len || cm_used(par, pos - u.len)); };
            if constexpr (F::BF) {
                constexpr int UPR = HDP / 8, RPI = NT / UPR;         // 16-byte units of a key, keys a step
                const int lu = pt % UPR, lr = pt / UPR;
                const bool in = lu * 8 < hd;
                uint32_t done = it;                                  // tiles handed over
                auto hand_over = [&](uint32_t to) {
                    ct_fence_async();
                    __syncwarp();
                    if (lane == 0) for (uint32_t i = done; i < to; i++) mbar_arrive(full(i % NST));
                    done = to;
                };
#pragma unroll 1
                for (int t = u.first; t < u.stop; t++) {
                    const uint32_t st = it % NST, free = ((it / NST) & 1u) ^ 1u;
                    if (!__all_sync(0xffffffffu, ct_try(empty(st), free))) {
                        // the stage is freed by MMAs that may be waiting for what is under way
                        asm volatile("cp.async.wait_group 0;" ::: "memory");
                        hand_over(it);
                        wait(empty(st), free, 47);
                    }
                    const uint32_t ks = cm_smem(ring + st * F::STAGE) + (lu / 8) * F::KATOM;
                    const bool tail = (t + 1) * KT > u.len;
#pragma unroll 4
                    for (int i = 0; i < (KT + RPI - 1) / RPI; i++) {
                        const int r = lr + i * RPI, pos = t * KT + r;
                        if (r >= KT) break;
                        const bool ok = in && (tail ? there(pos) : true);
                        const int64_t off = ok ? pos * a.c.ts + lu * 16 : 0;
                        const uint32_t to = r * 128 + (((lu & 7) ^ (r & 7)) * 16);
                        cm_cp16(ks + to, kb + off, ok);
                        cm_cp16(ks + F::STAGE / 2 + to, vb + off, ok);
                    }
                    asm volatile("cp.async.commit_group;" ::: "memory");
                    it++;
                    if (it - done > (uint32_t)LAG) {                 // all but the last LAG tiles are there
                        asm volatile("cp.async.wait_group %0;" ::"n"(LAG) : "memory");
                        hand_over(it - LAG);
                    }
                }
                asm volatile("cp.async.wait_group 0;" ::: "memory");
                hand_over(it);
            } else {
                // A thread has 8 dims of KT / RPI keys: two loads each for keys and values, of the next tile while this one is turned
                // into terms.
                constexpr int UPR = HDP / 8, RPI = NT / UPR, N = (KT + RPI - 1) / RPI;
                const int lu = pt % UPR, lr = pt / UPR;
                const bool in = lu * 8 < hd;
                float4 x[4 * N];
                auto fetch = [&](int t) {
                    const bool tail = (t + 1) * KT > u.len;
#pragma unroll
                    for (int i = 0; i < N; i++) {
                        const int pos = t * KT + lr + i * RPI;
                        const bool ok = in && lr + i * RPI < KT && (tail ? there(pos) : true);
                        const int64_t off = pos * a.c.ts + lu * 32;
                        const float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
                        x[4 * i] = ok ? *(const float4 *)(kb + off) : z; x[4 * i + 1] = ok ? *(const float4 *)(kb + off + 16) : z;
                        x[4 * i + 2] = ok ? *(const float4 *)(vb + off) : z; x[4 * i + 3] = ok ? *(const float4 *)(vb + off + 16) : z;
                    }
                };
                fetch(u.first);
#pragma unroll 1
                for (int t = u.first; t < u.stop; t++, it++) {
                    const uint32_t st = it % NST;
                    wait(empty(st), ((it / NST) & 1u) ^ 1u, 47);
                    char *ks = ring + st * F::STAGE + (lu / 8) * F::KATOM;
#pragma unroll
                    for (int i = 0; i < N; i++)
#pragma unroll
                        for (int kv = 0; kv < 2; kv++) {
                            const int r = lr + i * RPI;
                            if (r >= KT) continue;
                            const float4 f0 = x[4 * i + 2 * kv], f1 = x[4 * i + 2 * kv + 1];
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
                                *(uint4 *)(ks + kv * (F::STAGE / 2) + k * ATOMS * F::KATOM + r * 128 + (((lu & 7) ^ (r & 7)) * 16)) = make_uint4(w[0], w[1], w[2], w[3]);
                            }
                        }
                    if (t + 1 < u.stop) fetch(t + 1);
                    ct_fence_async();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(full(st));
                }
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    if (warp == F::SW) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(F::TMEM) : "memory");
    }
}

template <class KE, class QE, int HDP>
int ct_run_as(const char *who, CmArgs a, int max_keys) {
    using F = CtCfg<KE, QE, HDP>;
    using J = CmCfg<KE, QE, HDP, F::M>;
    a.tiles = (int)cdiv(a.M, F::M);
    static bool set = false;
    if (!set) {
        CUDA_CHECK(cudaFuncSetAttribute(k_cache_attention_tc<KE, QE, HDP>, cudaFuncAttributeMaxDynamicSharedMemorySize, F::SMEM));
        set = true;
    }
    const int rows = a.c.rows;
    const int64_t row_units = (int64_t)a.c.nkv * a.tiles, row_chunks = row_units * cdiv(a.c.cap, F::KT);
    int64_t most = 0x70000000 / row_chunks;
    if (a.weights) {
        a.pitch = cdiv((int64_t)a.c.cap, CM_WKEYS) * CM_WKEYS;
        most = std::min(most, std::max<int64_t>(1, ((int64_t)2 << 30) / (a.c.nkv * a.M * a.pitch * 4)));
    }
    if (most < 1) return cache_refuse(who, "%lld pieces of keys in a row", (long long)row_chunks);
    const int step = (int)std::min<int64_t>(rows, most);
    const int64_t units = step * row_units, spans = a.weights ? cdiv(a.pitch, CM_WKEYS) * step * a.c.nkv : 0;
    if (units * F::M + spans > 0x7fffffff) return cache_refuse(who, "%lld query tiles", (long long)units);
    const int ctas = (int)std::max<int64_t>(1, std::min<int64_t>(ctx().sm_count, units * cdiv(max_keys, F::KT)));
    const size_t ranges = ((size_t)units * 8 + 255) & ~(size_t)255, part = (size_t)(units + ctas) * J::SLOT * 4;
    const size_t sc = a.weights ? (size_t)step * a.c.nkv * a.M * a.pitch * 4 : 0;
    char *scratch = (char *)cache_scratch(who, sc + ranges + part);
    if (!scratch) return -1;
    a.scores = a.weights ? (float *)scratch : nullptr;
    a.range = (int2 *)(scratch + sc);
    a.part = (float *)(scratch + sc + ranges);
    const int split = ctas > 4 * units;
    for (int r = 0; r < rows; r += step) {
        const int nr = std::min(step, rows - r);
        a.row0 = r;
        a.items = nr;
        LAUNCH_PDL((k_cache_attention_tc<KE, QE, HDP>), ctas, F::THREADS, F::SMEM, a, tc_err_flag());
        const int64_t joins = nr * row_units * (F::M / (split ? 1 : CM_THREADS / (HDP / 4)));
        LAUNCH_PDL((k_cache_join<KE, QE, HDP, F::M, false>), (unsigned)(joins + spans / step * nr), CM_THREADS, 0, a, (int)joins, split);
    }
    return 0;
}

} // namespace ncmb
