// Rotary positions by a plan (ncmb_rope_plan, ncmb_rope; include/ncm_b200.h): halves or neighbouring pairs, all or the first dims
// of a head, frequencies scaled for long contexts, forward and back.
#include "rope.cuh"

#include <algorithm>

namespace ncmb {

int rope_check(const char *who, const NcmbRope *r, int hd) {
    if (r->dims < 2 || r->dims > NCMB_ROPE_MAX || r->dims % 2 || r->dims > hd) return cache_refuse(who, "a plan for %d dims, heads of %d", r->dims, hd);
    if (r->layout != NCMB_ROPE_HALVES && r->layout != NCMB_ROPE_PAIRS) return cache_refuse(who, "layout %d of pairs", r->layout);
    return 0;
}

namespace {

constexpr int RO_THREADS = 256, RO_TOKENS = 32, RO_BATCH = 4;

struct RopeArgs {
    const char *x; char *y;
    int64_t xs[3], ys[3];            // bytes
    const int *pos;
    uint32_t tokens, T;
    int n_head, hd, inverse;         // hd: the dims that are moved, in place those that turn
    int per;                         // tokens a CTA
    RopeShare share;
};

// A CTA has `per` tokens: their places in memory and their angles once, in shared memory, then all items of their heads, RO_BATCH of a thread on their way at a
// time, the first of them while the angles are formed. Bound by DRAM: 8 x 4000 tokens of 40 heads of 128 in bf16, 655 MB: 100 us (6.5 TB/s).
template <class E, int V, bool PAIRS>
__global__ void __launch_bounds__(RO_THREADS, V * sizeof(E) == 16 ? 4 : 6) k_rope(const __grid_constant__ NcmbRope r, const __grid_constant__ RopeArgs a) {
    extern __shared__ __align__(16) float2 cs[];         // [per][rope_row(dims)]
    __shared__ int64_t xo[RO_TOKENS], yo[RO_TOKENS];
    __shared__ int place[RO_TOKENS];
    const int tid = threadIdx.x, row = rope_row(r.dims);
    const uint32_t n0 = blockIdx.x * (uint32_t)a.per;
    const int here = (int)min((uint32_t)a.per, a.tokens - n0);
    RopeWalk at(tid, a.share);
    const RopeItem it = rope_item<V, PAIRS>(at.u, a.share.items, r.dims, a.hd);
    pdl_wait();
    pdl_launch_dependents();
    if (tid < here) {
        const uint32_t n = n0 + tid, b = n / a.T, t = n - b * a.T;
        xo[tid] = b * a.xs[0] + t * a.xs[1];
        yo[tid] = b * a.ys[0] + t * a.ys[1];
        place[tid] = a.pos ? a.pos[n] : (int)t;
    }
    __syncthreads();
    RopeVec<E, V> p[RO_BATCH], q[RO_BATCH];
    RopeWalk from = at;
    auto load = [&](int k) {
        if (at.tok < here) {
            const E *x = (const E *)(a.x + xo[at.tok] + at.h * a.xs[2]);
            p[k] = *(const RopeVec<E, V> *)(x + it.d0);
            if (it.d1 >= 0) q[k] = *(const RopeVec<E, V> *)(x + it.d1);
        }
        at.next(a.share);
    };
#pragma unroll
    for (int k = 0; k < RO_BATCH; k++) load(k);
    rope_angles(tid, here, a.share, [&](int t, int i) { cs[t * row + rope_place<V, PAIRS>(i, r.dims)] = rope_angle(r, i, place[t], a.inverse); });
    __syncthreads();
    while (from.tok < here) {
#pragma unroll
        for (int k = 0; k < RO_BATCH; k++) {
            if (from.tok < here) {
                float f[V], g[V];
                rope_unpack<E, V>(p[k], f);
                if (it.d1 >= 0) rope_unpack<E, V>(q[k], g);
                rope_turn<V, PAIRS>(it, r.dims, cs + from.tok * row, f, g);
                E *y = (E *)(a.y + yo[from.tok] + from.h * a.ys[2]);
                rope_store<E, V>(y + it.d0, f);
                if (it.d1 >= 0) rope_store<E, V>(y + it.d1, g);
            }
            from.next(a.share);
            load(k);
        }
    }
}

template <class E, int V> void run_rope(const NcmbRope &r, RopeArgs &a) {
    a.share = rope_share(&r, rope_items(&r, a.hd, V), a.n_head, RO_THREADS);
    // A thread's items all on their way at once, and CTAs for all SMs (8 x 4000 tokens of 40 x 128 in bf16, 4 / 8 / 20 items a thread: 100 / 107 / 115 us);
    // short vectors are paced by instructions, so there the angles are shared by more (dims 50 of it, halves, 4 / 20 items: 293 / 277).
    const int64_t per_token = (int64_t)a.n_head * a.share.items, rounds = V * sizeof(E) == 16 ? RO_BATCH : 20;
    a.per = (int)std::max<int64_t>(1, std::min<int64_t>({RO_TOKENS, rounds * RO_THREADS / per_token, a.tokens / (4 * ctx().sm_count)}));
    const size_t smem = (size_t)a.per * rope_row(r.dims) * sizeof(float2);
    const unsigned grid = (unsigned)cdiv(a.tokens, a.per);
    if (r.layout == NCMB_ROPE_HALVES) LAUNCH_PDL((k_rope<E, V, false>), grid, RO_THREADS, smem, r, a);
    else if constexpr (V * sizeof(E) == 16) LAUNCH_PDL((k_rope<E, V, true>), grid, RO_THREADS, smem, r, a);
}

} // namespace
} // namespace ncmb

using namespace ncmb;

extern "C" int ncmb_rope_plan(NcmbRope *r, int dims, int layout, double theta, int scaling, double factor, double trained, double low, double high,
                              double magnitude) {
    const char *who = "ncmb_rope_plan";
    if (!r) return cache_refuse(who, "no plan to fill");
    if (dims < 2 || dims > NCMB_ROPE_MAX || dims % 2) return cache_refuse(who, "%d dims: even, 2 to %d", dims, NCMB_ROPE_MAX);
    if (layout != NCMB_ROPE_HALVES && layout != NCMB_ROPE_PAIRS) return cache_refuse(who, "layout %d of pairs", layout);
    if (scaling < NCMB_ROPE_PLAIN || scaling > NCMB_ROPE_PARTS) return cache_refuse(who, "scaling %d", scaling);
    if (!(theta > 0 && theta < INFINITY) || !(factor > 0 && factor < INFINITY) || !(fabs(magnitude) < INFINITY)) return cache_refuse(who, "theta %g, factor %g, magnitude %g", theta, factor, magnitude);
    if (scaling == NCMB_ROPE_PARTS && !(trained > 0 && trained < INFINITY && low < high && fabs(low) < INFINITY && fabs(high) < INFINITY))
        return cache_refuse(who, "a trained context of %g, parts from %g to %g turns", trained, low, high);
    const double two_pi = 6.283185307179586476925;
    *r = NcmbRope{};
    r->dims = dims;
    r->layout = layout;
    r->magnitude = (float)magnitude;
    if (scaling == NCMB_ROPE_BASE && dims > 2) theta *= pow(factor, dims / (dims - 2.0));
    for (int i = 0; i < dims / 2; i++) {
        double f = pow(theta, -2.0 * i / dims);
        if (scaling == NCMB_ROPE_LINEAR) f /= factor;
        if (scaling == NCMB_ROPE_PARTS) {
            const double g = fmin(1.0, fmax(0.0, (trained * f / two_pi - low) / (high - low)));
            f *= g + (1.0 - g) / factor;
        }
        r->turns[i] = f / two_pi;
    }
    return 0;
}

extern "C" int ncmb_rope(const NcmbRope *r, const void *x, const int64_t *xs, void *y, const int64_t *ys, int type, int rows, int T, int n_head, int hd,
                         const int *pos, int inverse) {
    const char *who = "ncmb_rope";
    if (!r || !xs || !ys) return cache_refuse(who, "a null pointer");
    if (type != NCMB_F32 && type != NCMB_BF16) return cache_refuse(who, "type %d", type);
    if (rows < 0 || T < 0 || n_head < 1 || hd < 8 || hd > NCMB_ROPE_MAX || hd % 8) return cache_refuse(who, "%d rows of %d tokens, %d heads of %d: a multiple of 8 up to %d", rows, T, n_head, hd, NCMB_ROPE_MAX);
    if (rope_check(who, r, hd)) return -1;
    const int64_t es = type == NCMB_BF16 ? 2 : 4, tokens = (int64_t)rows * T;
    if ((int64_t)n_head * hd > 1 << 24 || tokens > 0x7fffffff) return cache_refuse(who, "%lld tokens of %d heads", (long long)tokens, n_head);
    if (tokens == 0) return 0;
    if (!x || !y || ((uintptr_t)x | (uintptr_t)y) % 16 || ((uintptr_t)pos) % 4) return cache_refuse(who, "x and y have to be 16-byte aligned");
    RopeArgs a = {};
    for (int i = 0; i < 3; i++) {
        if (xs[i] < 0 || ys[i] < 0 || (xs[i] * es) % 16 || (ys[i] * es) % 16) return cache_refuse(who, "strides have to be positive multiples of 16 bytes");
        const int n = i == 0 ? rows : i == 1 ? T : n_head;
        if (n > 1 && ys[i] < hd) return cache_refuse(who, "a stride of the result is smaller than the head dim");
        if (x == y && n > 1 && xs[i] != ys[i]) return cache_refuse(who, "in place with other strides");
        a.xs[i] = xs[i] * es;
        a.ys[i] = ys[i] * es;
    }
    if (cache_device(who)) return -1;
    a.x = (const char *)x; a.y = (char *)y; a.pos = pos; a.tokens = (uint32_t)tokens; a.T = T; a.n_head = n_head; a.hd = x == y ? (r->layout == NCMB_ROPE_PAIRS ? std::min(hd, (r->dims + 7) & ~7) : r->dims) : hd; a.inverse = inverse != 0;
    ProfScope prof(NCMB_K_ELEM, 3.0 * tokens * n_head * hd, 2.0 * tokens * n_head * hd * es);
    switch (rope_vec(r, (int)es)) {
        case 8: run_rope<__nv_bfloat16, 8>(*r, a); break;
        case 4: if (es == 2) run_rope<__nv_bfloat16, 4>(*r, a); else run_rope<float, 4>(*r, a); break;
        case 2: if (es == 2) run_rope<__nv_bfloat16, 2>(*r, a); else run_rope<float, 2>(*r, a); break;
        default: if (es == 2) run_rope<__nv_bfloat16, 1>(*r, a); else run_rope<float, 1>(*r, a); break;
    }
    return 0;
}
