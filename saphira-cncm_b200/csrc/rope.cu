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

constexpr int RO_THREADS = 256, RO_BATCH = 2;

struct RopeArgs {
    const char *x; char *y;
    int64_t xs[3], ys[3];            // bytes
    const int *pos;
    int64_t tokens;
    int T, n_head, hd, inverse;      // hd: the dims that are moved, in place those that turn
    int per, items;                  // tokens a CTA, items a head
};

// A CTA has `per` tokens: their angles once, in shared memory, then all items of their heads. Loads of a thread's first items are under way
// while the angles are formed.
template <class E, int V, bool PAIRS>
__global__ void __launch_bounds__(RO_THREADS) k_rope(const __grid_constant__ NcmbRope r, const __grid_constant__ RopeArgs a) {
    extern __shared__ float2 cs[];               // [per][dims / 2]
    const int tid = threadIdx.x, pairs = r.dims / 2;
    pdl_wait();
    pdl_launch_dependents();
    const int64_t n0 = (int64_t)blockIdx.x * a.per;
    const int here = (int)min((int64_t)a.per, a.tokens - n0), per_token = a.n_head * a.items, total = here * per_token;
    float p[RO_BATCH][V], q[RO_BATCH][V];
    RopeItem it[RO_BATCH];
    E *to[RO_BATCH];
    int tok[RO_BATCH];
    auto load = [&](int i0) {
#pragma unroll
        for (int k = 0; k < RO_BATCH; k++) {
            const int i = i0 + k * RO_THREADS;
            if (i >= total) continue;
            tok[k] = i / per_token;
            const int j = i - tok[k] * per_token, h = j / a.items;
            it[k] = rope_item<V, PAIRS>(j - h * a.items, r.dims, a.hd);
            const uint32_t n = (uint32_t)n0 + tok[k], b = n / (uint32_t)a.T, t = n - b * (uint32_t)a.T;
            const E *from = (const E *)(a.x + b * a.xs[0] + t * a.xs[1] + h * a.xs[2]);
            to[k] = (E *)(a.y + b * a.ys[0] + t * a.ys[1] + h * a.ys[2]);
            rope_load<E, V>(from + it[k].d0, p[k]);
            if (it[k].d1 >= 0) rope_load<E, V>(from + it[k].d1, q[k]);
        }
    };
    load(tid);
    for (int i = tid; i < here * pairs; i += RO_THREADS) {
        const uint32_t n = (uint32_t)n0 + i / pairs;
        cs[i] = rope_angle(r, i % pairs, a.pos ? a.pos[n] : (int)(n % (uint32_t)a.T), a.inverse);
    }
    __syncthreads();
    for (int i0 = tid; i0 < total; i0 += RO_BATCH * RO_THREADS) {
        if (i0 != tid) load(i0);
#pragma unroll
        for (int k = 0; k < RO_BATCH; k++) {
            if (i0 + k * RO_THREADS >= total) continue;
            rope_turn<V, PAIRS>(it[k], cs + tok[k] * pairs, p[k], q[k]);
            rope_store<E, V>(to[k] + it[k].d0, p[k]);
            if (it[k].d1 >= 0) rope_store<E, V>(to[k] + it[k].d1, q[k]);
        }
    }
}

template <class E, int V> void run_rope(const NcmbRope &r, RopeArgs &a) {
    a.items = rope_items(&r, a.hd, V);
    // a few rounds of the CTA's threads, and no fewer CTAs than SMs
    const int64_t per_token = (int64_t)a.n_head * a.items;
    a.per = (int)std::max<int64_t>(1, std::min<int64_t>({16, 4 * RO_THREADS / per_token, a.tokens / ctx().sm_count}));
    const size_t smem = (size_t)a.per * (r.dims / 2) * sizeof(float2);
    const unsigned grid = (unsigned)cdiv(a.tokens, a.per);
    if (r.layout == NCMB_ROPE_HALVES) LAUNCH_PDL((k_rope<E, V, false>), grid, RO_THREADS, smem, r, a);
    else if constexpr (V >= 2) LAUNCH_PDL((k_rope<E, V, true>), grid, RO_THREADS, smem, r, a);
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
    a.x = (const char *)x; a.y = (char *)y; a.pos = pos; a.tokens = tokens; a.T = T; a.n_head = n_head; a.hd = x == y ? r->dims : hd; a.inverse = inverse != 0;
    ProfScope prof(NCMB_K_ELEM, 3.0 * tokens * n_head * hd, 2.0 * tokens * n_head * hd * es);
    switch (rope_vec(r, (int)es)) {
        case 8: run_rope<__nv_bfloat16, 8>(*r, a); break;
        case 4: if (es == 2) run_rope<__nv_bfloat16, 4>(*r, a); else run_rope<float, 4>(*r, a); break;
        case 2: if (es == 2) run_rope<__nv_bfloat16, 2>(*r, a); else run_rope<float, 2>(*r, a); break;
        default: if (es == 2) run_rope<__nv_bfloat16, 1>(*r, a); else run_rope<float, 1>(*r, a); break;
    }
    return 0;
}
