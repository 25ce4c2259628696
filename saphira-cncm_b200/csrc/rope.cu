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
constexpr int RO_SMEM = 48 * 1024 - RO_TOKENS * (8 + 8 + 4);        // what a launch may ask for beside the tokens' places

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
__global__ void __launch_bounds__(RO_THREADS, 4) k_rope(const __grid_constant__ NcmbRope r, const __grid_constant__ RopeArgs a) {
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

// Halves that are no whole vectors: an element's partner stands somewhere inside two vectors. The CTA's heads go through shared memory as they are; a
// thread takes the vector that it loaded, cuts its partners out of the two vectors that hold them -- at the same offset for all threads -- and writes
// 16 bytes. Cosines stand with every VE-th pair side by side, so that threads side by side read side by side.
// Bound by instructions: dims 50 of 8 x 4000 x 40 heads of 128 in bf16 183 us (an element at a time 269), dims 6 of 4 x 2000 in fp32 68 (84).
template <class E>
__global__ void __launch_bounds__(RO_THREADS, 4) k_rope_any(const __grid_constant__ NcmbRope r, const __grid_constant__ RopeArgs a) {
    constexpr int VE = 16 / sizeof(E), LOG = sizeof(E) == 4 ? 2 : 3;
    extern __shared__ __align__(16) char smem[];
    __shared__ int64_t xo[RO_TOKENS], yo[RO_TOKENS];
    __shared__ int place[RO_TOKENS];
    const int tid = threadIdx.x, half = r.dims / 2, row = rope_row(r.dims), stride = (half + VE - 1) >> LOG;
    uint4 *stage = (uint4 *)smem;                // [token][head][vector], and one more
    float2 *cs = (float2 *)(stage + a.per * a.share.heads * a.share.items + 1);
    const uint32_t n0 = blockIdx.x * (uint32_t)a.per;
    const int here = (int)min((uint32_t)a.per, a.tokens - n0), h0 = blockIdx.y * a.share.heads, heads = min(a.share.heads, a.n_head - h0);
    RopeWalk at(tid, a.share);
    pdl_wait();
    pdl_launch_dependents();
    if (tid < here) {
        const uint32_t n = n0 + tid, b = n / a.T, t = n - b * a.T;
        xo[tid] = b * a.xs[0] + t * a.xs[1] + h0 * a.xs[2];
        yo[tid] = b * a.ys[0] + t * a.ys[1] + h0 * a.ys[2];
        place[tid] = a.pos ? a.pos[n] : (int)t;
    }
    __syncthreads();
    const RopeWalk from = at;
    for (; at.tok < here; at.next(a.share)) {
        if (at.h >= heads) continue;
        const uint32_t to = (uint32_t)__cvta_generic_to_shared(stage + (at.tok * a.share.heads + at.h) * a.share.items + at.u);
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(a.x + xo[at.tok] + at.h * a.xs[2] + at.u * 16) : "memory");
    }
    rope_angles(tid, here, a.share, [&](int t, int i) { cs[t * row + (i & (VE - 1)) * stride + (i >> LOG)] = rope_angle(r, i, place[t], a.inverse); });
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    // what a thread's vector needs is the same for all of its heads: where its elements' cosines stand, the sign of their sines, its partners' vectors
    const int d0 = from.u * VE;
    const bool low = d0 < half, high = d0 + VE > half && d0 < r.dims;
    int at_cs[VE];
    uint32_t first = 0, turns = 0;               // bits: elements of the first half, those that turn
#pragma unroll
    for (int e = 0; e < VE; e++) {
        const int d = d0 + e, i = d < half ? d : d - half;
        if (d < half) first |= 1u << e;
        if (d < r.dims) turns |= 1u << e;
        at_cs[e] = d < r.dims ? (i & (VE - 1)) * stride + (i >> LOG) : 0;
    }
    // elements s ... s + VE - 1 of a head (those outside it are not used)
    auto cut = [&](const uint4 *head, int s, float (&y)[VE]) {
        const int v = s >> LOG, o = s & (VE - 1), w0 = sizeof(E) == 4 ? o : o >> 1;
        const uint4 l = head[max(v, 0)], h = head[v + 1];
        const uint32_t w[8] = {l.x, l.y, l.z, l.w, h.x, h.y, h.z, h.w};
        uint32_t c[5];
#pragma unroll
        for (int i = 0; i < 5; i++) {
            const uint32_t even = w0 & 2 ? w[i + 2] : w[i], odd = w0 & 2 ? w[min(i + 3, 7)] : w[i + 1];
            c[i] = w0 & 1 ? odd : even;
        }
        if (sizeof(E) == 2) {
#pragma unroll
            for (int i = 0; i < 4; i++) c[i] = __funnelshift_r(c[i], c[i + 1], (o & 1) * 16);
        }
        rope_unpack<E, VE>(make_uint4(c[0], c[1], c[2], c[3]), y);
    };
#pragma unroll 2
    for (at = from; at.tok < here; at.next(a.share)) {
        if (at.h >= heads) continue;
        const uint4 *head = stage + (at.tok * a.share.heads + at.h) * a.share.items;
        const float2 *f = cs + at.tok * row;
        float x[VE];
        rope_unpack<E, VE>(head[at.u], x);
        if (turns) {
            float p[VE], q[VE];
            if (low) cut(head, d0 + half, p);
            if (high) cut(head, d0 - half, q);
#pragma unroll
            for (int e = 0; e < VE; e++) {
                const float2 c = f[at_cs[e]];
                const float y = x[e] * c.x + (first >> e & 1 ? -p[e] : q[e]) * c.y;
                if (turns >> e & 1) x[e] = y;
            }
        }
        rope_store<E, VE>((E *)(a.y + yo[at.tok] + at.h * a.ys[2]) + d0, x);
    }
}

template <class E> void run_rope(const NcmbRope &r, RopeArgs &a) {
    constexpr int V = 16 / sizeof(E);
    const bool any = rope_vec(&r, sizeof(E)) < V;
    // a thread's items all on their way at once, and CTAs for all SMs (8 x 4000 tokens of 40 x 128 in bf16, 4 / 8 / 20 items a thread: 100 / 107 / 115 us)
    const int items = any ? (int)cdiv(a.hd, V) : rope_items(&r, a.hd, V), held = (any ? 2 * RO_BATCH : RO_BATCH) * (RO_THREADS / items), heads = any ? std::min(a.n_head, held) : a.n_head;
    a.share = rope_share(&r, items, heads, RO_THREADS);
    const int angles = rope_row(r.dims) * (int)sizeof(float2), staged = any ? heads * items * 16 : 0, spare = any ? 16 : 0;      // bytes a token, and once
    a.per = (int)std::max<int64_t>(1, std::min<int64_t>({any ? RO_TOKENS / 2 : RO_TOKENS, held / heads, (RO_SMEM - spare) / (angles + staged), a.tokens / (4 * ctx().sm_count)}));
    const size_t smem = (size_t)a.per * (angles + staged) + spare;
    const unsigned grid = (unsigned)cdiv(a.tokens, a.per);
    if (any) LAUNCH_PDL((k_rope_any<E>), dim3(grid, (unsigned)cdiv(a.n_head, heads)), RO_THREADS, smem, r, a);
    else if (r.layout == NCMB_ROPE_HALVES) LAUNCH_PDL((k_rope<E, V, false>), grid, RO_THREADS, smem, r, a);
    else LAUNCH_PDL((k_rope<E, V, true>), grid, RO_THREADS, smem, r, a);
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
    if (!(theta > 0 && theta < INFINITY) || !(factor > 0 && factor < INFINITY) || !(fabs((float)magnitude) < INFINITY)) return cache_refuse(who, "theta %g, factor %g, magnitude %g", theta, factor, magnitude);
    if (scaling == NCMB_ROPE_PARTS && !(trained > 0 && trained < INFINITY && low < high && fabs(low) < INFINITY && fabs(high) < INFINITY))
        return cache_refuse(who, "a trained context of %g, parts from %g to %g turns", trained, low, high);
    const double two_pi = 6.283185307179586476925;
    NcmbRope plan = {};
    plan.dims = dims;
    plan.layout = layout;
    plan.magnitude = (float)magnitude;
    if (scaling == NCMB_ROPE_BASE && dims > 2) theta *= pow(factor, dims / (dims - 2.0));
    for (int i = 0; i < dims / 2; i++) {
        double f = pow(theta, -2.0 * i / dims);
        if (scaling == NCMB_ROPE_LINEAR) f /= factor;
        if (scaling == NCMB_ROPE_PARTS) {
            const double g = fmin(1.0, fmax(0.0, (trained * f / two_pi - low) / (high - low)));
            f *= g + (1.0 - g) / factor;
        }
        if (!(f < INFINITY)) return cache_refuse(who, "theta %g, factor %g: pair %d turns without a limit", theta, factor, i);
        plan.turns[i] = f / two_pi;
    }
    *r = plan;
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
    a.x = (const char *)x; a.y = (char *)y; a.pos = pos; a.tokens = (uint32_t)tokens; a.T = T; a.n_head = n_head; a.hd = x == y ? (r->dims + 7) & ~7 : hd; a.inverse = inverse != 0;
    ProfScope prof(NCMB_K_ELEM, 3.0 * tokens * n_head * hd, 2.0 * tokens * n_head * hd * es);
    if (es == 2) run_rope<__nv_bfloat16>(*r, a);
    else run_rope<float>(*r, a);
    return 0;
}
