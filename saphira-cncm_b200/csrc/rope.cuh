// Rotary positions: what ncmb_rope and ncmb_paged_append share.
//
// A pair (x1, x2) at angle a = 2 pi p f, f full turns a position: y1 = m (x1 cos a - x2 sin a), y2 = m (x2 cos a + x1 sin a). p f is formed in 64
// bits and only its fraction of a turn goes on in fp32, in two parts: at position 10^6 an fp32 product is off by 0.06 radians, a fraction in one part
// by 9e-8. The second part costs no time (8 x 4000 tokens of 40 x 128 in bf16: 97.6 us either way).
//
// A thread's item is two vectors of V elements of a head. HALVES: the vectors at i and i + dims / 2, V pairs; PAIRS: the vectors i and i + half of
// the head's vectors, each of V / 2 pairs; dims that stay: likewise. So threads side by side have vectors side by side. V is 16 bytes where the dims allow it.
#pragma once
#include "cache.cuh"

#include <type_traits>

namespace ncmb {

// 0 when the plan is one that heads of hd can be rotated by, else -1 with a message
int rope_check(const char *who, const NcmbRope *r, int hd);

// elements of a vector: 16 bytes, or what halves that are no whole number of them leave whole
inline int rope_vec(const NcmbRope *r, int elem_bytes) {
    int v = 16 / elem_bytes;
    while (r && r->layout == NCMB_ROPE_HALVES && r->dims / 2 % v) v >>= 1;
    return v;
}
// items of a head
inline int rope_items(const NcmbRope *r, int hd, int v) {
    if (!r || r->layout == NCMB_ROPE_PAIRS) return (int)cdiv(hd, 2 * v);
    return r->dims / 2 / v + (int)cdiv(hd - r->dims, 2 * v);
}

// How a CTA's threads share the items of its tokens' heads and the tokens' angles, by divisions that the host does: a thread has item u of every step-th
// head, and goes from one to the next, and from one angle to the next, by additions.
struct RopeShare {
    int items, heads, step, dtok, dh;            // items a head, heads a token; step: heads that the threads cover at once
    int pairs, dt, dp;                           // pairs a token; from a thread's angle to its next: tokens and pairs
    uint32_t by_items, by_heads, by_pairs;       // x / d = x * by >> 16, rounded up: exact for x, d up to 256
};
inline RopeShare rope_share(const NcmbRope *r, int items, int heads, int threads) {
    RopeShare s;
    s.items = items; s.heads = heads; s.step = threads / items; s.dtok = s.step / heads; s.dh = s.step % heads;
    s.pairs = r ? r->dims / 2 : 1; s.dt = threads / s.pairs; s.dp = threads % s.pairs;
    auto by = [](int d) { return (uint32_t)cdiv(65536, d); };
    s.by_items = by(items); s.by_heads = heads > 256 ? 0 : by(heads); s.by_pairs = by(s.pairs);
    return s;
}

// cosines and sines of a token in shared memory: pairs in whole vectors
__host__ __device__ inline int rope_row(int dims) { return (dims / 2 + 7) & ~7; }

#ifdef __CUDACC__
// a vector as it is in memory
template <int BYTES> struct RopeRaw { using T = uint4; };
template <> struct RopeRaw<8> { using T = uint2; };
template <> struct RopeRaw<4> { using T = uint32_t; };
template <> struct RopeRaw<2> { using T = unsigned short; };
template <class E, int V> using RopeVec = typename RopeRaw<V * (int)sizeof(E)>::T;
template <class E, int V> __device__ __forceinline__ void rope_unpack(const RopeVec<E, V> &v, float (&x)[V]) {
    uint32_t u[4] = {0, 0, 0, 0};
    if constexpr (sizeof(v) == 16) { u[0] = v.x; u[1] = v.y; u[2] = v.z; u[3] = v.w; }
    else if constexpr (sizeof(v) == 8) { u[0] = v.x; u[1] = v.y; }
    else u[0] = v;
#pragma unroll
    for (int i = 0; i < V; i++) x[i] = __uint_as_float(sizeof(E) == 4 ? u[i] : i & 1 ? u[i / 2] & 0xffff0000u : u[i / 2] << 16);
}
// rounds once, to the nearest
template <class E, int V> __device__ __forceinline__ void rope_store(E *p, const float (&x)[V]) {
    if constexpr (sizeof(E) == 4) {
        if constexpr (V == 8) { *(float4 *)p = make_float4(x[0], x[1], x[2], x[3]); *(float4 *)(p + 4) = make_float4(x[4], x[5], x[6], x[7]); }
        else if constexpr (V == 4) *(float4 *)p = make_float4(x[0], x[1], x[2], x[3]);
        else if constexpr (V == 2) *(float2 *)p = make_float2(x[0], x[1]);
        else *p = x[0];
    } else if constexpr (V == 1) {
        *p = __float2bfloat16(x[0]);
    } else {
        uint32_t u[V / 2];
#pragma unroll
        for (int i = 0; i < V / 2; i++) { const __nv_bfloat162 t = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]); u[i] = *(const uint32_t *)&t; }
        if constexpr (V == 8) *(uint4 *)p = make_uint4(u[0], u[1], u[2], u[3]);
        else if constexpr (V == 4) *(uint2 *)p = make_uint2(u[0], u[1]);
        else *(uint32_t *)p = u[0];
    }
}

// cosine and sine of pair i at position pos, times the magnitude; what fp32 leaves of the angle by the first terms of both about it
__device__ __forceinline__ float2 rope_angle(const NcmbRope &r, int i, int pos, bool inverse) {
    const double t = (double)pos * r.turns[i], u = 2.0 * (t - rint(t));
    const float near = (float)u, rest = (float)(u - near) * 3.14159265f;
    float s, c;
    sincospif(near, &s, &c);
    const float cr = fmaf(-rest, s, c), sr = fmaf(rest, c, s);
    return make_float2(cr * r.magnitude, (inverse ? -sr : sr) * r.magnitude);
}

// where item u of a head stands, what its vectors are rotated by, if at all
struct RopeItem {
    int d0, d1;              // dims of its two vectors; d1 < 0: there is no second
    int pair;                // first pair of the first one's rotation, or -1; PAIRS: of the second, as far behind as it stands
};
template <int V, bool PAIRS> __device__ __forceinline__ RopeItem rope_item(int u, int items, int dims, int hd) {
    RopeItem it;
    const int rot = PAIRS ? 0 : dims / 2 / V;
    if (!PAIRS && u < rot) { it.d0 = u * V; it.d1 = it.d0 + dims / 2; it.pair = it.d0; return it; }
    it.d0 = (PAIRS ? 0 : dims) + (u - rot) * V;
    it.d1 = it.d0 + (items - rot) * V;
    if (it.d1 >= hd) it.d1 = -1;
    it.pair = PAIRS ? it.d0 / 2 : -1;
    return it;
}
// The items of a thread
struct RopeWalk {
    int u, tok, h;                   // tok: beyond the CTA's when there is none left
    __device__ RopeWalk(int tid, const RopeShare &s) {
        const int p = tid * s.by_items >> 16;
        u = tid - p * s.items;
        tok = p < s.step ? p * s.by_heads >> 16 : 1 << 20;       // more than 256 heads: by 0, the first token's
        h = p < s.step ? p - tok * s.heads : 0;
    }
    __device__ void next(const RopeShare &s) {
        tok += s.dtok;
        h += s.dh;
        if (h >= s.heads) { h -= s.heads; tok++; }
    }
};
// The tokens' angles, each once: angle(token, pair)
template <class F> __device__ __forceinline__ void rope_angles(int tid, int here, const RopeShare &s, F angle) {
    int t = tid * s.by_pairs >> 16, i = tid - t * s.pairs;
    while (t < here) {
        angle(t, i);
        t += s.dt;
        i += s.dp;
        if (i >= s.pairs) { i -= s.pairs; t++; }
    }
}
// Cosines and sines of a token in shared memory: those that a vector needs are read two pairs (16 bytes) at a time, and vectors side by side by
// threads side by side, so two pairs of all vectors stand together, then the next two.
template <int V, bool PAIRS> __device__ __forceinline__ int rope_place(int pair, int dims) {
    constexpr int W = PAIRS ? V / 2 : V;         // pairs of a vector
    if constexpr (W < 2) return pair;
    const int vecs = (dims / 2 + W - 1) / W, v = pair / W, i = pair % W;
    return (i / 2 * vecs + v) * 2 + (i & 1);
}
// a, b: the item's vectors; cs: the token's cosines and sines
template <int V, bool PAIRS> __device__ __forceinline__ void rope_turn(const RopeItem &it, int dims, const float2 *cs, float (&a)[V], float (&b)[V]) {
    constexpr int W = PAIRS ? V / 2 : V;
    const int pairs = dims / 2, vecs = (pairs + W - 1) / W;
    auto factors = [&](int pair, float2 (&f)[W]) {
        if constexpr (W < 2) f[0] = cs[pair];
        else {
            const float4 *p = (const float4 *)cs + pair / W;
#pragma unroll
            for (int i = 0; i < W / 2; i++) {
                const float4 u = p[i * vecs];
                f[2 * i] = make_float2(u.x, u.y);
                f[2 * i + 1] = make_float2(u.z, u.w);
            }
        }
    };
    if constexpr (PAIRS) {
        static_assert(V >= 2, "a pair is in one vector");
        auto one = [&](int pair, float (&x)[V]) {
            if (pair >= pairs) return;
            float2 f[W];
            factors(pair, f);
#pragma unroll
            for (int i = 0; i < W; i++) {
                if (pair + i >= pairs) break;            // the last vector's dims beyond
                const float p = x[2 * i], q = x[2 * i + 1];
                x[2 * i] = p * f[i].x - q * f[i].y;
                x[2 * i + 1] = q * f[i].x + p * f[i].y;
            }
        };
        one(it.pair, a);
        if (it.d1 >= 0) one(it.d1 / 2, b);
    } else if (it.pair >= 0) {
        float2 f[W];
        factors(it.pair, f);
#pragma unroll
        for (int i = 0; i < V; i++) {
            const float p = a[i], q = b[i];
            a[i] = p * f[i].x - q * f[i].y;
            b[i] = q * f[i].x + p * f[i].y;
        }
    }
}
#endif

} // namespace ncmb
