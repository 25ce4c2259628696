// Attention of a row's new tokens -- a decode step's one, a run, or a tree of drafted ones -- to its pages (ncmb_paged_attention,
// include/ncm_b200.h): the tiles of cache_mma.cuh, or of cache_tc.cuh for many query rows, with keys and values found through the row's table.
#include "cache_tc.cuh"
#include "paged.cuh"

namespace ncmb {
namespace {

template <class KE, class QE, int HDP>
int run_paged_hd(const char *who, const CmArgs &a, int max_keys) {
    // (as for ncmb_cache_attention: no wide tiles for fp32 caches of more than 64 dims)
    if constexpr (sizeof(KE) == 2 || HDP == 64) { if (takes_wide<KE, QE, HDP>(a, max_keys)) return ct_run_as<KE, QE, HDP, true>(who, a, max_keys); }
    auto none = [] {};
    return a.M <= 8 ? cm_run_as<KE, QE, HDP, 8, false, true>(who, a, max_keys, none) : cm_run_as<KE, QE, HDP, 16, false, true>(who, a, max_keys, none);
}
template <class KE, class QE>
int run_paged(const char *who, const CmArgs &a, int max_keys) {
    return a.c.hd <= 64 ? run_paged_hd<KE, QE, 64>(who, a, max_keys) : run_paged_hd<KE, QE, 128>(who, a, max_keys);
}

} // namespace
} // namespace ncmb

using namespace ncmb;

extern "C" int ncmb_paged_attention(const NcmbPaged *c, const void *q, int64_t ldq, void *out, int64_t ldo, int act_type, int n_head, int T,
                                    const int *parents, float scale, int max_len) {
    const char *who = "ncmb_paged_attention";
    PagedDev d;
    if (paged_check(who, c, d)) return -1;
    const int cap = c->max_pages * c->page;
    if (act_type != NCMB_F32 && !(act_type == NCMB_BF16 && c->type == NCMB_BF16)) return cache_refuse(who, "activations of type %d with a cache of type %d", act_type, c->type);
    if (n_head < 1 || n_head % c->n_kv) return cache_refuse(who, "%d heads over %d kv heads", n_head, c->n_kv);
    if (T < 1 || T > NCMB_MAX_NODES || T > cap) return cache_refuse(who, "%d new tokens: 1 to %d, and no more than a row's pages hold", T, NCMB_MAX_NODES);
    if ((int64_t)T * (n_head / c->n_kv) > 1 << 30) return cache_refuse(who, "%d new tokens of %d heads a kv head", T, n_head / c->n_kv);
    const int64_t es = act_type == NCMB_BF16 ? 2 : 4;
    if (!q || !out || ((uintptr_t)q | (uintptr_t)out) % 16 || (ldq * es) % 16 || (ldo * es) % 16 || ldq < (int64_t)n_head * c->hd || ldo < (int64_t)n_head * c->hd)
        return cache_refuse(who, "q and out have to be 16-byte aligned, with rows of n_head * hd at multiples of 16 bytes");
    if ((uintptr_t)parents % 4) return cache_refuse(who, "parents have to be 4-byte aligned");
    if (!(fabsf(scale) < INFINITY)) return cache_refuse(who, "scale %g", scale);
    if (c->rows == 0) return 0;
    if (cache_device(who)) return -1;
    CmArgs a = {};
    a.c = CacheDev{d.k, d.v, 0, d.hs, d.ts, d.rows, d.nkv, d.hd, cap, d.len};
    a.table = d.table; a.table_stride = d.table_stride; a.ps = d.ps; a.page_log = d.page_log; a.n_pages = d.n_pages; a.max_pages = d.max_pages;
    a.q = (const char *)q; a.out = (char *)out; a.ldq = ldq * es; a.ldo = ldo * es;
    a.H = n_head; a.G = n_head / c->n_kv; a.T = T; a.M = T * a.G; a.parents = parents;
    a.c2 = (scale == 0.f ? 1.0f / sqrtf((float)c->hd) : scale) * 1.44269504f;
    if (max_len <= 0 || max_len > cap - T) max_len = cap - T;
    const double keys = (double)c->rows * c->n_kv * (max_len + T);      // by the bound: lengths are on the device
    ProfScope prof(NCMB_K_ATTN, 4.0 * keys * a.M * c->hd, 2.0 * keys * c->hd * d.es);
    if (c->type == NCMB_F32) return run_paged<float, float>(who, a, max_len + T);
    if (act_type == NCMB_F32) return run_paged<__nv_bfloat16, float>(who, a, max_len + T);
    return run_paged<__nv_bfloat16, __nv_bfloat16>(who, a, max_len + T);
}
