// Paged caches (paged_cache.cu, paged_attention.cu) as kernels see them.
#pragma once
#include "cache.cuh"

namespace ncmb {

struct PagedDev {
    char *k, *v;
    int64_t ps, hs, ts;              // strides in bytes
    int rows, nkv, hd, page_log, n_pages, max_pages, es;
    const int *table;
    int64_t table_stride;
    const int *len;
};
// whether two arrays share memory; none of no bytes, or that is not there, does
inline bool paged_overlap(const void *a, size_t na, const void *b, size_t nb) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return a && b && na && nb && x < y + nb && y < x + na;
}
// 0 when the cache's description is one the kernels take (see ncm_b200.h), else -1 with a message
int paged_check(const char *who, const NcmbPaged *c, PagedDev &d);

#ifdef __CUDACC__
// entry i of a row's table, -1 where it is no page
__device__ __forceinline__ int paged_entry(const PagedDev &c, int row, int i) {
    const int p = i < c.max_pages ? c.table[row * c.table_stride + i] : -1;
    return (unsigned)p < (unsigned)c.n_pages ? p : -1;
}
#endif

} // namespace ncmb
