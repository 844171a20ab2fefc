// paged.cuh -- the page table of a paged block cache, shared by the kernels
// that write, read back, attend to and thin out such a cache (sm_100a).
//
// Pools are [pages, Hkv, page_size, record]; token t of sequence b lies in
// page table[b][t / page_size] at slot t % page_size.
#pragma once
#include "ecc_common.cuh"

namespace ecc {

// Unsigned 32-bit division by a runtime constant d >= 1 (round-up method:
// s = ceil(log2 d), m = floor(2^32 (2^s - d) / d) + 1, q = (umulhi(n,m) + n) >> s),
// valid for every n < 2^32.
struct FastDiv {
    uint32_t d, m, s;
};
static inline FastDiv make_fastdiv(uint32_t d) {
    FastDiv f;
    f.d = d;
    f.s = 0;
    while ((1ull << f.s) < d) ++f.s;
    f.m = (uint32_t)((((1ull << 32) * ((1ull << f.s) - d)) / d) + 1);
    return f;
}
__device__ __forceinline__ uint32_t fdiv(uint32_t n, FastDiv f) {
    return (uint32_t)(((uint64_t)__umulhi(n, f.m) + n) >> f.s);
}

namespace paged {

// A length, position or page number out of range (one flag per translation
// unit; ecc_device_status reports 5 for any of them).
static __device__ int g_paged_error;

struct PageTable {
    const int *table;  // [B][stride], width columns used
    int64_t stride;
    int width, page_size, n_pages;
    int capacity;  // tokens a row of the table can name
    FastDiv div;
    __device__ __forceinline__ uint32_t page_of(int t) const { return fdiv((uint32_t)t, div); }
    // page of token t < capacity of sequence b, or -1 (flagged) when the table names none
    __device__ __forceinline__ int page(int b, int t, int &slot) const {
        const uint32_t pi = page_of(t);
        slot = t - (int)pi * page_size;
        const int p = __ldg(table + b * stride + pi);
        if ((uint32_t)p < (uint32_t)n_pages) return p;
        atomicExch(&g_paged_error, 5);
        return -1;
    }
};

static inline int make_table(const ecc_pages_t &p, PageTable *t) {
    if (!p.table) return ECC_ERR_NULL;
    if (p.width < 1 || p.page_size < 1 || p.n_pages < 1 || p.n_pages >= (1ll << 31)) return ECC_ERR_SHAPE;
    // a 16-token group never straddles two pages; one page per sequence may have any size
    if (p.width > 1 && p.page_size % 16) return ECC_ERR_SHAPE;
    if ((int64_t)p.width * p.page_size > (1ll << 30)) return ECC_ERR_SHAPE;
    if ((uintptr_t)p.table % 4) return ECC_ERR_ALIGN;
    t->table = p.table;
    t->stride = p.table_stride;
    t->width = p.width;
    t->page_size = p.page_size;
    t->n_pages = (int)p.n_pages;
    t->capacity = p.width * p.page_size;
    t->div = make_fastdiv((uint32_t)p.page_size);
    return ECC_OK;
}

}  // namespace paged
}  // namespace ecc
