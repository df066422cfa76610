// Paged key-value cache: where a row's slot lies (include/mmhip.h, "paged key-value cache").
#pragma once
#include "common.h"

struct PagedMap {
    const int* table; long ld; int width, shift, n_pages, Hkv;   // page = 1 << shift
    // row index in the pool ([n_pages][Hkv][page] rows) of slot `slot` of row b, or -1 where the slot does not exist
    __device__ __forceinline__ long row(int b, int hkv, int slot) const {
        const int e = slot >> shift;
        if (slot < 0 || e >= width) return -1;
        const int pg = table[(long)b * ld + e];
        if ((unsigned)pg >= (unsigned)n_pages) return -1;
        return (((long)pg * Hkv + hkv) << shift) + (slot & ((1 << shift) - 1));
    }
    __device__ __forceinline__ int capacity() const { return width << shift; }
};

// log2(page) if it is a power of two in [4, 1024], else -1
static inline int paged_shift(int64_t page) {
    for (int s = 2; s <= 10; s++) if (page == (1 << s)) return s;
    return -1;
}
// whether what B rows' tables can name is more than the last-level cache (256 MB) holds: never more than the pool has, however wide the
// tables are and however many rows share a page
static inline bool paged_past_cache(int64_t B, int64_t Hkv, int64_t d, int64_t page, int64_t n_pages, int64_t width, int dtype) {
    return (B * width < n_pages ? B * width : n_pages) > (256LL << 20) / (page * Hkv * d * (dtype == MM_BF16 ? 4 : 8));
}
// what every entry point asks of a pool and its table; 0 or a negative code with the message set
static inline int paged_check(const char* who, const void* kpool, const void* vpool, const int* table, int64_t B, int64_t Hkv, int64_t d,
                              int64_t page, int64_t n_pages, int64_t width, int64_t ld_table, int dtype) {
    MM_CHECK(dtype == MM_F32 || dtype == MM_BF16, "%s: bad dtype %d", who, dtype);
    MM_CHECK(B >= 0 && B <= 65535 && Hkv > 0 && Hkv <= 65535, "%s: B=%lld Hkv=%lld (at most 65535 of each)", who, (long long)B, (long long)Hkv);
    MM_CHECK(d > 0 && d <= 512 && d % 4 == 0, "%s: head_dim %lld (a multiple of 4, at most 512)", who, (long long)d);
    MM_CHECK(paged_shift(page) >= 0, "%s: page size %lld (a power of two, 4 to 1024)", who, (long long)page);
    MM_CHECK(n_pages > 0 && n_pages < (1LL << 31), "%s: n_pages=%lld", who, (long long)n_pages);
    MM_CHECK(width > 0 && width * page < (1LL << 30) && ld_table >= 0, "%s: table width %lld (at most 2^30 slots)", who, (long long)width);
    MM_CHECK(B == 0 || (kpool && vpool && table), "%s: null pointer", who);
    MM_CHECK((((uintptr_t)kpool | (uintptr_t)vpool) % 16) == 0, "%s: the pools must be 16-byte aligned", who);
    return MM_OK;
}
