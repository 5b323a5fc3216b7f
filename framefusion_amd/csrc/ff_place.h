// Where a position of a sequence lies in the paged cache.  Plain C++: also compiled for the host by the tests.
#pragma once

#include <stdint.h>

#if defined(__HIPCC__)
#define FF_BOTH __device__ __host__
#else
#define FF_BOTH
#endif

namespace ff {

// Row of the cache that holds kv head `head` of position `pos`, counted in rows of dh channels from the start of the keys (or
// values); -1: the position has no place (negative, past the table, or its entry names no page).  The product is formed in 64
// bits: 2^31 rows are 550 GB of 16-bit keys at dh = 128, but 69 GB of 4-bit keys at dh = 64.
FF_BOTH inline int64_t cache_row(const int32_t* table, int64_t table_width, int64_t n_pages, int page_size, int kv_heads, int head,
                                 int64_t pos) {
    if (pos < 0 || pos >= table_width * page_size) return -1;
    const uint32_t p = (uint32_t)pos, slot = p / (uint32_t)page_size;
    const int32_t page = table[slot];
    if (page < 0 || page >= n_pages) return -1;
    return ((int64_t)page * kv_heads + head) * page_size + (p - slot * (uint32_t)page_size);
}

}  // namespace ff
