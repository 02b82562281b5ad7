// Index arithmetic of paged caches, shared by the kernels and the host (plain C++: it also compiles without nvcc).
//
// A pool holds num_pages pages of [num_kv_heads, page_rows, head_dim] elements per tensor; a block table row lists the
// pages of a request in the order of its positions.
#pragma once
#include <stddef.h>

#ifdef __CUDACC__
#define SHAINET_HD __host__ __device__ __forceinline__
#else
#define SHAINET_HD inline
#endif

namespace shainet {

constexpr int PAGED_MAX_PAGE_ROWS = 4096;

// A table cell is followed, and a slot used, only where it lies in the pool.
SHAINET_HD bool page_in_pool(int page, int num_pages) { return page >= 0 && page < num_pages; }
SHAINET_HD bool slot_in_pool(int slot, int num_pages, int page_rows) {
    return slot >= 0 && slot < (long long)num_pages * page_rows;
}

// A length that a table row can hold, max_len positions at most; anything else is an empty request.
SHAINET_HD int max_len_of(int table_width, int page_rows) {
    const long long n = (long long)table_width * page_rows;
    return n < 0x7fffffff ? (int)n : 0x7fffffff;
}
SHAINET_HD int valid_len(int len, int max_len) { return (unsigned)len <= (unsigned)max_len ? len : 0; }

// Quotient by page_rows without a division: n / d for 0 <= n < 2^31, 1 <= d <= 2^31 as (n * mul) >> shift, with
// shift = 31 + ceil(log2 d) and mul = ceil(2^shift / d) (Granlund and Montgomery 1994: mul * d exceeds 2^shift by less
// than d <= 2^(shift - 31), so the error of n * mul / 2^shift stays below 1 / d).
struct FastDiv {
    unsigned mul;
    int shift;
};
inline FastDiv fast_div(int d) {
    FastDiv f;
    f.shift = 31;
    while ((1ll << (f.shift - 31)) < d) ++f.shift;
    f.mul = (unsigned)(((1ull << f.shift) + d - 1) / d);
    return f;
}
SHAINET_HD int divide(int n, FastDiv f) { return (int)(((unsigned long long)(unsigned)n * f.mul) >> f.shift); }

// Pages of n positions: n / page_rows rounded up.
SHAINET_HD int pages_of(int n, FastDiv by, int page_rows) {
    const int q = divide(n, by);
    return q + (n > q * page_rows ? 1 : 0);
}

// Row of a tensor's pool, in units of head_dim elements: 64 bits, a pool may hold more than 2^31 elements.
SHAINET_HD size_t pool_row(int page, int num_kv_heads, int kv_head, int page_rows, int row) {
    return ((size_t)page * num_kv_heads + kv_head) * page_rows + row;
}

}  // namespace shainet
