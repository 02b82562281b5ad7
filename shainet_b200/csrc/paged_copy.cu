// Rows between a contiguous cache [num_kv_heads, capacity, head_dim] and pages [num_pages, num_kv_heads, page_rows,
// head_dim] of the same element type: a prompt that ran on the cache moves into its pages by its slot map (scatter), the
// pages of a request come back for the next turn by its table row (gather).
//
// A copy: every byte is read once and written once, so HBM bounds it.  Rows are whole 16-byte pieces (128 to 512 bytes);
// neighbouring lanes take neighbouring pieces of a row, neighbouring rows of one kv head lie side by side on both sides
// within a page, so accesses are whole sectors at any page size.
#include "kernels.h"
#include "paged_index.h"

namespace shainet {

namespace {

constexpr int COPY_THREADS = 256;

template <bool SCATTER, int CHUNKS>   // CHUNKS: 16-byte pieces of a row
__global__ void __launch_bounds__(COPY_THREADS) paged_copy_kernel(PagedCopyArgs a) {
    const int piece = threadIdx.x % CHUNKS;
    const int i = blockIdx.x * (COPY_THREADS / CHUNKS) + threadIdx.x / CHUNKS;
    const int h = blockIdx.y;
    if (i >= a.rows) return;
    int page, row;
    if (SCATTER) {
        const int slot = a.index[i];
        if (slot < 0) return;
        if (!slot_in_pool(slot, a.num_pages, a.page_rows)) {
            report_status(a.status, DEV_BAD_PAGE, 11);
            return;
        }
        page = slot / a.page_rows;
        row = slot - page * a.page_rows;
    } else {
        page = a.index[i / a.page_rows];
        row = i % a.page_rows;
        if (!page_in_pool(page, a.num_pages)) {
            report_status(a.status, DEV_BAD_PAGE, 12);
            return;
        }
    }
    const size_t at_page = pool_row(page, a.num_kv_heads, h, a.page_rows, row) * CHUNKS + piece;
    const size_t at_cache = ((size_t)h * a.capacity + a.row0 + i) * CHUNKS + piece;
    if (SCATTER) {
        const uint4 k = reinterpret_cast<const uint4*>(a.k_cache)[at_cache], v = reinterpret_cast<const uint4*>(a.v_cache)[at_cache];
        reinterpret_cast<uint4*>(a.k_pages)[at_page] = k;
        reinterpret_cast<uint4*>(a.v_pages)[at_page] = v;
    } else {
        const uint4 k = reinterpret_cast<const uint4*>(a.k_pages)[at_page], v = reinterpret_cast<const uint4*>(a.v_pages)[at_page];
        reinterpret_cast<uint4*>(a.k_cache)[at_cache] = k;
        reinterpret_cast<uint4*>(a.v_cache)[at_cache] = v;
    }
}

template <bool SCATTER, int CHUNKS>
cudaError_t launch(const PagedCopyArgs& a, cudaStream_t s) {
    const int per = COPY_THREADS / CHUNKS;
    const dim3 grid((a.rows + per - 1) / per, a.num_kv_heads);
    paged_copy_kernel<SCATTER, CHUNKS><<<grid, COPY_THREADS, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_paged_copy(const PagedCopyArgs& a, bool scatter, cudaStream_t s) {
    switch (a.row_bytes) {
        case 128: return scatter ? launch<true, 8>(a, s) : launch<false, 8>(a, s);
        case 256: return scatter ? launch<true, 16>(a, s) : launch<false, 16>(a, s);
        case 512: return scatter ? launch<true, 32>(a, s) : launch<false, 32>(a, s);
    }
    return cudaErrorInvalidValue;
}

}  // namespace shainet
