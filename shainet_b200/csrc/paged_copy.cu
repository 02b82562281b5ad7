// Rows between a contiguous cache [num_kv_heads, capacity, head_dim] and pages [num_pages, num_kv_heads, page_rows,
// head_dim] of the same element type: a prompt that ran on the cache moves into its pages by its slot map (scatter), the
// pages of a request come back for the next turn by its table row (gather).
//
// A copy: every byte is read once and written once, so HBM bounds it.  Rows are whole 16-byte pieces (128 to 512 bytes);
// neighbouring lanes take neighbouring pieces of a row, neighbouring rows of one kv head lie side by side on both sides
// within a page, so accesses are whole sectors at any page size.  Measured: 8192 bfloat16 rows of 8 heads x 128 scattered in 13.0 us
// (5.2 TB/s read and written, 80 % of a copy's rate; 14.3 with one row a thread), 1900 rows gathered in 3.7 us, a launch and its latency.
#include "kernels.h"

namespace shainet {

namespace {

constexpr int COPY_THREADS = 256;
constexpr int COPY_ROWS = 4;     // rows of a thread, all requested before the first is stored

template <bool SCATTER, int CHUNKS>   // CHUNKS: 16-byte pieces of a row
__global__ void __launch_bounds__(COPY_THREADS) paged_copy_kernel(PagedCopyArgs a) {
    constexpr int STEP = COPY_THREADS / CHUNKS;
    const int piece = threadIdx.x % CHUNKS, h = blockIdx.y;
    const int i0 = blockIdx.x * (STEP * COPY_ROWS) + threadIdx.x / CHUNKS;
    // The next kernel in the stream is not let in before this one's last stores have been issued; that they can be seen is
    // promised to its own wait alone, so the launch behind a gather reads no row of that cache ahead of it.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    size_t at_page[COPY_ROWS];
    bool on[COPY_ROWS];
#pragma unroll
    for (int k = 0; k < COPY_ROWS; ++k) {
        const int i = i0 + k * STEP;
        on[k] = i < a.rows;
        if (SCATTER) {
            const int slot = on[k] ? a.index[i] : -1;
            if (slot >= 0 && !slot_in_pool(slot, a.num_pages, a.page_rows)) report_bad_page(a.status, 11);
            on[k] = slot_in_pool(slot, a.num_pages, a.page_rows);
            const int page = divide(on[k] ? slot : 0, a.by_page);
            at_page[k] = pool_row(page, a.num_kv_heads, h, a.page_rows, (on[k] ? slot : 0) - page * a.page_rows) * CHUNKS + piece;
        } else {
            const int col = divide(on[k] ? i : 0, a.by_page), page = a.index[col];
            if (on[k] && !page_in_pool(page, a.num_pages)) {
                report_bad_page(a.status, 12);
                on[k] = false;
            }
            at_page[k] = pool_row(on[k] ? page : 0, a.num_kv_heads, h, a.page_rows, (on[k] ? i : 0) - (on[k] ? col * a.page_rows : 0)) * CHUNKS + piece;
        }
    }
    const size_t at_cache = ((size_t)h * a.capacity + a.row0 + i0) * CHUNKS + piece;
    uint4 *kp = static_cast<uint4*>(a.k_pages), *vp = static_cast<uint4*>(a.v_pages);
    uint4 *kc = static_cast<uint4*>(a.k_cache), *vc = static_cast<uint4*>(a.v_cache);
    uint4 k[COPY_ROWS], v[COPY_ROWS];
#pragma unroll
    for (int x = 0; x < COPY_ROWS; ++x)
        if (on[x]) {
            const size_t c = at_cache + (size_t)x * STEP * CHUNKS;
            k[x] = __ldcs(SCATTER ? kc + c : kp + at_page[x]);
            v[x] = __ldcs(SCATTER ? vc + c : vp + at_page[x]);
        }
#pragma unroll
    for (int x = 0; x < COPY_ROWS; ++x)
        if (on[x]) {
            const size_t c = at_cache + (size_t)x * STEP * CHUNKS;
            (SCATTER ? kp + at_page[x] : kc + c)[0] = k[x];
            (SCATTER ? vp + at_page[x] : vc + c)[0] = v[x];
        }
}

template <bool SCATTER, int CHUNKS>
cudaError_t launch(const PagedCopyArgs& a, cudaStream_t s) {
    const int per = COPY_THREADS / CHUNKS * COPY_ROWS;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((a.rows + per - 1) / per, a.num_kv_heads);
    cfg.blockDim = dim3(COPY_THREADS);
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, paged_copy_kernel<SCATTER, CHUNKS>, a);
}

}  // namespace

cudaError_t launch_paged_copy(PagedCopyArgs a, bool scatter, cudaStream_t s) {
    a.by_page = fast_div(a.page_rows);
    switch (a.row_bytes) {
        case 128: return scatter ? launch<true, 8>(a, s) : launch<false, 8>(a, s);
        case 256: return scatter ? launch<true, 16>(a, s) : launch<false, 16>(a, s);
        case 512: return scatter ? launch<true, 32>(a, s) : launch<false, 32>(a, s);
    }
    return cudaErrorInvalidValue;
}

}  // namespace shainet
