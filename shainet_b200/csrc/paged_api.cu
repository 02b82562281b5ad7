// Host side of the paged entries of include/shainet_attn.h: argument checks, handles, launches.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <new>

#include "host_state.h"
#include "paged_index.h"

using namespace shainet;

struct shainet_attn_paged {
    shainet_attn_ctx* ctx = nullptr;
    HeadShape hs{};
    int page_rows = 0;
    int es = 4;
    PagedPlan plan{};
    float* workspace = nullptr;     // device, plan.part_floats
    unsigned* counters = nullptr;   // device, 3 * plan.ctas, zero between calls
};

namespace {

bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

int check_pool(int num_pages, int page_rows) {
    if (page_rows < 1 || page_rows > PAGED_MAX_PAGE_ROWS)
        return fail(SHAINET_ATTN_E_INVALID, "page_rows %d outside [1, %d]", page_rows, PAGED_MAX_PAGE_ROWS);
    if (num_pages < 1 || (long long)num_pages * page_rows > 0x7fffffffll)
        return fail(SHAINET_ATTN_E_INVALID, "%d pages of %d rows: the pool holds 1 to 2^31 - 1 rows", num_pages, page_rows);
    return SHAINET_ATTN_OK;
}

int check_table(int requests, int table_width) {
    if (table_width < 1) return fail(SHAINET_ATTN_E_INVALID, "table_width %d < 1", table_width);
    if ((long long)requests * table_width > 0x7fffffffll)
        return fail(SHAINET_ATTN_E_INVALID, "a block table of %d x %d cells is larger than 2^31 - 1", requests, table_width);
    return SHAINET_ATTN_OK;
}

// What decode and the copies share: the handle fits the context, the pool and the block's cache.
int check_paged(shainet_attn_ctx* ctx, const shainet_attn_paged* paged, const shainet_attn_kv* kv, const void* k_pages,
                const void* v_pages, int num_pages) {
    if (!ctx || !paged || !kv) return fail(SHAINET_ATTN_E_INVALID, "null context, handle or cache");
    if (paged->ctx != ctx || kv->ctx != ctx) return fail(SHAINET_ATTN_E_INVALID, "handle or cache belongs to another context");
    if (kv->hs.num_heads != paged->hs.num_heads || kv->hs.num_kv_heads != paged->hs.num_kv_heads ||
        kv->hs.head_dim != paged->hs.head_dim || kv->es != paged->es)
        return fail(SHAINET_ATTN_E_INVALID, "the cache's head layout or format is not the handle's");
    if (!k_pages || !v_pages) return fail(SHAINET_ATTN_E_INVALID, "null page pointer");
    if (!aligned16(k_pages) || !aligned16(v_pages)) return fail(SHAINET_ATTN_E_INVALID, "page pointers must be 16-byte aligned");
    int rc = check_pool(num_pages, paged->page_rows);
    if (!rc && (unsigned long long)num_pages * paged->page_rows * paged->hs.num_kv_heads > 0xfffffffeull)   // row numbers of the kernels: 32 bits
        rc = fail(SHAINET_ATTN_E_UNSUPPORTED, "%d pages of %d rows and %d kv heads: a pool holds at most 2^32 - 2 rows of all heads", num_pages,
                  paged->page_rows, paged->hs.num_kv_heads);
    return rc;
}

// A paged call's kernel touches nothing before all work ahead of it in the stream is complete, and lets the next kernel
// launch only then or at its end.  (What the kernel itself has written, the rows of a gather, counts for the next one only
// behind that one's own wait.)
int copy_rows(shainet_attn_ctx* ctx, const shainet_attn_paged* paged, const shainet_attn_kv* kv, void* k_pages, void* v_pages,
              int num_pages, const int32_t* index, int row0, int rows, bool scatter, cudaStream_t s) {
    PagedCopyArgs a{};
    a.k_pages = k_pages;
    a.v_pages = v_pages;
    a.k_cache = kv->k;
    a.v_cache = kv->v;
    a.index = index;
    a.num_pages = num_pages;
    a.page_rows = paged->page_rows;
    a.num_kv_heads = paged->hs.num_kv_heads;
    a.capacity = kv->cap;
    a.row0 = row0;
    a.rows = rows;
    a.row_bytes = paged->hs.head_dim * paged->es;
    a.status = ctx->status_dev;
    CU(launch_paged_copy(a, scatter, s));
    return SHAINET_ATTN_OK;
}

// decode_lens: nullable where the step is not asked for them (step_dev asks).
int plan_step(shainet_attn_ctx* ctx, int requests, const int32_t* lens, const int32_t* delta, int32_t* block_table, int table_width,
              int page_rows, int32_t* free_pages, int num_pages, const int32_t* free_count, int32_t* lens_out, int32_t* free_count_out,
              int32_t* first, int32_t* slots, int max_tokens, int32_t* decode_lens, int32_t* status, void* stream) {
    if (requests < 0) return fail(SHAINET_ATTN_E_INVALID, "requests %d < 0", requests);
    if (requests > SHAINET_ATTN_PAGED_MAX_REQUESTS)
        return fail(SHAINET_ATTN_E_UNSUPPORTED, "%d requests: a step plans at most %d", requests, SHAINET_ATTN_PAGED_MAX_REQUESTS);
    if (max_tokens < 0) return fail(SHAINET_ATTN_E_INVALID, "max_tokens %d < 0", max_tokens);
    int rc = check_pool(num_pages, page_rows);
    if (!rc) rc = check_table(requests, table_width);
    if (rc) return rc;
    if ((requests > 0 && (!lens || !delta || !block_table || !lens_out)) || !free_pages || !free_count || !free_count_out || !first ||
        (max_tokens > 0 && !slots) || !status)
        return fail(SHAINET_ATTN_E_INVALID, "null array");
    for (const void* p : {(const void*)lens, (const void*)delta, (const void*)block_table, (const void*)free_pages, (const void*)free_count,
                          (const void*)lens_out, (const void*)free_count_out, (const void*)first, (const void*)slots, (const void*)decode_lens,
                          (const void*)status})
        if (!aligned4(p)) return fail(SHAINET_ATTN_E_INVALID, "int32 arrays must be 4-byte aligned");
    if (!ctx) return fail(SHAINET_ATTN_E_INVALID, "null context");
    DeviceGuard g(ctx->device);
    PagedPlanArgs a{};
    a.lens = lens;
    a.delta = delta;
    a.block_table = block_table;
    a.free_pages = free_pages;
    a.free_count = free_count;
    a.lens_out = lens_out;
    a.free_count_out = free_count_out;
    a.first = first;
    a.slots = slots;
    a.decode_lens = decode_lens;
    a.status = status;
    a.requests = requests;
    a.table_width = table_width;
    a.page_rows = page_rows;
    a.num_pages = num_pages;
    a.max_tokens = max_tokens;
    CU(launch_paged_plan(a, stream ? (cudaStream_t)stream : ctx->stream));
    return SHAINET_ATTN_OK;
}

}  // namespace

extern "C" {

int shainet_attn_paged_plan_dev(shainet_attn_ctx* ctx, int requests, const int32_t* lens, const int32_t* delta,
                                int32_t* block_table, int table_width, int page_rows, int32_t* free_pages, int num_pages,
                                const int32_t* free_count, int32_t* lens_out, int32_t* free_count_out, int32_t* first,
                                int32_t* slots, int max_tokens, int32_t* status, void* stream) {
    return plan_step(ctx, requests, lens, delta, block_table, table_width, page_rows, free_pages, num_pages, free_count, lens_out,
                     free_count_out, first, slots, max_tokens, nullptr, status, stream);
}

int shainet_attn_paged_step_dev(shainet_attn_ctx* ctx, int requests, const int32_t* lens, const int32_t* delta,
                                int32_t* block_table, int table_width, int page_rows, int32_t* free_pages, int num_pages,
                                const int32_t* free_count, int32_t* lens_out, int32_t* free_count_out, int32_t* first,
                                int32_t* slots, int max_tokens, int32_t* decode_lens, int32_t* status, void* stream) {
    if (requests > 0 && (!decode_lens || decode_lens == lens || decode_lens == lens_out))
        return fail(SHAINET_ATTN_E_INVALID, "decode_lens is null or one of the arrays of the lengths");
    return plan_step(ctx, requests, lens, delta, block_table, table_width, page_rows, free_pages, num_pages, free_count, lens_out,
                     free_count_out, first, slots, max_tokens, decode_lens, status, stream);
}

int shainet_attn_paged_create(shainet_attn_ctx* ctx, shainet_attn_paged** out, int num_heads, int num_kv_heads, int head_dim,
                              int page_rows, int format) {
    if (!out) return fail(SHAINET_ATTN_E_INVALID, "null pointer");
    *out = nullptr;
    if (num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0)
        return fail(SHAINET_ATTN_E_INVALID, "%d query heads over %d kv heads", num_heads, num_kv_heads);
    if (head_dim != 64 && head_dim != 128)
        return fail(SHAINET_ATTN_E_UNSUPPORTED, "head_dim %d: paged attention needs head_dim 64 or 128", head_dim);
    if (format != SHAINET_ATTN_KV_F32 && format != SHAINET_ATTN_KV_BF16) return fail(SHAINET_ATTN_E_INVALID, "unknown cache format %d", format);
    int rc = check_pool(1, page_rows);
    if (rc) return rc;
    if (!ctx) return fail(SHAINET_ATTN_E_INVALID, "null context");
    shainet_attn_paged* p = new (std::nothrow) shainet_attn_paged();
    if (!p) return fail(SHAINET_ATTN_E_NOMEM, "out of host memory");
    p->ctx = ctx;
    p->hs = HeadShape{num_heads, num_kv_heads, head_dim};
    p->page_rows = page_rows;
    p->es = format == SHAINET_ATTN_KV_BF16 ? 2 : 4;
    p->plan = paged_decode_plan(p->hs, p->es, ctx->sm_count);
    ctx->live_caches++;
    DeviceGuard g(ctx->device);
    cudaError_t e = cudaMalloc(&p->workspace, p->plan.part_floats * sizeof(float));
    if (e == cudaSuccess) e = cudaMalloc(&p->counters, 3 * p->plan.ctas * sizeof(unsigned));
    if (e == cudaSuccess) e = cudaMemsetAsync(p->counters, 0, 3 * p->plan.ctas * sizeof(unsigned), ctx->stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize(ctx->stream);
    if (e != cudaSuccess) {
        shainet_attn_paged_destroy(p);
        return fail_cuda(e, "workspace of a paged handle");
    }
    *out = p;
    return SHAINET_ATTN_OK;
}

int shainet_attn_paged_destroy(shainet_attn_paged* p) {
    if (!p) return SHAINET_ATTN_OK;
    DeviceGuard g(p->ctx->device);
    cudaStreamSynchronize(p->ctx->stream);
    if (p->workspace) cudaFree(p->workspace);
    if (p->counters) cudaFree(p->counters);
    cudaGetLastError();
    p->ctx->live_caches--;
    delete p;
    return SHAINET_ATTN_OK;
}

int shainet_attn_paged_decode_dev(shainet_attn_ctx* ctx, shainet_attn_paged* paged, const shainet_attn_kv* kv, void* k_pages,
                                  void* v_pages, int num_pages, const float* q, const float* k_new, const float* v_new, float* out,
                                  const int32_t* block_table, int table_width, const int32_t* lens, int requests, float scale,
                                  void* stream) {
    if (requests < 0) return fail(SHAINET_ATTN_E_INVALID, "requests %d < 0", requests);
    int rc = check_table(requests, table_width);
    if (!rc) rc = check_paged(ctx, paged, kv, k_pages, v_pages, num_pages);
    if (rc || requests == 0) return rc;
    if (!q || !k_new || !v_new || !out || !block_table || !lens) return fail(SHAINET_ATTN_E_INVALID, "null tensor pointer");
    if (!aligned16(q) || !aligned16(k_new) || !aligned16(v_new) || !aligned16(out))
        return fail(SHAINET_ATTN_E_INVALID, "device pointers must be 16-byte aligned");
    if (!aligned4(block_table) || !aligned4(lens)) return fail(SHAINET_ATTN_E_INVALID, "int32 arrays must be 4-byte aligned");
    DeviceGuard g(ctx->device);
    PagedDecodeArgs a{};
    a.k_pages = k_pages;
    a.v_pages = v_pages;
    a.num_pages = num_pages;
    a.page_rows = paged->page_rows;
    a.q = q;
    a.k_new = k_new;
    a.v_new = v_new;
    a.b_q = kv->b_q;
    a.b_k = kv->b_k;
    a.b_v = kv->b_v;
    a.q_norm = kv->q_norm;
    a.k_norm = kv->k_norm;
    a.inv_freq = kv->inv_freq;
    a.eps = kv->eps;
    a.out = out;
    a.block_table = block_table;
    a.table_width = table_width;
    a.lens = lens;
    a.requests = requests;
    a.hs = paged->hs;
    a.scale = scale;
    a.kv_elem_bytes = paged->es;
    a.status = ctx->status_dev;
    CU(launch_paged_decode(a, paged->plan, paged->workspace, paged->counters, stream ? (cudaStream_t)stream : ctx->stream));
    return SHAINET_ATTN_OK;
}

int shainet_attn_paged_scatter_dev(shainet_attn_ctx* ctx, shainet_attn_paged* paged, const shainet_attn_kv* kv, void* k_pages,
                                   void* v_pages, int num_pages, const int32_t* slots, int row0, int rows, void* stream) {
    if (row0 < 0 || rows < 0) return fail(SHAINET_ATTN_E_INVALID, "rows %d from %d", rows, row0);
    int rc = check_paged(ctx, paged, kv, k_pages, v_pages, num_pages);
    if (rc) return rc;
    if ((long long)row0 + rows > kv->len) return fail(SHAINET_ATTN_E_INVALID, "rows %d from %d of a cache of %d", rows, row0, kv->len);
    if (rows == 0) return SHAINET_ATTN_OK;
    if (!slots || !aligned4(slots)) return fail(SHAINET_ATTN_E_INVALID, "null or misaligned slots");
    DeviceGuard g(ctx->device);
    return copy_rows(ctx, paged, kv, k_pages, v_pages, num_pages, slots, row0, rows, true, stream ? (cudaStream_t)stream : ctx->stream);
}

int shainet_attn_paged_gather_dev(shainet_attn_ctx* ctx, shainet_attn_paged* paged, shainet_attn_kv* kv, const void* k_pages,
                                  const void* v_pages, int num_pages, const int32_t* table_row, int rows, void* stream) {
    if (rows < 0) return fail(SHAINET_ATTN_E_INVALID, "rows %d < 0", rows);
    int rc = check_paged(ctx, paged, kv, k_pages, v_pages, num_pages);
    if (rc) return rc;
    if (rows > 0 && (!table_row || !aligned4(table_row))) return fail(SHAINET_ATTN_E_INVALID, "null or misaligned table row");
    DeviceGuard g(ctx->device);
    cudaStream_t s = stream ? (cudaStream_t)stream : ctx->stream;
    if (rows > 0) {
        // a reserved cache maps whole tiles of 128 rows
        const bool grows = kv->reserved ? (size_t)std::min<long long>(kv->cap, (rows + 127ll) / 128 * 128) * kv->hs.head_dim * kv->es >
                                              kv->pages_per_head * kv->page_bytes
                                        : rows > kv->cap || !kv->k;
        cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
        CU(cudaStreamIsCapturing(s, &capture));
        if (grows && capture != cudaStreamCaptureStatusNone)
            return fail(SHAINET_ATTN_E_STATE, "the cache cannot grow to %d rows on a stream that is being captured", rows);
        rc = kv_ensure_rows(kv, rows, s);
        if (!rc)
            rc = copy_rows(ctx, paged, kv, const_cast<void*>(k_pages), const_cast<void*>(v_pages), num_pages, table_row, 0, rows, false, s);
        if (rc) return rc;
        if (capture != cudaStreamCaptureStatusNone) kv->refilled_by_graph = true;
    }
    kv->refilled = true;
    kv->len = rows;
    return SHAINET_ATTN_OK;
}

}  // extern "C"
