// Block tables and slot maps of a batch of requests, built on the device from the requests' lengths, sm_100a.
//
// Per request r with length l, change d and pages of P rows: before = ceil(l / P), after = ceil((l + d) / P); the request
// grows by max(after - before, 0) pages, frees max(before - after, 0) and has max(d, 0) new tokens.  Exclusive sums of
// the three over the requests give every page that moves and every token its place, so after one scan all cells of the
// outputs are independent: the i-th page a request grows by is entry f + freed - 1 - i of the stack that the f free
// pages and the freed ones behind them form; the page of a new token comes from the request's old table row or, by the
// same index, from the stack.  A freed page that is popped again in the same step is looked up in the table row that
// frees it, never in the stack cell that is being written, so nothing waits for a write of this launch.
//
// What bounds it is latency, not bytes (a few hundred KB at most): one round of loads, a scan over at most 8192 requests
// that every CTA does for itself in shared memory, one or two dependent loads per output.  Steps are spread over one cluster
// of eight CTAs, whose barrier separates the reads of lens and free_count from the writes of lens_out and free_count_out,
// which may be the same arrays; the smallest ones take one CTA.  Measured: 8 requests 2.7 us, 256 requests with
// 15000 new tokens 6.1 us, of which an empty launch is 2.
#include <algorithm>
#include <atomic>
#include "../../include/shainet_attn.h"
#include "kernels.h"

namespace shainet {

namespace {

constexpr int PLAN_THREADS = 1024;      // at most; a small step takes 256
constexpr int PLAN_CLUSTER = 8;
constexpr unsigned FULL = 0xffffffffu;
enum PlanStatus { PLAN_OK = 0, PLAN_SHORT = 1, PLAN_LENGTH = 2, PLAN_TOKENS = 3, PLAN_STACK = 4 };

struct Sums {
    long long tokens;
    int grow, shrink;
};

__device__ __forceinline__ Sums operator+(Sums a, Sums b) { return {a.tokens + b.tokens, a.grow + b.grow, a.shrink + b.shrink}; }

// Sums over the lanes up to this one.
__device__ __forceinline__ Sums scan_warp(Sums v, int lane) {
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const Sums up{__shfl_up_sync(FULL, v.tokens, off), __shfl_up_sync(FULL, v.grow, off), __shfl_up_sync(FULL, v.shrink, off)};
        if (lane >= off) v = v + up;
    }
    return v;
}
__device__ __forceinline__ Sums of_lane(Sums v, int from) {
    return {__shfl_sync(FULL, v.tokens, from), __shfl_sync(FULL, v.grow, from), __shfl_sync(FULL, v.shrink, from)};
}

// The last r with sums[r] <= x (sums is non-decreasing, sums[0] == 0): the request that owns element x.
__device__ __forceinline__ int owner_of(const int* sums, int n, int x) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (sums[mid] <= x) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

__device__ __forceinline__ Sums change_of(int len, int delta, FastDiv by, int page_rows) {
    const int before = pages_of(len, by, page_rows), after = pages_of(len + delta, by, page_rows);
    return {delta > 0 ? delta : 0, after > before ? after - before : 0, before > after ? before - after : 0};
}

__global__ void __launch_bounds__(PLAN_THREADS) paged_plan_kernel(PagedPlanArgs a) {
    extern __shared__ int plan_smem[];
    const int R = a.requests, P = a.page_rows, T = blockDim.x, W = T / 32;
    int* s_len = plan_smem;
    int* s_delta = s_len + R;
    int* s_new = s_delta + R;     // exclusive sums over the requests
    int* s_grow = s_new + R;
    int* s_shrink = s_grow + R;
    __shared__ Sums warp_sums[32];
    __shared__ int s_bad;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) s_bad = R;
    // the arrays may come from the kernel ahead in the stream; the next one may launch and wait for this one's end
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int f = a.free_count[0];
    __syncthreads();
    // a length or step that does not fit becomes an empty request and ends in an error below
    for (int r = tid; r < R; r += T) {
        int len = a.lens[r], delta = a.delta[r];
        const long long after = (long long)len + delta;
        if ((unsigned)len > (unsigned)a.max_len || after < 0 || after > a.max_len) {
            atomicMin(&s_bad, r);
            delta = 0;
        }
        s_len[r] = len;
        s_delta[r] = delta;
    }
    // a thread sums a run of requests, the runs are scanned over the CTA
    const int run = (R + T - 1) / T, r0 = min(tid * run, R), r1 = min(r0 + run, R);
    if (run > 1) __syncthreads();
    auto change = [&](int r) {
        const int len = s_len[r];
        return (unsigned)len > (unsigned)a.max_len ? Sums{0, 0, 0} : change_of(len, s_delta[r], a.by_page, P);
    };
    Sums mine{0, 0, 0};
    for (int r = r0; r < r1; ++r) mine = mine + change(r);
    const Sums incl = scan_warp(mine, lane);
    if (lane == 31) warp_sums[warp] = incl;
    __syncthreads();
    const Sums warps = scan_warp(lane < W ? warp_sums[lane] : Sums{0, 0, 0}, lane);
    const Sums total = of_lane(warps, 31), base = of_lane(warps, warp > 0 ? warp - 1 : 0);
    Sums at{incl.tokens - mine.tokens, incl.grow - mine.grow, incl.shrink - mine.shrink};
    if (warp > 0) at = at + base;
    for (int r = r0; r < r1; ++r) {
        s_new[r] = (int)at.tokens;     // exact where it is used: the total is at most max_tokens
        s_grow[r] = at.grow;
        s_shrink[r] = at.shrink;
        at = at + change(r);
    }
    __syncthreads();
    const int freed = total.shrink;
    const long long left = (long long)f + freed - total.grow;
    int code = PLAN_OK, detail = 0;
    if (s_bad < R) code = PLAN_LENGTH, detail = s_bad;
    else if (f < 0 || (long long)f + freed > a.num_pages) code = PLAN_STACK, detail = f;
    else if (total.tokens > a.max_tokens) code = PLAN_TOKENS, detail = (int)min(total.tokens, (long long)0x7fffffff);
    else if (left < 0) code = PLAN_SHORT, detail = (int)-left;

    // every CTA has read lens and free_count before any writes lens_out and free_count_out
    int ctas = 1, rank = 0;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    if (ctas > 1)
        asm volatile("barrier.cluster.arrive.aligned;\n barrier.cluster.wait.aligned;" ::: "memory");

    const unsigned t0 = rank * T + tid, step = ctas * T;               // unsigned: the last step may pass 2^31
    const bool ok = code == PLAN_OK;
    if (t0 == 0) {
        a.status[0] = code;
        a.status[1] = detail;
        a.free_count_out[0] = ok ? (int)left : f;
        a.first[R] = ok ? (int)total.tokens : 0;
    }
    for (unsigned r = t0; r < R; r += step) {
        a.lens_out[r] = s_len[r] + (ok ? s_delta[r] : 0);
        a.first[r] = ok ? s_new[r] : 0;
        if (a.decode_lens) a.decode_lens[r] = ok && s_delta[r] == 1 ? s_len[r] + 1 : 0;
    }
    if (!ok) {
        for (unsigned t = t0; t < a.max_tokens; t += step) a.slots[t] = -1;
        return;
    }
    // the k-th freed page
    auto freed_page = [&](int k) {
        const int r = owner_of(s_shrink, R, k);
        return a.block_table[(size_t)r * a.table_width + pages_of(s_len[r] + s_delta[r], a.by_page, P) + k - s_shrink[r]];
    };
    // the i-th page that is popped
    auto popped_page = [&](int i) {
        const int at = f + freed - 1 - i;
        return at < f ? a.free_pages[at] : freed_page(at - f);
    };
    for (unsigned k = t0; k < freed; k += step) a.free_pages[f + k] = freed_page(k);
    for (unsigned i = t0; i < total.grow; i += step) {
        const int r = owner_of(s_grow, R, i);
        a.block_table[(size_t)r * a.table_width + pages_of(s_len[r], a.by_page, P) + i - s_grow[r]] = popped_page(i);
    }
    for (unsigned t = t0; t < a.max_tokens; t += step) {
        int slot = -1;
        if (t < total.tokens) {
            const int r = owner_of(s_new, R, t);
            const int pos = s_len[r] + (t - s_new[r]), col = divide(pos, a.by_page), before = pages_of(s_len[r], a.by_page, P);
            const int page = col < before ? a.block_table[(size_t)r * a.table_width + col] : popped_page(s_grow[r] + col - before);
            if (page_in_pool(page, a.num_pages)) slot = page * P + (pos - col * P);     // else: not a slot of another page
        }
        a.slots[t] = slot;
    }
}

}  // namespace

cudaError_t launch_paged_plan(PagedPlanArgs a, cudaStream_t s) {
    a.max_len = max_len_of(a.table_width, a.page_rows);
    a.by_page = fast_div(a.page_rows);
    // One CTA where a thread has one token or request at most, else the cluster (us, one / eight CTAs: 8 chats 2.7 / 2.9, 64
    // requests and 960 tokens 5.0 / 4.5, 256 requests and 15000 tokens 8.3 / 6.1, 2000 requests 13.0 / 8.7).  256 threads a CTA for small steps,
    // whose scan and barriers are shorter (8 chats 2.7, with 1024 threads 3.5).
    const bool wide = a.max_tokens + (long long)a.requests > 256;
    const bool narrow = a.max_tokens <= 1024 && a.requests <= 256;
    const size_t smem = (size_t)a.requests * 5 * sizeof(int);
    static std::atomic<unsigned long long> configured{0};   // bit per device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !(configured.load(std::memory_order_acquire) >> dev & 1ull)) {
        e = cudaFuncSetAttribute(paged_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SHAINET_ATTN_PAGED_MAX_REQUESTS * 5 * (int)sizeof(int));
        if (e != cudaSuccess) return e;
        if (dev < 64) configured.fetch_or(1ull << dev, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(wide ? PLAN_CLUSTER : 1);
    cfg.blockDim = dim3(narrow ? 256 : PLAN_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cfg.gridDim.x;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = wide ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, paged_plan_kernel, a);
}

}  // namespace shainet
