// Attention of one new token per request over keys and values in pages, sm_100a.
//
// o = sum_j softmax_j(scale q . k_j) v_j over the positions j < len, q and the new k row with bias, per-head RMSNorm and
// RoPE at position len - 1, the new rows written into their page.  One CTA per (query head, request).
#include <cuda_bf16.h>
#include <math.h>
#include "kernels.h"
#include "paged_index.h"

namespace shainet {

namespace {

constexpr unsigned FULL = 0xffffffffu;
constexpr float LOG2E = 1.4426950408889634f;
constexpr int THREADS = 128;

template <int ES>
__device__ __forceinline__ float load_el(const void* p, size_t i) {
    if constexpr (ES == 4) return static_cast<const float*>(p)[i];
    else return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

template <int HD, int ES>
__global__ void __launch_bounds__(THREADS) paged_decode_simple_kernel(PagedDecodeArgs a) {
    constexpr int PL = HD / 64, CL = HD / 32;
    const int h = blockIdx.x, r = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int H = a.hs.num_heads, KV = a.hs.num_kv_heads, G = H / KV, kv_h = h / G;
    const int P = a.page_rows;
    __shared__ float sx[3][HD];
    __shared__ float so[4][HD], sm[4], sl[4];
    int len = a.lens[r];
    float* out = a.out + ((size_t)r * H + h) * HD;
    if (!length_fits(len, a.table_width, P)) {
        if (threadIdx.x == 0) report_status(a.status, DEV_BAD_PAGE, 13);
        len = 0;
    }
    if (len == 0) {
        for (int d = threadIdx.x; d < HD; d += THREADS) out[d] = 0.0f;
        return;
    }
    const int* table = a.block_table + (size_t)r * a.table_width;
    const int pos = len - 1;
    if (warp < 3) {   // q, k, v of this head
        const float* src = warp == 0 ? a.q + ((size_t)r * H + h) * HD : (warp == 1 ? a.k_new : a.v_new) + ((size_t)r * KV + kv_h) * HD;
        const float* bias = warp == 0 ? a.b_q : warp == 1 ? a.b_k : a.b_v;
        if (bias) bias += (size_t)(warp == 0 ? h : kv_h) * HD;
        const float* w = warp == 0 ? a.q_norm : warp == 1 ? a.k_norm : nullptr;
        float x[CL];
        float ss = 0.0f;
        for (int c = 0; c < CL; ++c) {
            x[c] = src[lane + 32 * c];
            if (bias) x[c] = __fadd_rn(x[c], bias[lane + 32 * c]);
            ss = fmaf(x[c], x[c], ss);
        }
        for (int off = 16; off > 0; off >>= 1) ss += __shfl_xor_sync(FULL, ss, off);
        if (w) {
            const float inv = (float)(1.0 / sqrt((double)(ss / (float)HD) + a.eps));
            for (int c = 0; c < CL; ++c) x[c] = __fmul_rn(__fmul_rn(x[c], inv), w[lane + 32 * c]);
        }
        if (warp < 2) {
            for (int k = 0; k < PL; ++k) {
                float sn, cs;
                sincosf(__fmul_rn((float)pos, a.inv_freq[lane + 32 * k]), &sn, &cs);
                const float x0 = x[k], x1 = x[k + PL];
                x[k] = __fsub_rn(__fmul_rn(x0, cs), __fmul_rn(x1, sn));
                x[k + PL] = __fadd_rn(__fmul_rn(x1, cs), __fmul_rn(x0, sn));
            }
        }
        const int page = table[pos / P];
        const bool store = warp > 0 && h % G == 0 && page_in_pool(page, a.num_pages);
        const size_t at = pool_row(store ? page : 0, KV, kv_h, P, pos % P) * HD;
        for (int c = 0; c < CL; ++c) {
            if (warp > 0 && ES == 2) x[c] = __bfloat162float(__float2bfloat16_rn(x[c]));
            sx[warp][lane + 32 * c] = x[c];
            if (store) {
                void* dst = warp == 1 ? a.k_pages : a.v_pages;
                if (ES == 4) static_cast<float*>(dst)[at + lane + 32 * c] = x[c];
                else static_cast<__nv_bfloat16*>(dst)[at + lane + 32 * c] = __float2bfloat16_rn(x[c]);
            }
        }
    }
    __syncthreads();
    float q[CL], o[CL], m = -INFINITY, l = 0.0f;
    for (int c = 0; c < CL; ++c) {
        q[c] = sx[0][lane + 32 * c];
        o[c] = 0.0f;
    }
    for (int j = warp; j < len; j += 4) {
        const int page = table[j / P];
        const bool there = page_in_pool(page, a.num_pages);
        if (!there && lane == 0) report_status(a.status, DEV_BAD_PAGE, 14);
        const size_t at = pool_row(there ? page : 0, KV, kv_h, P, j % P) * HD;
        float s = 0.0f, v[CL];
        for (int c = 0; c < CL; ++c) {
            float k = 0.0f;
            v[c] = 0.0f;
            if (j == pos) {
                k = sx[1][lane + 32 * c];
                v[c] = sx[2][lane + 32 * c];
            } else if (there) {
                k = load_el<ES>(a.k_pages, at + lane + 32 * c);
                v[c] = load_el<ES>(a.v_pages, at + lane + 32 * c);
            }
            s = fmaf(q[c], k, s);
        }
        for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(FULL, s, off);
        s *= a.scale;
        const float mn = fmaxf(m, s), al = exp2f((m - mn) * LOG2E), p = exp2f((s - mn) * LOG2E);
        m = mn;
        l = fmaf(l, al, p);
        for (int c = 0; c < CL; ++c) o[c] = fmaf(p, v[c], o[c] * al);
    }
    for (int c = 0; c < CL; ++c) so[warp][lane + 32 * c] = o[c];
    if (lane == 0) sm[warp] = m, sl[warp] = l;
    __syncthreads();
    for (int d = threadIdx.x; d < HD; d += THREADS) {
        float M = -INFINITY, L = 0.0f, acc = 0.0f;
        for (int w = 0; w < 4; ++w) M = fmaxf(M, sm[w]);
        for (int w = 0; w < 4; ++w) {
            const float wt = sm[w] == -INFINITY ? 0.0f : exp2f((sm[w] - M) * LOG2E);
            L = fmaf(wt, sl[w], L);
            acc = fmaf(wt, so[w][d], acc);
        }
        out[d] = acc / L;
    }
}

}  // namespace

cudaError_t launch_paged_decode(const PagedDecodeArgs& a, cudaStream_t s) {
    const dim3 grid(a.hs.num_heads, a.requests);
    if (a.hs.head_dim == 128) {
        if (a.kv_elem_bytes == 4) paged_decode_simple_kernel<128, 4><<<grid, THREADS, 0, s>>>(a);
        else paged_decode_simple_kernel<128, 2><<<grid, THREADS, 0, s>>>(a);
    } else {
        if (a.kv_elem_bytes == 4) paged_decode_simple_kernel<64, 4><<<grid, THREADS, 0, s>>>(a);
        else paged_decode_simple_kernel<64, 2><<<grid, THREADS, 0, s>>>(a);
    }
    return cudaGetLastError();
}

}  // namespace shainet
