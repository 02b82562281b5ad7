// 4-bit weights with group scales: host side of shainet_attn_q4_* and the product kernel, sm_100a.
//
// y[m, n] = sum_k x[m, k] * s[n, k / group] * (nibble[n, k] - 8).  One warp per output and row.
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <new>
#include <vector>

#include "host_state.h"

using namespace shainet;

struct shainet_attn_q4 {
    shainet_attn_ctx* ctx = nullptr;
    int K = 0, N = 0, group = 32;
    uint8_t* q = nullptr;
    float* scales = nullptr;
};

namespace {

__global__ void __launch_bounds__(256) q4_gemv_simple_kernel(const float* x, const uint8_t* q, const float* scales, float* y, int N, int K, int group) {
    const int n = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (n >= N) return;
    for (int m = blockIdx.y; m < (int)gridDim.z * 65535; m += 65535) {
        float acc = 0.0f;
        for (int k = lane; k < K; k += 32) {
            const int b = q[(size_t)n * ((K + 1) / 2) + k / 2];
            const float w = (float)((k & 1 ? b >> 4 : b & 15) - 8);
            acc = fmaf(w * scales[(size_t)n * ((K + group - 1) / group) + k / group], x[(size_t)m * K + k], acc);
        }
        for (int off = 16; off > 0; off >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, off);
        if (lane == 0) y[(size_t)m * N + n] = acc;
        break;
    }
}

size_t packed_bytes(int K, int N) { return (size_t)N * ((K + 1) / 2); }
size_t scale_count(int K, int N, int group) { return (size_t)N * ((K + group - 1) / group); }

// As the Q8_0 quantiser: per output and group scale = max|w| / 7 (1 for an all-zero group), round to nearest even.
void quantize_q4(const float* w, int K, int N, int group, uint8_t* packed, float* scales) {
    const int groups = (K + group - 1) / group, bytes = (K + 1) / 2;
    for (int n = 0; n < N; ++n) {
        uint8_t* row = packed + (size_t)n * bytes;
        std::fill(row, row + bytes, (uint8_t)0x88);
        for (int g = 0; g < groups; ++g) {
            const int base = g * group, lim = std::min(base + group, K);
            float max_abs = 0.0f;
            for (int k = base; k < lim; ++k) max_abs = std::max(max_abs, fabsf(w[(size_t)k * N + n]));
            const float scale = max_abs > 0.0f ? max_abs / 7.0f : 1.0f, inv = 1.0f / scale;
            scales[(size_t)n * groups + g] = scale;
            for (int k = base; k < lim; ++k) {
                const float v = std::min(7.0f, std::max(-7.0f, nearbyintf(w[(size_t)k * N + n] * inv)));
                const uint8_t u = (uint8_t)((int)v + 8);
                row[k / 2] = (uint8_t)((k & 1) ? (row[k / 2] & 0x0f) | (u << 4) : (row[k / 2] & 0xf0) | u);
            }
        }
    }
}

int check_shape(int K, int N, int group) {
    if (K <= 0 || N <= 0) return fail(SHAINET_ATTN_E_INVALID, "weight shape %d x %d", K, N);
    if (group != 32 && group != 64 && group != 128) return fail(SHAINET_ATTN_E_UNSUPPORTED, "group %d: 32, 64 or 128", group);
    return SHAINET_ATTN_OK;
}

}  // namespace

extern "C" {

int shainet_attn_q4_create(shainet_attn_ctx* ctx, shainet_attn_q4** out, const float* w, int K, int N, int group) {
    if (!out || !w) return fail(SHAINET_ATTN_E_INVALID, "null pointer");
    *out = nullptr;
    int rc = check_shape(K, N, group);
    if (rc) return rc;
    if (!ctx) return fail(SHAINET_ATTN_E_INVALID, "null context");
    std::vector<uint8_t> q(packed_bytes(K, N));
    std::vector<float> sc(scale_count(K, N, group));
    quantize_q4(w, K, N, group, q.data(), sc.data());
    return shainet_attn_q4_create_raw(ctx, out, q.data(), sc.data(), K, N, group);
}

static int create_from(shainet_attn_ctx* ctx, shainet_attn_q4** out, const uint8_t* packed, const float* scales, int K, int N, int group, cudaMemcpyKind kind) {
    if (!out || !packed || !scales) return fail(SHAINET_ATTN_E_INVALID, "null pointer");
    *out = nullptr;
    int rc = check_shape(K, N, group);
    if (rc) return rc;
    if (!ctx) return fail(SHAINET_ATTN_E_INVALID, "null context");
    DeviceGuard g(ctx->device);
    shainet_attn_q4* w = new (std::nothrow) shainet_attn_q4();
    if (!w) return fail(SHAINET_ATTN_E_NOMEM, "out of host memory");
    w->ctx = ctx;
    w->K = K;
    w->N = N;
    w->group = group;
    const size_t qb = packed_bytes(K, N), sb = scale_count(K, N, group) * sizeof(float);
    cudaError_t e = cudaMalloc(&w->q, qb);
    if (e == cudaSuccess) e = cudaMalloc(&w->scales, sb);
    if (e == cudaSuccess) e = cudaMemcpyAsync(w->q, packed, qb, kind, ctx->stream);
    if (e == cudaSuccess) e = cudaMemcpyAsync(w->scales, scales, sb, kind, ctx->stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize(ctx->stream);
    if (e != cudaSuccess) {
        shainet_attn_q4_destroy(w);
        return fail_cuda(e, "upload of a 4-bit weight");
    }
    *out = w;
    return SHAINET_ATTN_OK;
}

int shainet_attn_q4_create_raw(shainet_attn_ctx* ctx, shainet_attn_q4** out, const uint8_t* packed, const float* scales, int K, int N, int group) {
    return create_from(ctx, out, packed, scales, K, N, group, cudaMemcpyHostToDevice);
}

int shainet_attn_q4_create_dev(shainet_attn_ctx* ctx, shainet_attn_q4** out, const uint8_t* packed, const float* scales, int K, int N, int group) {
    return create_from(ctx, out, packed, scales, K, N, group, cudaMemcpyDeviceToDevice);
}

int shainet_attn_q4_destroy(shainet_attn_q4* w) {
    if (!w) return SHAINET_ATTN_OK;
    DeviceGuard g(w->ctx->device);
    cudaStreamSynchronize(w->ctx->stream);
    if (w->q) cudaFree(w->q);
    if (w->scales) cudaFree(w->scales);
    cudaGetLastError();
    delete w;
    return SHAINET_ATTN_OK;
}

int shainet_attn_q4_export(shainet_attn_q4* w, uint8_t* packed, float* scales) {
    if (!w || !packed || !scales) return fail(SHAINET_ATTN_E_INVALID, "null pointer");
    DeviceGuard g(w->ctx->device);
    CU(cudaMemcpy(packed, w->q, packed_bytes(w->K, w->N), cudaMemcpyDeviceToHost));
    CU(cudaMemcpy(scales, w->scales, scale_count(w->K, w->N, w->group) * sizeof(float), cudaMemcpyDeviceToHost));
    if (w->K & 1)
        for (int n = 0; n < w->N; ++n) {
            uint8_t& b = packed[(size_t)(n + 1) * ((w->K + 1) / 2) - 1];
            b = (uint8_t)((b & 0x0f) | 0x80);
        }
    return SHAINET_ATTN_OK;
}

int shainet_attn_q4_gemv_dev(shainet_attn_ctx* ctx, const shainet_attn_q4* w, const float* x, float* y, int rows, void* stream) {
    if (rows < 0) return fail(SHAINET_ATTN_E_INVALID, "rows %d < 0", rows);
    if (!ctx || !w) return fail(SHAINET_ATTN_E_INVALID, "null context or weight");
    if (w->ctx != ctx) return fail(SHAINET_ATTN_E_INVALID, "weight belongs to another context");
    if (rows == 0) return SHAINET_ATTN_OK;
    if (!x || !y) return fail(SHAINET_ATTN_E_INVALID, "null pointer");
    if (!aligned16(x) || !aligned16(y)) return fail(SHAINET_ATTN_E_INVALID, "device pointers must be 16-byte aligned");
    if (rows > 65535) return fail(SHAINET_ATTN_E_UNSUPPORTED, "%d rows", rows);
    DeviceGuard g(ctx->device);
    ctx->last_fused = false;
    q4_gemv_simple_kernel<<<dim3((w->N + 7) / 8, rows, 1), 256, 0, stream ? (cudaStream_t)stream : ctx->stream>>>(x, w->q, w->scales, y, w->N, w->K, w->group);
    CU(cudaGetLastError());
    return SHAINET_ATTN_OK;
}

}  // extern "C"
