// Products of activation rows with 4-bit weights and group scales, sm_100a.
//
//   y[m, n] = sum_k x[m, k] * s[n, k / group] * (nibble[n, k] - 8)
//
// Layout.  Weights are kept in the order in which the matrix units take them: a block of 16 outputs x 64 inputs is 512
// bytes, 16 a lane; word s of a lane holds its four operand registers of inputs 16s .. 16s + 15, nibble i the first and
// nibble i + 4 the second value of register i.  Scales lie as [16 outputs][group][output g and g + 8].  Outputs are padded to
// 16 with scale 0, inputs to 64 with value 0.
//
// Arithmetic.  The weights are exact as bfloat16: a nibble is dropped into the mantissa of 128 and 136 subtracted (4
// instructions for 4 values).  Activations are fp32 and enter as three bfloat16 planes each, x = hi + mid + lo exactly (24
// bits cut into 8 + 8 + 8), so no operand is rounded.  m16n8k16 multiplications with fp32 accumulators; the sums of 32
// inputs start from zero and are added in fp32 with their scale, so sums that the matrix units cut off stay short.
//   * One or two rows: the planes are the columns of one multiplication (2 rows x 3 planes of 8).
//   * More rows: eight rows a multiplication, three of them for the planes, up to 40 rows a pass over the weights.
//
// Work.  A CTA takes NT blocks of outputs at a time and splits their inputs over its eight warps, each with a ring of its own
// in shared memory that asynchronous copies fill RING blocks ahead; the warps' sums meet in shared memory.  With one row
// HBM bounds it (0.5 byte and 4 / group bytes a weight), with many the matrix units.  The first weights are requested
// before the wait for the kernel ahead in the stream: they never depend on it.
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>
#include <new>
#include <vector>

#include "host_state.h"

using namespace shainet;

struct shainet_attn_q4 {
    shainet_attn_ctx* ctx = nullptr;
    int K = 0, N = 0, group = 32;
    uint4* q = nullptr;        // [N / 16][K / 64][32 lanes], rounded up
    float* scales = nullptr;   // [N / 16][groups][8][2], rounded up
};

namespace {

constexpr unsigned FULL = 0xffffffffu;
constexpr int WARPS = 8, THREADS = WARPS * 32;
constexpr int MAX_MT = 5;               // rows of eight in one pass
constexpr int SMEM_MAX = 220 * 1024;

int blocks_of(int n, int d) { return (n + d - 1) / d; }
// groups per 16 outputs as stored: whole blocks of 64 inputs
int stored_groups(int K, int group) { return group == 32 ? 2 * blocks_of(K, 64) : blocks_of(K, group); }

// ---- layout ----
__device__ __forceinline__ int nibble_of(const uint8_t* packed, int K, int N, int n, int k) {
    if (n >= N || k >= K) return 8;
    const uint8_t b = packed[(size_t)n * ((K + 1) / 2) + (k >> 1)];
    return (k & 1) ? b >> 4 : b & 15;
}

__global__ void __launch_bounds__(256) q4_pack_kernel(const uint8_t* packed, uint4* q, int K, int N, int kbs, long long blocks) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    for (long long b = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); b < blocks; b += (long long)gridDim.x * 8) {
        const int nt = (int)(b / kbs), kb = (int)(b - (long long)nt * kbs);
        uint32_t w[4];
        for (int s = 0; s < 4; ++s) {
            w[s] = 0;
            for (int i = 0; i < 4; ++i) {
                const int n = nt * 16 + g + 8 * (i & 1), k = kb * 64 + s * 16 + 2 * t + 8 * (i >> 1);
                w[s] |= (uint32_t)nibble_of(packed, K, N, n, k) << (4 * i) | (uint32_t)nibble_of(packed, K, N, n, k + 1) << (4 * i + 16);
            }
        }
        q[b * 32 + lane] = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

__global__ void __launch_bounds__(256) q4_unpack_kernel(const uint4* q, uint8_t* packed, int K, int N, int kbs) {
    const long long bytes = (K + 1) / 2, total = (long long)N * bytes;
    for (long long x = (long long)blockIdx.x * 256 + threadIdx.x; x < total; x += (long long)gridDim.x * 256) {
        const int n = (int)(x / bytes), j = (int)(x - n * bytes);
        int v = 0;
        for (int h = 0; h < 2; ++h) {
            const int k = 2 * j + h, g = n & 7, kk = k & 15, t = (kk & 7) >> 1, i = ((n >> 3) & 1) + 2 * (kk >> 3);
            const uint32_t* w = reinterpret_cast<const uint32_t*>(q + ((size_t)(n >> 4) * kbs + (k >> 6)) * 32 + g * 4 + t);
            v |= (k < K ? (w[(k & 63) >> 4] >> (4 * i + 16 * (k & 1))) & 15 : 8) << (4 * h);
        }
        packed[x] = (uint8_t)v;
    }
}

// scales [N, ceil(K / group)] <-> [N / 16][stored groups][8][2]
__global__ void __launch_bounds__(256) q4_scales_kernel(const float* from, float* to, int N, int groups, int stored, long long total, bool pack) {
    for (long long x = (long long)blockIdx.x * 256 + threadIdx.x; x < total; x += (long long)gridDim.x * 256) {
        const int r = (int)(x & 15), n = (int)(x / 16 / stored) * 16 + (r >> 1) + 8 * (r & 1), g = (int)(x / 16 % stored);
        const bool in = n < N && g < groups;
        const size_t at = (size_t)n * groups + g;
        if (pack) to[x] = in ? from[at] : 0.0f;
        else if (in) to[at] = from[x];
    }
}

// ---- product ----
__device__ __forceinline__ uint32_t smem_at(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// d += a b, or d = a b with FIRST
template <bool FIRST>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(FIRST ? 0.f : d[0]), "f"(FIRST ? 0.f : d[1]),
                   "f"(FIRST ? 0.f : d[2]), "f"(FIRST ? 0.f : d[3]));
}

// One word -> the four operand registers of 16 inputs: pairs of (nibble - 8) as bfloat16, exact.
__device__ __forceinline__ void unpack(uint32_t w, uint32_t (&a)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t v;
        asm("lop3.b32 %0, %1, 0x000f000f, 0x43004300, 0xea;" : "=r"(v) : "r"(w >> (4 * i)));      // (w & mask) | 128.0
        asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(a[i]) : "r"(v), "r"(0x3f803f80u), "r"(0xc308c308u));   // * 1 - 136
    }
}

// Two fp32 values as three packed bfloat16 pairs, exactly: the upper halves, then the upper halves of what is left.
__device__ __forceinline__ void planes(float x0, float x1, uint32_t (&p)[3]) {
    const uint32_t u0 = __float_as_uint(x0), u1 = __float_as_uint(x1);
    p[0] = __byte_perm(u0, u1, 0x7632);
    const float r0 = x0 - __uint_as_float(u0 & 0xffff0000u), r1 = x1 - __uint_as_float(u1 & 0xffff0000u);
    const uint32_t v0 = __float_as_uint(r0), v1 = __float_as_uint(r1);
    p[1] = __byte_perm(v0, v1, 0x7632);
    const float s0 = r0 - __uint_as_float(v0 & 0xffff0000u), s1 = r1 - __uint_as_float(v1 & 0xffff0000u);
    p[2] = __byte_perm(__float_as_uint(s0), __float_as_uint(s1), 0x7632);
}

// MT = 0: one or two rows, their planes kept in shared memory; else 8 * MT rows at most.
template <int MT_, int NT_>
struct Cfg {
    static constexpr int MT = MT_, NT = NT_;
    static constexpr int COLS = MT == 0 ? 8 : 8 * MT;                 // columns of the sums: planes and rows, or rows
    static constexpr int UNIT = NT * 640;                             // a ring place: NT blocks, 128 bytes for the scales of each
    static constexpr int RING = MT == 0 ? 8 : NT == 1 ? 6 : 4;        // places of a warp's ring
    static constexpr int RED = COLS + 2;                              // floats between outputs in the sums' meeting place
    static constexpr int SUMS = (MT == 0 ? 2 : 1) * WARPS * NT * 16 * RED * 4;
    static constexpr size_t FIXED = (size_t)WARPS * RING * UNIT + SUMS;
};

// Inputs that a warp owns: blocks [first, first + count) of 64.
__host__ __device__ __forceinline__ int slice_of(int kbs) { return (kbs + WARPS - 1) / WARPS; }

template <class C>
__global__ void __launch_bounds__(THREADS, C::MT == 0 ? 2 : 1) q4_gemv_kernel(Q4GemvArgs a, int kbs, int stored, int blocks) {
    constexpr int MT = C::MT, NT = C::NT;
    extern __shared__ __align__(16) unsigned char q4_smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    unsigned char* ring = q4_smem + (size_t)warp * C::RING * C::UNIT;
    float* red = reinterpret_cast<float*>(q4_smem + (size_t)WARPS * C::RING * C::UNIT);
    uint4* xs = reinterpret_cast<uint4*>(q4_smem + C::FIXED);          // MT = 0: [pairs of 16 inputs][32 lanes]
    const int slice = slice_of(kbs), kb0 = min(warp * slice, kbs), kb1 = min(kb0 + slice, kbs), mine = kb1 - kb0;
    const int sets = (blocks + NT - 1) / NT;                           // of NT blocks of 16 outputs
    const int m0 = blockIdx.y * a.pass_rows, rows = min(a.pass_rows, a.M - m0);
    const float* x = a.x + (size_t)m0 * a.K;
    const int per_kb = a.group == 32 ? 2 : 1, kb_shift = a.group == 128 ? 1 : 0;

    // ---- copies: for every set of this CTA the blocks of the warp's slice ----
    int ld_set = blockIdx.x, ld_kb = kb0;
    uint32_t fill = 0;
    const uint32_t ring_at = smem_at(ring);
    auto fetch = [&]() {
        if (mine > 0 && ld_set < sets) {
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const int nt = min(ld_set * NT + i, blocks - 1);       // behind the last block: read again, not used
                copy16(ring_at + fill + i * 640 + lane * 16, a.q + ((size_t)nt * kbs + ld_kb) * 32 + lane);
                if (lane < 4 * per_kb)
                    copy16(ring_at + fill + i * 640 + 512 + lane * 16, a.scales + ((size_t)nt * stored + (ld_kb * per_kb >> kb_shift)) * 16 + lane * 4);
            }
            fill = fill == (C::RING - 1) * C::UNIT ? 0 : fill + C::UNIT;
            if (++ld_kb == kb1) ld_kb = kb0, ld_set += gridDim.x;
        }
        copy_commit();
    };
#pragma unroll 1
    for (int i = 0; i < C::RING - 1; ++i) fetch();
    asm volatile("griddepcontrol.wait;" ::: "memory");                 // x may come from the kernel ahead, y may be read by it
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    // x of one row and input; zero behind the last input
    auto x_at = [&](const float* row, int k) { return k < a.K ? __ldcg(row + k) : 0.0f; };
    if constexpr (MT == 0) {
        // column g: plane g / 2 of row g % 2
        const int plane = g >> 1;
        const bool on = plane < 3 && (g & 1) < rows;
        const float* row = x + (size_t)((g & 1) < rows ? g & 1 : 0) * a.K;
#pragma unroll 2
        for (int p = kb0 * 2; p < kb1 * 2; ++p) {
            uint32_t b[4];
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                const int k = p * 32 + (h >> 1) * 16 + (h & 1) * 8 + 2 * t;
                uint32_t v[3];
                planes(x_at(row, k), x_at(row, k + 1), v);
                b[h] = !on ? 0u : plane == 0 ? v[0] : plane == 1 ? v[1] : v[2];
            }
            xs[(size_t)p * 32 + lane] = make_uint4(b[0], b[1], b[2], b[3]);
        }
        __syncwarp();
    }
    const float* xrow[MT == 0 ? 1 : MT];
    if constexpr (MT > 0)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) xrow[mt] = x + (size_t)min(mt * 8 + g, rows - 1) * a.K;      // rows behind the last: not stored
    const bool even = (a.K & 1) == 0;

    uint32_t take = 0;
    int turn = 0;
#pragma unroll 1
    for (int set = blockIdx.x; set < sets; set += gridDim.x, ++turn) {
        float total[NT][MT == 0 ? 1 : MT][4];
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int mt = 0; mt < (MT == 0 ? 1 : MT); ++mt)
#pragma unroll
                for (int c = 0; c < 4; ++c) total[i][mt][c] = 0.0f;
#pragma unroll 1
        for (int kb = kb0; kb < kb1; ++kb) {
            copy_wait<C::RING - 2>();
            __syncwarp();
            const unsigned char* unit = ring + take;
#pragma unroll
            for (int h = 0; h < 2; ++h) {                              // 32 inputs
                uint32_t w[NT][2];
                float2 sc[NT];
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    const uint2 v = *reinterpret_cast<const uint2*>(unit + i * 640 + lane * 16 + h * 8);
                    w[i][0] = v.x, w[i][1] = v.y;
                    sc[i] = *reinterpret_cast<const float2*>(unit + i * 640 + 512 + (per_kb == 2 ? h * 64 : 0) + g * 8);
                }
                uint32_t op[NT][2][4];
#pragma unroll
                for (int i = 0; i < NT; ++i) unpack(w[i][0], op[i][0]), unpack(w[i][1], op[i][1]);
                if constexpr (MT == 0) {
                    const uint4 b = xs[(size_t)(kb * 2 + h) * 32 + lane];
#pragma unroll
                    for (int i = 0; i < NT; ++i) {
                        float c[4];
                        mma<true>(c, op[i][0], b.x, b.y);
                        mma<false>(c, op[i][1], b.z, b.w);
                        total[i][0][0] = fmaf(sc[i].x, c[0], total[i][0][0]);
                        total[i][0][1] = fmaf(sc[i].x, c[1], total[i][0][1]);
                        total[i][0][2] = fmaf(sc[i].y, c[2], total[i][0][2]);
                        total[i][0][3] = fmaf(sc[i].y, c[3], total[i][0][3]);
                    }
                } else {
                    const int k0 = kb * 64 + h * 32 + 2 * t;
                    const bool whole = even && kb * 64 + 64 <= a.K;
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        float2 v[4];
                        if (whole) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) v[i] = __ldcg(reinterpret_cast<const float2*>(xrow[mt] + k0 + i * 8));
                        } else {
#pragma unroll
                            for (int i = 0; i < 4; ++i) v[i] = make_float2(x_at(xrow[mt], k0 + i * 8), x_at(xrow[mt], k0 + i * 8 + 1));
                        }
                        uint32_t b[4][3];
#pragma unroll
                        for (int i = 0; i < 4; ++i) planes(v[i].x, v[i].y, b[i]);
#pragma unroll
                        for (int i = 0; i < NT; ++i) {
                            float c[4];
                            mma<true>(c, op[i][0], b[0][2], b[1][2]);
                            mma<false>(c, op[i][1], b[2][2], b[3][2]);
                            mma<false>(c, op[i][0], b[0][1], b[1][1]);
                            mma<false>(c, op[i][1], b[2][1], b[3][1]);
                            mma<false>(c, op[i][0], b[0][0], b[1][0]);
                            mma<false>(c, op[i][1], b[2][0], b[3][0]);
                            total[i][mt][0] = fmaf(sc[i].x, c[0], total[i][mt][0]);
                            total[i][mt][1] = fmaf(sc[i].x, c[1], total[i][mt][1]);
                            total[i][mt][2] = fmaf(sc[i].y, c[2], total[i][mt][2]);
                            total[i][mt][3] = fmaf(sc[i].y, c[3], total[i][mt][3]);
                        }
                    }
                }
            }
            __syncwarp();
            take = take == (C::RING - 1) * C::UNIT ? 0 : take + C::UNIT;
            fetch();
        }
        // ---- the warps' sums ----
        float* meet = red + (MT == 0 ? (turn & 1) * (WARPS * 16 * C::RED) : 0);
        float* to = meet + warp * NT * 16 * C::RED;
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int mt = 0; mt < (MT == 0 ? 1 : MT); ++mt)
#pragma unroll
                for (int r = 0; r < 2; ++r)
                    *reinterpret_cast<float2*>(to + (i * 16 + g + 8 * r) * C::RED + mt * 8 + 2 * t) = make_float2(total[i][mt][2 * r], total[i][mt][2 * r + 1]);
        __syncthreads();
        if constexpr (MT == 0) {
            // one warp adds, another one every time; the next sums go to the other half
            if (warp == (turn & (WARPS - 1))) {
                const int n = lane & 15, m = lane >> 4, out = set * 16 + n;
                if (m < rows && out < a.N) {
                    float sum = 0.0f;
#pragma unroll
                    for (int w = 0; w < WARPS; ++w) {
                        const float* s = meet + (w * 16 + n) * C::RED + m;
                        sum += s[4] + s[2] + s[0];
                    }
                    a.y[(size_t)(m0 + m) * a.N + out] = sum;
                }
            }
        } else {
#pragma unroll 1
            for (int e = tid; e < NT * 16 * rows; e += THREADS) {
                const int m = e / (NT * 16), n = e - m * (NT * 16), out = set * NT * 16 + n;
                float sum = 0.0f;
#pragma unroll
                for (int w = 0; w < WARPS; ++w) sum += meet[(w * NT * 16 + n) * C::RED + m];
                if (out < a.N) a.y[(size_t)(m0 + m) * a.N + out] = sum;
            }
            __syncthreads();
        }
    }
    copy_wait<0>();
}

template <int MT, int NT>
cudaError_t launch(const Q4GemvArgs& a, int sm_count, cudaStream_t s) {
    using C = Cfg<MT, NT>;
    const int kbs = blocks_of(a.K, 64), blocks = blocks_of(a.N, 16), sets = blocks_of(blocks, NT);
    const size_t smem = C::FIXED + (MT == 0 ? (size_t)kbs * 1024 : 0);
    static std::atomic<unsigned long long> configured{0};   // bit per device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !(configured.load(std::memory_order_acquire) >> dev & 1ull)) {
        e = cudaFuncSetAttribute(q4_gemv_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_MAX);
        if (e != cudaSuccess) return e;
        if (dev < 64) configured.fetch_or(1ull << dev, std::memory_order_release);
    }
    const int passes = blocks_of(a.M, a.pass_rows);
    const int per_sm = MT == 0 && smem <= 112 * 1024 ? 2 : 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(std::min(sets, std::max(1, sm_count * per_sm / std::min(passes, per_sm))), passes);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, q4_gemv_kernel<C>, a, kbs, stored_groups(a.K, a.group), blocks);
}

template <int MT>
cudaError_t launch_rows(const Q4GemvArgs& a, int sm_count, cudaStream_t s) {
    // four blocks of outputs share the planes of x where that still leaves a CTA for most SMs
    return blocks_of(a.N, 16) >= 4 * (sm_count * 3 / 4) ? launch<MT, 4>(a, sm_count, s) : launch<MT, 1>(a, sm_count, s);
}

}  // namespace

namespace shainet {

cudaError_t launch_q4_gemv(Q4GemvArgs a, int sm_count, cudaStream_t s) {
    a.pass_rows = a.M;
    if (a.M <= 2 && Cfg<0, 1>::FIXED + (size_t)blocks_of(a.K, 64) * 1024 <= SMEM_MAX) return launch<0, 1>(a, sm_count, s);
    const int passes = blocks_of(a.M, 8 * MAX_MT);
    a.pass_rows = blocks_of(a.M, passes);
    switch (blocks_of(a.pass_rows, 8)) {
        case 1: return launch_rows<1>(a, sm_count, s);
        case 2: return launch_rows<2>(a, sm_count, s);
        case 3: return launch_rows<3>(a, sm_count, s);
        case 4: return launch_rows<4>(a, sm_count, s);
        default: return launch_rows<5>(a, sm_count, s);
    }
}

}  // namespace shainet

namespace {

size_t packed_bytes(int K, int N) { return (size_t)N * ((K + 1) / 2); }
size_t scale_count(int K, int N, int group) { return (size_t)N * blocks_of(K, group); }
int grid_of(long long items) { return (int)std::min<long long>((items + 255) / 256, 16384); }

// As the Q8_0 quantiser: per output and group scale = max|w| / 7 (1 for an all-zero group), round to nearest even.
void quantize_q4(const float* w, int K, int N, int group, uint8_t* packed, float* scales) {
    const int groups = blocks_of(K, group), bytes = (K + 1) / 2;
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
    if (K > (1 << 24) || N > (1 << 28)) return fail(SHAINET_ATTN_E_UNSUPPORTED, "weight shape %d x %d: at most 2^24 x 2^28", K, N);
    if (group != 32 && group != 64 && group != 128) return fail(SHAINET_ATTN_E_UNSUPPORTED, "group %d: 32, 64 or 128", group);
    return SHAINET_ATTN_OK;
}

int create_from(shainet_attn_ctx* ctx, shainet_attn_q4** out, const uint8_t* packed, const float* scales, int K, int N, int group, bool host) {
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
    const int kbs = blocks_of(K, 64), nts = blocks_of(N, 16), stored = stored_groups(K, group);
    const long long blocks = (long long)kbs * nts, slots = (long long)nts * stored * 16;
    const size_t qb = packed_bytes(K, N), sb = scale_count(K, N, group) * sizeof(float);
    uint8_t* dq = nullptr;
    float* ds = nullptr;
    cudaStream_t s = ctx->stream;
    cudaError_t e = cudaMalloc(&w->q, (size_t)blocks * 512);
    if (e == cudaSuccess) e = cudaMalloc(&w->scales, (size_t)slots * sizeof(float));
    if (e == cudaSuccess && host) {
        e = cudaMalloc(&dq, qb);
        if (e == cudaSuccess) e = cudaMalloc(&ds, sb);
        if (e == cudaSuccess) e = cudaMemcpyAsync(dq, packed, qb, cudaMemcpyHostToDevice, s);
        if (e == cudaSuccess) e = cudaMemcpyAsync(ds, scales, sb, cudaMemcpyHostToDevice, s);
    }
    if (e == cudaSuccess) {
        q4_pack_kernel<<<grid_of(blocks * 32), 256, 0, s>>>(host ? dq : packed, w->q, K, N, kbs, blocks);
        q4_scales_kernel<<<grid_of(slots), 256, 0, s>>>(host ? ds : scales, w->scales, N, blocks_of(K, group), stored, slots, true);
        e = cudaGetLastError();
    }
    const cudaError_t done = cudaStreamSynchronize(s);
    if (e == cudaSuccess) e = done;
    if (dq) cudaFree(dq);
    if (ds) cudaFree(ds);
    if (e != cudaSuccess) {
        shainet_attn_q4_destroy(w);
        return fail_cuda(e, "layout of a 4-bit weight");
    }
    *out = w;
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
    std::vector<uint8_t> q;
    std::vector<float> sc;
    try {
        q.resize(packed_bytes(K, N));
        sc.resize(scale_count(K, N, group));
    } catch (const std::bad_alloc&) {
        return fail(SHAINET_ATTN_E_NOMEM, "out of host memory");
    }
    quantize_q4(w, K, N, group, q.data(), sc.data());
    return create_from(ctx, out, q.data(), sc.data(), K, N, group, true);
}

int shainet_attn_q4_create_raw(shainet_attn_ctx* ctx, shainet_attn_q4** out, const uint8_t* packed, const float* scales, int K, int N, int group) {
    return create_from(ctx, out, packed, scales, K, N, group, true);
}

int shainet_attn_q4_create_dev(shainet_attn_ctx* ctx, shainet_attn_q4** out, const uint8_t* packed, const float* scales, int K, int N, int group) {
    return create_from(ctx, out, packed, scales, K, N, group, false);
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
    const int groups = blocks_of(w->K, w->group), stored = stored_groups(w->K, w->group);
    const size_t qb = packed_bytes(w->K, w->N), sb = scale_count(w->K, w->N, w->group) * sizeof(float);
    const long long slots = (long long)blocks_of(w->N, 16) * stored * 16;
    uint8_t* dq = nullptr;
    float* ds = nullptr;
    cudaStream_t s = w->ctx->stream;
    cudaError_t e = cudaMalloc(&dq, qb);
    if (e == cudaSuccess) e = cudaMalloc(&ds, sb);
    if (e == cudaSuccess) {
        q4_unpack_kernel<<<grid_of((long long)qb), 256, 0, s>>>(w->q, dq, w->K, w->N, blocks_of(w->K, 64));
        q4_scales_kernel<<<grid_of(slots), 256, 0, s>>>(w->scales, ds, w->N, groups, stored, slots, false);
        e = cudaGetLastError();
    }
    if (e == cudaSuccess) e = cudaMemcpyAsync(packed, dq, qb, cudaMemcpyDeviceToHost, s);
    if (e == cudaSuccess) e = cudaMemcpyAsync(scales, ds, sb, cudaMemcpyDeviceToHost, s);
    const cudaError_t done = cudaStreamSynchronize(s);
    if (e == cudaSuccess) e = done;
    if (dq) cudaFree(dq);
    if (ds) cudaFree(ds);
    return e == cudaSuccess ? SHAINET_ATTN_OK : fail_cuda(e, "export of a 4-bit weight");
}

int shainet_attn_q4_gemv_dev(shainet_attn_ctx* ctx, const shainet_attn_q4* w, const float* x, float* y, int rows, void* stream) {
    if (rows < 0) return fail(SHAINET_ATTN_E_INVALID, "rows %d < 0", rows);
    if (!ctx || !w) return fail(SHAINET_ATTN_E_INVALID, "null context or weight");
    if (w->ctx != ctx) return fail(SHAINET_ATTN_E_INVALID, "weight belongs to another context");
    if (rows == 0) return SHAINET_ATTN_OK;
    if (!x || !y) return fail(SHAINET_ATTN_E_INVALID, "null pointer");
    if (!aligned16(x) || !aligned16(y)) return fail(SHAINET_ATTN_E_INVALID, "device pointers must be 16-byte aligned");
    if (rows > 1 << 20) return fail(SHAINET_ATTN_E_UNSUPPORTED, "%d rows: a call takes at most 2^20", rows);
    DeviceGuard g(ctx->device);
    Q4GemvArgs a{};
    a.x = x;
    a.q = w->q;
    a.scales = w->scales;
    a.y = y;
    a.M = rows;
    a.N = w->N;
    a.K = w->K;
    a.group = w->group;
    ctx->last_fused = false;
    CU(launch_q4_gemv(a, ctx->sm_count, stream ? (cudaStream_t)stream : ctx->stream));
    return SHAINET_ATTN_OK;
}

}  // extern "C"
