// Products of activation rows with 4-bit weights and group scales, sm_100a.
//
//   y[m, n] = sum_k x[m, k] * s[n, k / group] * (nibble[n, k] - 8)
//
// Layout.  Weights are kept in the order in which the matrix units take them: a block of 16 outputs x 64 inputs is 512
// bytes, 16 a lane; word s of lane (g, t) holds its four operand registers of multiplication s, nibble i the first and nibble
// i + 4 the second value of register i: outputs g and g + 8, inputs 32 (s / 2) + 8t + 4 (s % 2) .. + 3.  (The order of the inputs
// is free as long as both operands share it: with this one a lane's inputs of x are neighbours.)  Scales lie as [16 outputs]
// [group][output g and g + 8].  Outputs are padded to 16 with scale 0, inputs to 64 with value 0.
//
// Arithmetic.  The weights are exact as bfloat16: a nibble is dropped into the mantissa of 128 and 136 subtracted (4
// instructions for 4 values; integers as the low mantissa bits of a power of two that is subtracted again are a published
// conversion: Kim, Henry, Fahim and Awadalla 2022, for half precision).  Activations are fp32 and enter as three bfloat16
// planes each, x = hi + mid + lo exactly (24 bits cut into 8 + 8 + 8; below 2^-110 the last of them lie under bfloat16's
// smallest step, 2^-133), so no operand is rounded.  m16n8k16 multiplications with fp32 accumulators; the sums of a whole
// group with one or two rows, of 32 inputs with more, start from zero and are added in fp32 with their scale, so sums that
// the matrix units cut off stay short, 128 inputs at most, and finite for |x| up to 2^117 (128 products of up to 8 |x|).
//   * One or two rows: the planes are the columns of one multiplication (2 rows x 3 planes of 8).
//   * Up to 24 rows: eight rows a multiplication, three of them for the planes.  More rows, and most products of more than
//     eight, are taken by q4_rows_tc.cu.
//
// Work.  A CTA takes NT blocks of outputs at a time and splits their inputs over its eight warps, each with a ring of its own
// in shared memory that asynchronous copies fill RING - 1 places ahead (with one or two rows one place, four blocks of inputs,
// requested when the one before it has arrived); the warps' sums meet in shared memory.  The first
// weights are requested before the wait for the kernel ahead in the stream: they never depend on it.
//
// Bounds.  One row: 0.5 byte and 4 / group bytes a weight from HBM, 11 instructions for 8 nibbles.  2048 -> 128256 in groups
// of 64 takes 30.6 to 31.3 us, 4.8 TB/s or 75 % of a copy's rate, with 53 % of the cycles of the integer pipe and 58 % of the
// issue slots taken: nothing is saturated, a warp waits for its one place in flight and then computes while the next one is
// under way.  2048 -> 512 takes 2.2 us, a launch.  Several rows: the latency of eight warps an SM, whose rows come from L2
// two steps ahead (8 x 2048 -> 8192 5.8 us; one step ahead 6.4 % to 14 % longer from 17 rows on).  Fetching them by
// asynchronous copies into shared memory was slower, and two scaled half-precision planes instead of three were not faster.
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <limits>
#include <new>
#include <vector>

#include "host_state.h"

using namespace shainet;

struct shainet_attn_q4 {
    shainet_attn_ctx* ctx = nullptr;
    int device = 0;
    int K = 0, N = 0, group = 32;
    uint4* q = nullptr;        // [N / 16][K / 64][32 lanes], rounded up
    float* scales = nullptr;   // [N / 16][groups][8][2], rounded up
};

namespace {

constexpr unsigned FULL = 0xffffffffu;
constexpr int WARPS = 8, THREADS = WARPS * 32;
constexpr int MAX_MT = 3;               // rows of eight, all in one pass over the weights
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
                const int n = nt * 16 + g + 8 * (i & 1), k = kb * 64 + (s >> 1) * 32 + 8 * t + 4 * (s & 1) + 2 * (i >> 1);
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
            const int k = 2 * j + h, g = n & 7, t = (k & 31) >> 3, s = 2 * ((k & 63) >> 5) + ((k & 7) >> 2), i = ((n >> 3) & 1) + 2 * ((k & 3) >> 1);
            const uint32_t* w = reinterpret_cast<const uint32_t*>(q + ((size_t)(n >> 4) * kbs + (k >> 6)) * 32 + g * 4 + t);
            v |= (k < K ? (w[s] >> (4 * i + 16 * (k & 1))) & 15 : 8) << (4 * h);
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
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// d += a b, or d = a b with FIRST
template <bool FIRST>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
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

// MT = 0: one or two rows, their planes kept in shared memory; else 8 * MT rows at most.  A ring place holds KU blocks of 64
// inputs of each of NT blocks of outputs, and their scales.
template <int MT_, int NT_, int G_>
struct Cfg {
    static constexpr int MT = MT_, NT = NT_, G = G_;                  // G: inputs of a group
    static constexpr int EVEN = G == 128 ? 2 : 1;                     // a warp's blocks of 64 inputs start with a group
    static constexpr int KU = MT == 0 ? 4 : 1;
    static constexpr int PLACE = KU * 640;                            // one block of outputs: 512 bytes a block of inputs, then scales
    static constexpr int UNIT = NT * PLACE;
    static constexpr int RING = MT == 0 ? 2 : NT == 1 ? 5 : 3;        // places of a warp's ring: one in use
    static constexpr int COLS = MT == 0 ? 8 : 8 * MT;                 // columns of the sums: planes and rows, or rows
    static constexpr int RED = COLS + 2;                              // floats between outputs in the sums' meeting place
    static constexpr int SET = WARPS * NT * 16 * RED;                 // floats of a set's sums
    static constexpr int SUMS = (MT == 0 ? 2 : 1) * SET * 4;
    static constexpr size_t FIXED = (size_t)WARPS * RING * UNIT + SUMS;
};

template <class C>
__global__ void __launch_bounds__(THREADS, C::MT == 0 ? (C::NT == 1 ? 3 : 2) : 1) q4_gemv_kernel(Q4GemvArgs a, int kbs, int stored, int blocks) {
    constexpr int MT = C::MT, NT = C::NT, KU = C::KU, TM = MT == 0 ? 1 : MT;
    extern __shared__ __align__(16) unsigned char q4_smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    unsigned char* ring = q4_smem + (size_t)warp * C::RING * C::UNIT;
    float* red = reinterpret_cast<float*>(q4_smem + (size_t)WARPS * C::RING * C::UNIT);
    unsigned char* xs = q4_smem + C::FIXED;                            // MT = 0: [pairs of 16 inputs][column][t][2 x 8 bytes]
    const int slice = ((kbs + WARPS - 1) / WARPS + C::EVEN - 1) / C::EVEN * C::EVEN, kb0 = min(warp * slice, kbs), kb1 = min(kb0 + slice, kbs);
    const int sets = (blocks + NT - 1) / NT;                           // of NT blocks of 16 outputs
    const int rows = a.M;

    // ---- copies: for every set of this CTA the blocks of the warp's slice ----
    const int turned = MT > 0 && kb0 < kb1 ? kb0 + blockIdx.x % (kb1 - kb0) : kb0;
    int ld_set = blockIdx.x, ld_kb = turned;
    uint32_t fill = 0;
    const uint32_t ring_at = static_cast<uint32_t>(__cvta_generic_to_shared(ring)) + lane * 16;
    auto fetch = [&]() {
        if (kb0 < kb1 && ld_set < sets) {
            const int cnt = min(KU, kb1 - ld_kb);
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const int nt = min(ld_set * NT + i, blocks - 1);       // behind the last block: read again, not used
                const uint32_t to = ring_at + fill + i * C::PLACE;
                const uint4* q = a.q + ((size_t)nt * kbs + ld_kb) * 32 + lane;
#pragma unroll
                for (int u = 0; u < KU; ++u)
                    if (u < cnt) copy16(to + u * 512, q + u * 32);
                const int g0 = C::G == 32 ? 2 * ld_kb : C::G == 64 ? ld_kb : ld_kb >> 1, gn = C::G == 32 ? 2 * cnt : C::G == 64 ? cnt : (cnt + 1) >> 1;
                if (lane < 4 * gn) copy16(to + KU * 512, a.scales + ((size_t)nt * stored + g0) * 16 + lane * 4);
            }
            fill = fill == (C::RING - 1) * C::UNIT ? 0 : fill + C::UNIT;
            ld_kb += cnt;
            if (ld_kb == kb1) ld_kb = kb0;
            if (ld_kb == turned) ld_set += gridDim.x;
        }
        copy_commit();
    };
#pragma unroll 1
    for (int i = 0; i < C::RING - 1; ++i) fetch();
    asm volatile("griddepcontrol.wait;" ::: "memory");                 // x may come from the kernel ahead, y may be read by it
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    // inputs k .. k + 3 of a row (k a multiple of four); zeros behind the last input
    const bool by_16 = (a.K & 3) == 0;
    auto four_at = [&](const float* row, int k) {
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (by_16) {
            if (k < a.K) v = __ldcg(reinterpret_cast<const float4*>(row + k));
        } else {
            if (k < a.K) v.x = __ldcg(row + k);
            if (k + 1 < a.K) v.y = __ldcg(row + k + 1);
            if (k + 2 < a.K) v.z = __ldcg(row + k + 2);
            if (k + 3 < a.K) v.w = __ldcg(row + k + 3);
        }
        return v;
    };
    if constexpr (MT == 0) {
        // Column plane * rows + row of a multiplication; the other columns' sums are not looked at, they take the last one's.
        // A lane makes the three planes of four inputs: eight steps of 16 inputs at a time, or four of both rows.
        const int per = rows == 1 ? 8 : 4, m = rows == 1 ? 0 : g & 1, first = rows == 1 ? g : g >> 1;
        const float* row = a.x + (size_t)m * a.K;
#pragma unroll 2
        for (int s = kb0 * 4 + first; s < kb1 * 4; s += per) {
            const float4 v = four_at(row, (s >> 1) * 32 + 8 * t + 4 * (s & 1));
            uint32_t p0[3], p1[3];
            planes(v.x, v.y, p0);
            planes(v.z, v.w, p1);
#pragma unroll
            for (int p = 0; p < 3; ++p)
                *reinterpret_cast<uint2*>(xs + ((size_t)(s >> 1) * 3 * rows + p * rows + m) * 64 + t * 16 + (s & 1) * 8) = make_uint2(p0[p], p1[p]);
        }
        __syncwarp();
    }

    // More rows: x is fetched AHEAD steps (of eight rows and 32 inputs) ahead, straight from L2.  CTAs start at different
    // blocks of their slices: all at the same one would ask the same lines of L2 at the same time (2 %).
    constexpr int AHEAD = 2, VN = AHEAD + 1;
    const float* xrow[TM];
#pragma unroll
    for (int mt = 0; mt < TM; ++mt) xrow[mt] = a.x + (size_t)min(mt * 8 + g, rows - 1) * a.K;      // rows behind the last: not stored
    float4 v[VN][2];
    auto load_step = [&](float4(&to)[2], int kb, int step) {
        const int h = step / TM, mt = step - h * TM, k = kb * 64 + h * 32 + 8 * t;
        to[0] = four_at(xrow[mt], k);
        to[1] = four_at(xrow[mt], k + 4);
    };
    if constexpr (MT > 0)
        if (kb0 < kb1) {
            load_step(v[0], turned, 0);
            load_step(v[1], turned, 1);
        }

    uint32_t take = 0;
    int turn = 0;
#pragma unroll 1
    for (int set = blockIdx.x; set < sets; set += gridDim.x, ++turn) {
        float total[NT][TM][4];
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int mt = 0; mt < TM; ++mt)
#pragma unroll
                for (int c = 0; c < 4; ++c) total[i][mt][c] = 0.0f;
#pragma unroll 1
        for (int at = kb0; at < kb1; at += KU) {
            const int kb = MT == 0 ? at : turned + at - kb0 < kb1 ? turned + at - kb0 : turned + at - kb1;
            copy_wait<C::RING - 2>();
            __syncwarp();
            fetch();                                                   // into the place that the last turn was done with
            const unsigned char* unit = ring + take;
            if constexpr (MT == 0) {
                const int pair = 3 * rows * 64;
                const unsigned char* xb = xs + (size_t)kb * 2 * pair + min(g, 3 * rows - 1) * 64 + t * 16;
                const unsigned char* qb = unit + lane * 16;
                const unsigned char* sb = unit + KU * 512 + g * 8;
                const int cnt = kb1 - kb;
                float c[NT][4];
                auto add = [&](int i, const float(&d)[4], int at) {
                    const float2 sc = *reinterpret_cast<const float2*>(sb + i * C::PLACE + at * 64);
                    total[i][0][0] = fmaf(sc.x, d[0], total[i][0][0]);
                    total[i][0][1] = fmaf(sc.x, d[1], total[i][0][1]);
                    total[i][0][2] = fmaf(sc.y, d[2], total[i][0][2]);
                    total[i][0][3] = fmaf(sc.y, d[3], total[i][0][3]);
                };
#pragma unroll
                for (int u = 0; u < KU; ++u) {
                    if (u >= cnt) break;
                    const uint4 b0 = *reinterpret_cast<const uint4*>(xb), b1 = *reinterpret_cast<const uint4*>(xb + pair);
                    xb += 2 * pair;
#pragma unroll
                    for (int i = 0; i < NT; ++i) {
                        const uint4 w = *reinterpret_cast<const uint4*>(qb + i * C::PLACE + u * 512);
                        uint32_t op[4][4];
                        unpack(w.x, op[0]), unpack(w.y, op[1]), unpack(w.z, op[2]), unpack(w.w, op[3]);
                        if (C::G == 128 && (u & 1)) mma<false>(c[i], op[0], b0.x, b0.y);
                        else mma<true>(c[i], op[0], b0.x, b0.y);
                        mma<false>(c[i], op[1], b0.z, b0.w);
                        if constexpr (C::G == 32) {
                            float d[4];
                            mma<true>(d, op[2], b1.x, b1.y);
                            mma<false>(d, op[3], b1.z, b1.w);
                            add(i, c[i], 2 * u);
                            add(i, d, 2 * u + 1);
                        } else {
                            mma<false>(c[i], op[2], b1.x, b1.y);
                            mma<false>(c[i], op[3], b1.z, b1.w);
                            if (C::G == 64) add(i, c[i], u);
                            else if ((u & 1) || u + 1 == cnt) add(i, c[i], u >> 1);
                        }
                    }
                }
            } else {
                uint32_t op[NT][2][4];
                float2 sc[NT];
                const int next = kb + 1 < kb1 ? kb + 1 : kb0;
#pragma unroll
                for (int s = 0; s < 2 * MT; ++s) {
                    const int h = s / MT, mt = s - h * MT;
                    if (s + AHEAD < 2 * MT) load_step(v[(s + AHEAD) % VN], kb, s + AHEAD);
                    else load_step(v[(s + AHEAD) % VN], next, s + AHEAD - 2 * MT);
                    if (mt == 0) {
#pragma unroll
                        for (int i = 0; i < NT; ++i) {
                            const uint2 w = *reinterpret_cast<const uint2*>(unit + i * C::PLACE + lane * 16 + h * 8);
                            unpack(w.x, op[i][0]), unpack(w.y, op[i][1]);
                            sc[i] = *reinterpret_cast<const float2*>(unit + i * C::PLACE + 512 + (C::G == 32 ? h * 64 : 0) + g * 8);
                        }
                    }
                    uint32_t b[4][3];
                    const float4 u0 = v[s % VN][0], u1 = v[s % VN][1];
                    planes(u0.x, u0.y, b[0]), planes(u0.z, u0.w, b[1]), planes(u1.x, u1.y, b[2]), planes(u1.z, u1.w, b[3]);
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
                // what is under way for the next block stands where that one looks for it
                constexpr int R = 2 * MT % VN;
                if constexpr (R != 0) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float4 w0 = v[R][i], w1 = v[(R + 1) % VN][i];
                        v[0][i] = w0, v[1][i] = w1;
                    }
                }
            }
            __syncwarp();
            take = take == (C::RING - 1) * C::UNIT ? 0 : take + C::UNIT;
        }
        // ---- the warps' sums ----
        float* meet = red + (MT == 0 ? (turn & 1) * C::SET : 0);
        float* to = meet + warp * NT * 16 * C::RED;
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int mt = 0; mt < TM; ++mt)
#pragma unroll
                for (int r = 0; r < 2; ++r)
                    *reinterpret_cast<float2*>(to + (i * 16 + g + 8 * r) * C::RED + mt * 8 + 2 * t) = make_float2(total[i][mt][2 * r], total[i][mt][2 * r + 1]);
        __syncthreads();
        if constexpr (MT == 0) {
            // one warp adds, another one every time; the next sums go to the other half
            if (warp == (turn & (WARPS - 1))) {
#pragma unroll 1
                for (int e = lane; e < NT * 16 * rows; e += 32) {
                    const int m = e / (NT * 16), n = e - m * (NT * 16), out = set * (NT * 16) + n;
                    float sum = 0.0f;
#pragma unroll
                    for (int w = 0; w < WARPS; ++w) {
                        const float* s = meet + (w * (NT * 16) + n) * C::RED + m;
                        sum += s[2 * rows] + s[rows] + s[0];
                    }
                    if (out < a.N) a.y[(size_t)m * a.N + out] = sum;
                }
            }
        } else {
#pragma unroll 1
            for (int e = tid; e < NT * 16 * rows; e += THREADS) {
                const int m = e / (NT * 16), n = e - m * (NT * 16), out = set * NT * 16 + n;
                float sum = 0.0f;
#pragma unroll
                for (int w = 0; w < WARPS; ++w) sum += meet[(w * NT * 16 + n) * C::RED + m];
                if (out < a.N) a.y[(size_t)m * a.N + out] = sum;
            }
            __syncthreads();
        }
    }
    copy_wait<0>();
}

size_t plane_bytes(const Q4GemvArgs& a) { return (size_t)blocks_of(a.K, 64) * 2 * 3 * a.M * 64; }

// One or two rows whose planes a CTA holds beside its rings: up to 28992 inputs of one, 14464 of two.
bool planes_fit(const Q4GemvArgs& a) {
    static_assert(Cfg<0, 1, 32>::FIXED == Cfg<0, 1, 64>::FIXED && Cfg<0, 1, 32>::FIXED == Cfg<0, 1, 128>::FIXED, "one rule for all groups");
    return a.M <= 2 && Cfg<0, 1, 32>::FIXED + plane_bytes(a) <= SMEM_MAX;
}

template <int MT, int NT, int G>
cudaError_t launch(const Q4GemvArgs& a, int sm_count, cudaStream_t s) {
    using C = Cfg<MT, NT, G>;
    const int kbs = blocks_of(a.K, 64), blocks = blocks_of(a.N, 16), sets = blocks_of(blocks, NT);
    const size_t smem = C::FIXED + (MT == 0 ? plane_bytes(a) : 0);
    static std::atomic<unsigned long long> configured{0};   // bit per device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !(configured.load(std::memory_order_acquire) >> dev & 1ull)) {
        e = cudaFuncSetAttribute(q4_gemv_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_MAX);
        if (e != cudaSuccess) return e;
        if (dev < 64) configured.fetch_or(1ull << dev, std::memory_order_release);
    }
    const int per_sm = MT == 0 ? std::max(1, std::min(NT == 1 ? 3 : 2, (int)(227 * 1024 / (smem + 1024)))) : 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(std::min(sets, sm_count * per_sm));
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

template <int MT, int G>
cudaError_t launch_rows(const Q4GemvArgs& a, int sm_count, cudaStream_t s) {
    // blocks of outputs that share the planes of x: four or two where that still leaves a CTA for most SMs (us with one, two and
    // four: 8 x 2048 -> 2048 3.8, 4.2, 5.5; 8 x 4096 -> 4096 10.8, 7.3, 9.7; 8 x 2048 -> 8192 11.3, 7.5, 5.7)
    const long long work = blocks_of(a.N, 16), most = sm_count * 3 / 4;
    return work >= 4 * most ? launch<MT, 4, G>(a, sm_count, s) : work >= 2 * most ? launch<MT, 2, G>(a, sm_count, s) : launch<MT, 1, G>(a, sm_count, s);
}

template <int G>
cudaError_t launch_group(const Q4GemvArgs& a, int sm_count, cudaStream_t s) {
    if (planes_fit(a)) {
        // two blocks of outputs share the reads of x's planes where every CTA has several of them (128256 outputs 32.9 us with one,
        // 30.7 with two; 20000 and 40000 the same)
        return blocks_of(a.N, 16) >= 8 * sm_count && Cfg<0, 2, G>::FIXED + plane_bytes(a) <= 112 * 1024 ? launch<0, 2, G>(a, sm_count, s) : launch<0, 1, G>(a, sm_count, s);
    }
    static_assert(MAX_MT == 3, "one instance for each");
    return a.M <= 8 ? launch_rows<1, G>(a, sm_count, s) : a.M <= 16 ? launch_rows<2, G>(a, sm_count, s) : launch_rows<3, G>(a, sm_count, s);
}

}  // namespace

namespace shainet {

cudaError_t launch_q4_gemv(const Q4GemvArgs& a, int sm_count, cudaStream_t s) {
    // The tensor cores of tcgen05 (us, here / there): from 25 rows on (700 x 900, 40 rows 6.8 / 5.5; 512 x 1000, 40 rows 4.3 / 4.6;
    // 2048 x 8192, 33 rows 17.6 / 10.6); from nine on but for short sums into few outputs, which end before that kernel has
    // filled its rings (16 rows: 512 x 1000 2.5 / 4.6, 1000 x 4000 4.6 / 4.7, 1500 x 400 5.0 / 4.6; 12 rows: 300 x 20000 8.8 / 5.0,
    // 64 x 60000 14 / 8, 2048 x 8192 9.9 / 8.4); from three on where a warp's slice is long (8 rows: 2048 x 8192 5.7 / 8.2, 8192 x 2048 10.4 / 10.9,
    // 11000 x 5000 33 / 18).
    const bool small = a.K <= 1024 && a.N <= 8192 && a.K * a.N <= 4 << 20;
    // One or two rows whose planes do not fit there: groups of 64 and 128 (two rows: 14528 x 4096 23.1 / 20.2, 16384 x 2048 21.7 / 17.1,
    // 28672 x 8192 59 / 53, 28672 x 9600 112 / 70, 28672 x 28672 221 / 197, 14528 x 20000 93 / 102; one: 30000 x 2048 39 / 29, 40000 x 5000
    // 116 / 50); groups of 32, whose sums it reads out twice as often, stay (two rows: 14528 x 4096 22.4 / 27.8, 28672 x 8192
    // 62 / 76, 28672 x 28672 236 / 297, 28672 x 1000 39.5 / 38.5, 28672 x 9600 118 / 100; one: 30000 x 2048 40 / 41).
    const bool wide = a.M > 2 ? a.K > 8192 : !planes_fit(a) && a.group > 32;
    if (a.M > 8 * MAX_MT || (a.M > 8 && !small) || wide) return launch_q4_rows(a, stored_groups(a.K, a.group), sm_count, s);
    return a.group == 32 ? launch_group<32>(a, sm_count, s) : a.group == 64 ? launch_group<64>(a, sm_count, s) : launch_group<128>(a, sm_count, s);
}

}  // namespace shainet

namespace {

size_t packed_bytes(int K, int N) { return (size_t)N * ((K + 1) / 2); }
size_t scale_count(int K, int N, int group) { return (size_t)N * blocks_of(K, group); }
int grid_of(long long items) { return (int)std::min<long long>((items + 255) / 256, 16384); }

// As the Q8_0 quantiser: per output and group scale = max|w| / 7 (1 for an all-zero group), round to nearest even.  Groups of
// tiny values, which that one has no rule for: a scale is fp32's smallest step at least, and where 1 / scale overflows the
// values are divided (0 times infinity would be no zero).  False where a weight is not finite: no nibble stands for it.
bool quantize_q4(const float* w, int K, int N, int group, uint8_t* packed, float* scales) {
    const int groups = blocks_of(K, group), bytes = (K + 1) / 2;
    for (int n = 0; n < N; ++n) {
        uint8_t* row = packed + (size_t)n * bytes;
        std::fill(row, row + bytes, (uint8_t)0x88);
        for (int g = 0; g < groups; ++g) {
            const int base = g * group, lim = std::min(base + group, K);
            float max_abs = 0.0f;
            for (int k = base; k < lim; ++k) {
                if (!std::isfinite(w[(size_t)k * N + n])) return false;
                max_abs = std::max(max_abs, fabsf(w[(size_t)k * N + n]));
            }
            const float scale = max_abs > 0.0f ? std::max(max_abs / 7.0f, std::numeric_limits<float>::denorm_min()) : 1.0f, inv = 1.0f / scale;
            const bool tiny = !std::isfinite(inv);
            scales[(size_t)n * groups + g] = scale;
            for (int k = base; k < lim; ++k) {
                const float v = std::min(7.0f, std::max(-7.0f, nearbyintf(tiny ? w[(size_t)k * N + n] / scale : w[(size_t)k * N + n] * inv)));
                const uint8_t u = (uint8_t)((int)v + 8);
                row[k / 2] = (uint8_t)((k & 1) ? (row[k / 2] & 0x0f) | (u << 4) : (row[k / 2] & 0xf0) | u);
            }
        }
    }
    return true;
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
    if (!host && (reinterpret_cast<uintptr_t>(scales) & 3u) != 0) return fail(SHAINET_ATTN_E_INVALID, "device scales must be 4-byte aligned");
    if (!ctx) return fail(SHAINET_ATTN_E_INVALID, "null context");
    DeviceGuard g(ctx->device);
    shainet_attn_q4* w = new (std::nothrow) shainet_attn_q4();
    if (!w) return fail(SHAINET_ATTN_E_NOMEM, "out of host memory");
    w->ctx = ctx;
    w->device = ctx->device;
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
    if (!quantize_q4(w, K, N, group, q.data(), sc.data())) return fail(SHAINET_ATTN_E_INVALID, "a weight is not finite");
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
    DeviceGuard g(w->device);      // not the context's: it may be gone
    cudaDeviceSynchronize();
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
    a.status = ctx->status_dev;
    CU(launch_q4_gemv(a, ctx->sm_count, stream ? (cudaStream_t)stream : ctx->stream));
    return SHAINET_ATTN_OK;
}

}  // extern "C"
