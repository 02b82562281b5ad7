// Products of several activation rows with 4-bit weights on the 5th-generation tensor cores (tcgen05), sm_100a; the formula and
// the layout are those of q4_gemv.cu.
//
// A CTA computes 256 outputs of up to NT rows, as two halves of 128.  The weights are the A operand: a thread owns an
// output, unpacks 64 of its nibbles at a time into bfloat16 (exact) and puts them into tensor memory.  The rows are the B
// operand: fp32 values as three bfloat16 planes (exact, as in q4_gemv.cu), made in the CTA, side by side as 3 NT columns of one
// multiplication.  The sums of 32 (groups of 32), 64 or 128 inputs start from zero in tensor memory; the accumulating warps, a
// thread an output again, add the three columns of a row and multiply by the group's scale in fp32.
//
// Where there are fewer tiles than SMs, the CTAs of a cluster share a tile's inputs and add their sums through distributed
// shared memory, in the order of their ranks.  Rows are cut into more passes where SMs would be idle even so.
//
// Bounds.  A multiplication of 16 inputs takes 64 cycles for up to 128 columns (40 rows), 96 for 192 (64 rows): 512 or 768 cycles a
// step of 64 inputs x 256 outputs.  A step takes 900 (12 rows), 1000 (33) and 1700 (64): the warps that unpack, make planes and
// accumulate take two thirds of the issue slots and each of the three chains is nearly as long as a step (without the unpacking
// 17 % less at 9 rows, with an eighth of the read-out 27 % less at 64, with an eighth of the planes 9 %).  That is why
// two warpgroups take the blocks of the rows in turn (124 -> 118 us at 64 x 2048 x 128256) and each half has a warp of its own
// that issues the multiplications, with slots and parities that are constants (one warp for both: 1450 cycles a step).  Rows
// through registers instead of the ring took 9 % longer, a read-out two places deep as long.
// Measured: 33 x 2048 -> 8200 10.6 us, 64 x 4096 -> 4096 16.5 us, 64 x 2048 -> 128256 118 to 126 us by the card (mma.sync, which takes 8.5 cycles of a
// quarter SM for 16 outputs and eight columns: 17.6, 27.4 and 426).  A launch with little to do takes 4.4 us.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "kernels.h"
#include "tcgen05.cuh"

namespace shainet {

namespace {

typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pack2(uint32_t lo, uint32_t hi) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
    return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
    f32x2 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ float half_of(f32x2 v, int h) {
    float lo, hi;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
    return h ? hi : lo;
}

// 16 or 4 bytes global -> shared; `bytes` 0: zeros, nothing is read
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <int N>
__device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

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

// Every warp is behind this before it waits for another one: the time limit of those waits does not run while the kernel ahead in
// the stream does.
__device__ __forceinline__ void launched_ahead() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// A place of a ring of N and the parity of its round.
template <int N>
struct Ring {
    int slot = 0;
    uint32_t parity = 0;
    __device__ __forceinline__ void next() {
        if (++slot == N) {
            slot = 0;
            parity ^= 1;
        }
    }
};

// NT: rows of a pass; G: inputs of a group.
template <int NT_, int G_>
struct Tile {
    static constexpr int NT = NT_, G = G_;
    static constexpr int OUTS = 256;
    static constexpr int GB = G == 128 ? 2 : 1;                  // blocks of 64 inputs that are summed in tensor memory
    static constexpr int PARTS = G == 32 ? 2 : 1;                // sums of one block
    static constexpr int COLS = (3 * NT + 15) / 16 * 16;         // columns of a multiplication
    static constexpr int D_COLS = (COLS + 31) / 32 * 32;
    static constexpr int A_COLS = 32, A_SLOTS = 2;               // 64 bfloat16 a lane; slots of each half
    static constexpr int TMEM_COLS = 512, TMEM_A = TMEM_COLS - 2 * A_SLOTS * A_COLS;
    static constexpr int DH = TMEM_A / D_COLS >= 4 ? 2 : 1;      // sums of each half
    static constexpr int NB = 4, B_BYTES = COLS * 128;           // stages of planes, 64 inputs each, 128-byte swizzle
    static constexpr int NX = NT <= 40 ? 3 : 2, X_BYTES = NT * 256;      // stages of fp32 rows, of two warpgroups
    static constexpr int NW = 6, W_BYTES = 1024;                 // stages of a converting warp: 32 outputs x 64 inputs
    static constexpr int NS = 8, S_BYTES = 128;                  // stages of an accumulating warp: a scale of 32 outputs
    static constexpr int AT_X = NB * B_BYTES, AT_W = AT_X + 2 * NX * X_BYTES, AT_S = AT_W + 8 * NW * W_BYTES, AT_BARS = AT_S + 8 * NS * S_BYTES;
    static constexpr int BARS = 2 * NB + 4 * A_SLOTS + 4 * DH;
    static constexpr int USED = AT_BARS + BARS * 8 + 16;
    // Never two CTAs on an SM, nor another kernel that allocates tensor memory beside one: a cluster's CTA could wait for columns
    // that are held by one which waits for a CTA of the first cluster.
    static constexpr int SMEM = USED < 200 * 1024 ? 200 * 1024 : USED;
    static_assert(2 * DH * D_COLS <= TMEM_A && SMEM <= 227 * 1024, "tensor and shared memory");
    static_assert(NT * OUTS * 4 <= AT_W, "a cluster's sums take the place of the rows");
    static_assert(NT % 8 == 0, "rows are read from tensor memory eight at a time");
};

constexpr int MAX_SPLITS = 8;      // CTAs of a cluster
constexpr int THREADS = 896;     // seven warpgroups: multiply, rows (two), convert (two), accumulate (two)

// fp32 accumulation, bfloat16 operands, both K-major
__host__ __device__ constexpr uint32_t instruction(int M, int N) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

__device__ __forceinline__ float4 load_cluster(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}

template <class C>
__global__ void __launch_bounds__(THREADS, 1) q4_rows_kernel(Q4GemvArgs a, int kbs, int stored, int blocks, int tiles) {
    constexpr int NT = C::NT, GB = C::GB, PARTS = C::PARTS, DH = C::DH, NB = C::NB;
    extern __shared__ __align__(1024) unsigned char qr_smem[];
    uint64_t* b_full = reinterpret_cast<uint64_t*>(qr_smem + C::AT_BARS);      // NB: four row warps
    uint64_t* b_free = b_full + NB;                                            // NB: both halves' multiplications
    uint64_t* a_full = b_free + NB;                                            // [half][slot]: four converting warps
    uint64_t* a_free = a_full + 2 * C::A_SLOTS;                                // [half][slot]: the multiplications
    uint64_t* d_full = a_free + 2 * C::A_SLOTS;                                // [half][DH]: the multiplications
    uint64_t* d_free = d_full + 2 * DH;                                        // [half][DH]: four accumulating warps
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(d_free + 2 * DH);
    const int warp = uniform_warp_index(), lane = threadIdx.x & 31, wg = warp >> 2, quad = warp & 3;
    if (threadIdx.x == 0) {
        for (int i = 0; i < NB; ++i) mbar_init(&b_full[i], 4), mbar_init(&b_free[i], 2);
        for (int i = 0; i < 2 * C::A_SLOTS; ++i) mbar_init(&a_full[i], 4), mbar_init(&a_free[i], 1);
        for (int i = 0; i < 2 * DH; ++i) mbar_init(&d_full[i], 1), mbar_init(&d_free[i], 4);
        fence_mbar_init();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(C::TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    constexpr uint32_t tmem = 0;     // all columns are this CTA's

    // The CTAs of a cluster take equal slices of the inputs, whole groups; clusters take tiles in turn.
    int splits = 1, z = 0;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(splits));
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(z));
    const int first = blockIdx.x / splits, step = gridDim.x / splits;
    const int groups = (kbs + GB - 1) / GB;
    const int kb0 = min(kbs, groups * z / splits * GB), kb1 = min(kbs, groups * (z + 1) / splits * GB);
    const int m0 = blockIdx.y * a.pass_rows, rows = min(a.pass_rows, a.M - m0);
    const int total = first < tiles ? ((tiles - first + step - 1) / step) * (kb1 - kb0) : 0;      // blocks of 64 inputs in all

    if (wg == 0) {
        fewer_registers<40>();
        // ---- multiply: a warp for each half.  Slots and parities of a round of NB blocks are constants: what this warp executes
        // between two multiplications is what bounds small tiles ----
        auto multiply = [&](auto half) {
            constexpr int h = decltype(half)::value;
            constexpr uint32_t idesc = instruction(128, C::COLS);
            const uint64_t desc0 = smem_desc_sw128(smem_u32(qr_smem), 16, 1024);
            uint32_t round = 0, d_round = 0;
            int left = kb1 - kb0, summed = 0;                                  // blocks of the slice that are left, of the sum that is open
#pragma unroll 1
            for (int n = 0; n < total; n += NB, round ^= 1) {
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    if (n + b >= total) return;
                    const bool fresh = GB == 1 || summed == 0, last = GB == 1 || summed == 1 || left == 1;
                    if (!mbar_wait(&b_full[b], round, a.status, 90)) return;
                    if (!mbar_wait(&a_full[h * 2 + (b & 1)], b >> 1, a.status, 91)) return;
#pragma unroll
                    for (int part = 0; part < PARTS; ++part) {
                        const int sum = b * PARTS + part;
                        const int place = DH == 1 ? 0 : GB == 1 ? sum & 1 : (int)(d_round & 1);
                        const uint32_t parity = GB == 1 ? (DH == 1 ? sum : sum >> 1) & 1 : DH == 1 ? d_round & 1 : d_round >> 1 & 1;
                        if (fresh && !mbar_wait(&d_free[h * DH + place], parity ^ 1u, a.status, 92)) return;
                        tc_fence_after();
                        const uint32_t d = tmem + (h * DH + place) * C::D_COLS;
                        if (elect_one()) {
#pragma unroll
                            for (int k = 0; k < 4 / PARTS; ++k) {
                                const int kk = part * (4 / PARTS) + k;
                                mma_ts_bf16(d, tmem + C::TMEM_A + (h * 2 + (b & 1)) * C::A_COLS + kk * 8, desc0 + (uint64_t)((b * C::B_BYTES + kk * 32) >> 4), idesc,
                                            !fresh || k > 0 ? 1u : 0u);
                            }
                            if (last) tc_commit(&d_full[h * DH + place]);
                            if (part == PARTS - 1) {                           // nobody waits for the last ones
                                if (n + b + 2 < total) tc_commit(&a_free[h * 2 + (b & 1)]);
                                if (n + b + NB < total) tc_commit(&b_free[b]);
                            }
                        }
                        __syncwarp();
                    }
                    if (GB == 2) {
                        summed = last ? 0 : 1;
                        d_round += last ? 1 : 0;
                        left = left == 1 ? kb1 - kb0 : left - 1;
                    }
                }
            }
        };
        launched_ahead();
        if (warp == 0) multiply(std::integral_constant<int, 0>{});
        if (warp == 2) multiply(std::integral_constant<int, 1>{});
    } else if (wg < 3) {
        // ---- rows: two warpgroups take blocks in turn; fp32 from L2 by asynchronous copies, every thread converts the pieces that
        // it requested ----
        fewer_registers<48>();
        constexpr int PIECES = NT / 8;
        const int tid = threadIdx.x - wg * 128, c4 = tid & 15, t0 = tid >> 4;  // piece j: row t0 + 8 j, inputs 4 c4 .. + 3
        const bool by_16 = (a.K & 3) == 0;
        const uint32_t raw = smem_u32(qr_smem + C::AT_X) + (wg - 1) * (C::NX * C::X_BYTES) + tid * 16;
        const unsigned char* from = qr_smem + C::AT_X + (wg - 1) * (C::NX * C::X_BYTES) + tid * 16;
        const float* row = a.x + (size_t)(m0 + min(t0, rows - 1)) * a.K + c4 * 4;
        const int pieces = t0 < rows ? (rows - t0 + 7) / 8 : 0;                // rows behind the last one: whatever stands in the stages
        const size_t stride = (size_t)8 * a.K;
        const int slice = kb1 - kb0;
        int ld = wg - 1, ld_kb = kb0 + (slice > 0 ? ld % slice : 0);
        uint32_t fill = 0;
        auto fetch = [&]() {
            if (ld < total) {
                const int left = a.K - ld_kb * 64 - c4 * 4;                    // inputs of this piece; zeros behind the last
                const float* src = left > 0 ? row + ld_kb * 64 : a.x;
                const size_t by = left > 0 ? stride : 0;
                if (by_16) {
                    const int bytes = left > 0 ? 16 : 0;
#pragma unroll
                    for (int j = 0; j < PIECES; ++j) {
                        if (j >= pieces) break;
                        copy16(raw + fill + j * 2048, src, bytes);
                        src += by;
                    }
                } else {
#pragma unroll 1
                    for (int j = 0; j < pieces; ++j)
                        for (int e = 0; e < 4; ++e) copy4(raw + fill + j * 2048 + e * 4, left > e ? src + j * by + e : a.x, left > e ? 4 : 0);
                }
                fill = fill == (C::NX - 1) * C::X_BYTES ? 0 : fill + C::X_BYTES;
                ld += 2;
                ld_kb += 2;
                while (ld_kb >= kb1) ld_kb -= slice;
            }
            copy_commit();
        };
        launched_ahead();                                                      // x may come from the kernel ahead
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
#pragma unroll 1
        for (int i = 0; i < C::NX - 1; ++i) fetch();
        uint32_t take = 0;
#pragma unroll 1
        for (int n = wg - 1; n < total; n += 2) {
            copy_wait<C::NX - 2>();
            fetch();                                                           // over what this thread converted last
            const int slot = n & (NB - 1);
            if (!mbar_wait(&b_free[slot], (uint32_t)(n / NB & 1) ^ 1u, a.status, 93)) break;
            unsigned char* stage = qr_smem + slot * C::B_BYTES + t0 * 128 + (((c4 >> 1) ^ t0) << 4) + (c4 & 1) * 8;
#pragma unroll
            for (int j = 0; j < PIECES; ++j) {
                if (j >= pieces) break;
                const float4 v = *reinterpret_cast<const float4*>(from + take + j * 2048);
                uint32_t p0[3], p1[3];
                planes(v.x, v.y, p0);
                planes(v.z, v.w, p1);
#pragma unroll
                for (int p = 0; p < 3; ++p) *reinterpret_cast<uint2*>(stage + (p * NT + 8 * j) * 128) = make_uint2(p0[p], p1[p]);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&b_full[slot]);
            take = take == (C::NX - 1) * C::X_BYTES ? 0 : take + C::X_BYTES;
        }
        copy_wait<0>();
    } else if (wg < 5) {
        // ---- convert: a thread an output of half h; constants, nothing to wait for but free places ----
        fewer_registers<64>();
        const int h = wg - 3, cw = warp - 12;
        unsigned char* ring = qr_smem + C::AT_W + cw * (C::NW * C::W_BYTES);
        const int g = lane >> 2, t = lane & 3;                                 // of the piece that this lane copies
        const uint32_t to = smem_u32(ring) + (g * 4 + (t ^ ((g >> 1) & 3))) * 16;
        int ld_tile = first, ld_kb = kb0;
        uint32_t fill = 0;
        const uint4* src[2];
        auto begin = [&]() {
#pragma unroll
            for (int i = 0; i < 2; ++i) {                                      // behind the last block: read again, not used
                const int nt = min(ld_tile * 16 + h * 8 + quad * 2 + i, blocks - 1);
                src[i] = a.q + ((size_t)nt * kbs + kb0) * 32 + lane;
            }
        };
        begin();
        auto fetch = [&]() {
            if (ld_tile < tiles) {
                copy16(to + fill, src[0], 16);
                copy16(to + fill + 512, src[1], 16);
                src[0] += 32, src[1] += 32;
                fill = fill == (C::NW - 1) * C::W_BYTES ? 0 : fill + C::W_BYTES;
                if (++ld_kb == kb1) {
                    ld_kb = kb0, ld_tile += step;
                    begin();
                }
            }
            copy_commit();
        };
#pragma unroll 1
        for (int i = 0; i < C::NW - 1; ++i) fetch();
        launched_ahead();
        const int rg = lane & 7, hi = (lane >> 3) & 1, turn = (rg >> 1) & 3;   // of the output that this lane unpacks
        const unsigned char* from = ring + (lane >> 4) * 512 + rg * 64;
        const uint32_t a_at = tmem + ((uint32_t)(quad * 32) << 16) + C::TMEM_A + h * C::A_SLOTS * C::A_COLS;
        Ring<C::A_SLOTS> ra;
        uint32_t take = 0;
#pragma unroll 1
        for (int n = 0; n < total; ++n) {
            copy_wait<C::NW - 2>();
            __syncwarp();
            fetch();
            uint32_t out[32];
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                const uint4 q = *reinterpret_cast<const uint4*>(from + take + ((p ^ turn) << 4));
                const uint32_t words[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    const uint32_t w = words[s] >> (4 * hi);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        uint32_t v;
                        asm("lop3.b32 %0, %1, 0x000f000f, 0x43004300, 0xea;" : "=r"(v) : "r"(w >> (8 * e)));      // (w & mask) | 128.0
                        asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(out[16 * (s >> 1) + 4 * p + 2 * (s & 1) + e])
                            : "r"(v), "r"(0x3f803f80u), "r"(0xc308c308u));                                       // * 1 - 136
                    }
                }
            }
            if (!mbar_wait(&a_free[h * C::A_SLOTS + ra.slot], ra.parity ^ 1u, a.status, 94)) break;
            tc_fence_after();
            tmem_st32(a_at + ra.slot * C::A_COLS, out);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&a_full[h * C::A_SLOTS + ra.slot]);
            ra.next();
            take = take == (C::NW - 1) * C::W_BYTES ? 0 : take + C::W_BYTES;
        }
        copy_wait<0>();
    } else {
        // ---- accumulate: a thread an output of half h, NT sums ----
        more_registers<120>();
        const int h = wg - 5, aw = warp - 20, r = h * 128 + quad * 32 + lane;
        const uint32_t scale_at = smem_u32(qr_smem + C::AT_S) + (aw * C::NS * 32 + lane) * 4;
        const float* scale_from = reinterpret_cast<const float*>(qr_smem + C::AT_S) + aw * C::NS * 32 + lane;
        int ld_tile = first, ld_g = 0;
        const int g0 = PARTS == 2 ? kb0 * 2 : kb0 / GB, gn = (PARTS == 2 ? kb1 * 2 : (kb1 + GB - 1) / GB) - g0;      // this CTA's groups
        int fill = 0;
        const float* src = nullptr;
        auto begin = [&]() { src = a.scales + ((size_t)min(ld_tile * 16 + (r >> 4), blocks - 1) * stored + g0) * 16 + (lane & 7) * 2 + ((lane >> 3) & 1); };
        begin();
        auto fetch = [&]() {
            if (ld_tile < tiles) {
                copy4(scale_at + fill * 128, src, 4);
                src += 16;
                fill = (fill + 1) & (C::NS - 1);
                if (++ld_g == gn) {
                    ld_g = 0, ld_tile += step;
                    begin();
                }
            }
            copy_commit();
        };
#pragma unroll 1
        for (int i = 0; i < C::NS - 1; ++i) fetch();
        launched_ahead();                                                      // y may be read by the kernel ahead
        const uint32_t d_at = tmem + ((uint32_t)(quad * 32) << 16);
        Ring<DH> rd;
        int take = 0;
        bool ok = true;
        for (int w = first; ok && w < tiles; w += step) {
            f32x2 acc[NT / 2];
#pragma unroll
            for (int c = 0; c < NT / 2; ++c) acc[c] = 0ull;
#pragma unroll 1
            for (int n = 0; n < gn; ++n) {
                copy_wait<C::NS - 2>();
                fetch();
                const uint32_t s = __float_as_uint(scale_from[take * 32]);
                const f32x2 s2 = pack2(s, s);
                take = (take + 1) & (C::NS - 1);
                if (!(ok = mbar_wait(&d_full[h * DH + rd.slot], rd.parity, a.status, 95))) break;
                tc_fence_after();
                const uint32_t da = d_at + (h * DH + rd.slot) * C::D_COLS;
#pragma unroll
                for (int c = 0; c < NT; c += 8) {
                    uint32_t v0[8], v1[8], v2[8];
                    tmem_ld8(da + c, v0);
                    tmem_ld8(da + NT + c, v1);
                    tmem_ld8(da + 2 * NT + c, v2);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 8; ++e) asm volatile("" : "+r"(v0[e]), "+r"(v1[e]), "+r"(v2[e]));      // used behind the wait only
                    if (c + 8 == NT) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&d_free[h * DH + rd.slot]);
                    }
#pragma unroll
                    for (int e = 0; e < 8; e += 2) {
                        const f32x2 low = add2(pack2(v2[e], v2[e + 1]), pack2(v1[e], v1[e + 1]));
                        acc[(c + e) / 2] = fma2(add2(low, pack2(v0[e], v0[e + 1])), s2, acc[(c + e) / 2]);
                    }
                }
                rd.next();
            }
            if (splits == 1) {
                if (!ok) break;
                const int out = w * C::OUTS + r;
                float* y = a.y + (size_t)m0 * a.N + out;
                if (out < a.N) {
#pragma unroll
                    for (int c = 0; c < NT; ++c)
                        if (c < rows) y[(size_t)c * a.N] = half_of(acc[c / 2], c & 1);
                }
            } else {
                // One tile.  Both halves are through, so every multiplication is: the sums take the place of the rows.
                asm volatile("bar.sync 1, 256;" ::: "memory");
                float* sums = reinterpret_cast<float*>(qr_smem) + r;
#pragma unroll
                for (int c = 0; c < NT; ++c) sums[c * C::OUTS] = half_of(acc[c / 2], c & 1);
            }
        }
        copy_wait<0>();
        if (splits > 1) {
            cluster_sync_all();
            // the rows of rank z, the parts in the order of their ranks
            const int mine = (rows - z + splits - 1) / splits, out0 = first * C::OUTS;
            const uint32_t sums = smem_u32(qr_smem);
#pragma unroll 1
            for (int e = threadIdx.x - 640; e < mine * (C::OUTS / 4); e += 256) {
                const int c = z + e / (C::OUTS / 4) * splits, o = e % (C::OUTS / 4) * 4;
                float4 part[MAX_SPLITS];
#pragma unroll
                for (int k = 0; k < MAX_SPLITS; ++k)
                    if (k < splits) part[k] = load_cluster(map_to_cta(sums + (c * C::OUTS + o) * 4, k));
                float4 sum = part[0];
#pragma unroll
                for (int k = 1; k < MAX_SPLITS; ++k)
                    if (k < splits) sum.x += part[k].x, sum.y += part[k].y, sum.z += part[k].z, sum.w += part[k].w;
                float* y = a.y + (size_t)(m0 + c) * a.N + out0 + o;
                if ((a.N & 3) == 0 && out0 + o < a.N) {
                    *reinterpret_cast<float4*>(y) = sum;
                } else {
                    const float four[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (out0 + o + i < a.N) y[i] = four[i];
                }
            }
        }
    }
    if (splits > 1 && wg < 5) cluster_sync_all();                              // the barrier ahead of the sums
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::TMEM_COLS) : "memory");
    }
    if (splits > 1) cluster_sync_all();                                        // nobody leaves while its sums are read
}

template <int NT, int G>
cudaError_t launch(const Q4GemvArgs& a, int stored, int sm_count, cudaStream_t s) {
    using C = Tile<NT, G>;
    const int kbs = (a.K + 63) / 64, blocks = (a.N + 15) / 16, tiles = (a.N + C::OUTS - 1) / C::OUTS, passes = (a.M + a.pass_rows - 1) / a.pass_rows;
    static std::atomic<unsigned long long> configured{0};   // bit per device
    static std::atomic<int> room[64][MAX_SPLITS + 1];       // clusters of a size that run at once
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !(configured.load(std::memory_order_acquire) >> dev & 1ull)) {
        e = cudaFuncSetAttribute(q4_rows_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
        if (e != cudaSuccess) return e;
        if (dev < 64) configured.fetch_or(1ull << dev, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg{};
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    // CTAs of a cluster: the most with which all clusters run at once (sizes that do not divide the SMs of a GPC leave some of
    // them idle), four blocks of inputs each at least
    int splits = 1;
    for (int k = MAX_SPLITS; k > 1; --k)
        if ((long long)tiles * passes * k <= sm_count && kbs >= 4 * k) {
            int most = dev < 64 ? room[dev][k].load(std::memory_order_relaxed) : 0;
            if (most == 0) {
                at[1].val.clusterDim.x = k;
                cfg.gridDim = dim3(k);
                e = cudaOccupancyMaxActiveClusters(&most, q4_rows_kernel<C>, &cfg);
                if (e != cudaSuccess) return e;
                if (dev < 64) room[dev][k].store(most, std::memory_order_relaxed);
            }
            if (tiles * passes <= most) {
                splits = k;
                break;
            }
        }
    at[1].val.clusterDim.x = splits;
    cfg.gridDim = dim3(splits > 1 ? tiles * splits : std::min(tiles, std::max(1, sm_count / passes)), passes);
    return cudaLaunchKernelEx(&cfg, q4_rows_kernel<C>, a, kbs, stored, blocks, tiles);
}

template <int G>
cudaError_t launch_group(Q4GemvArgs a, int stored, int sm_count, cudaStream_t s) {
    // Up to 64 rows a pass over the weights; fewer where SMs would be idle (5000 x 100, 64 rows: 13.9 us with one pass, 7.5 with four).
    int passes = (a.M + 63) / 64;
    const long long ctas = (long long)((a.N + 255) / 256) * std::min(MAX_SPLITS, std::max(1, a.K / 256));
    while (ctas * passes * 2 <= sm_count && a.M > 16 * passes) passes *= 2;
    a.pass_rows = (a.M + passes - 1) / passes;
    if (a.pass_rows <= 16) return launch<16, G>(a, stored, sm_count, s);
    if (a.pass_rows <= 32) return launch<32, G>(a, stored, sm_count, s);
    return a.pass_rows <= 40 ? launch<40, G>(a, stored, sm_count, s) : launch<64, G>(a, stored, sm_count, s);
}

}  // namespace

cudaError_t launch_q4_rows(const Q4GemvArgs& a, int stored, int sm_count, cudaStream_t s) {
    return a.group == 32 ? launch_group<32>(a, stored, sm_count, s) : a.group == 64 ? launch_group<64>(a, stored, sm_count, s) : launch_group<128>(a, stored, sm_count, s);
}

}  // namespace shainet
