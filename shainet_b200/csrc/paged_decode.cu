// Attention of one new token per request over keys and values in pages, split over the requests' lengths and joined,
// sm_100a.
//
//   o = sum_j softmax_j(scale q . k_j) v_j  over the positions j < len,
//
// q and the new k row with bias, per-head RMSNorm and RoPE at position len - 1 first, the new k and v rows written into
// their page.  One launch, nothing of the batch known to the host but its size.
//
// Work.  Positions are cut into tiles of 8 KB of K and V; a request has ceil(len / TW) of them for each of its kv heads
// (and for each tile of query heads, where a group has more than one).  All tiles of the batch form one line, and every
// CTA takes an equal share of it: the lengths are read on the device, so balance does not depend on how ragged they are
// and a captured call follows them.  The start and the end of a (request, kv head) pair cost about as much as PAIR_COST
// tiles, so a pair stands on the line with that many places more.  A CTA walks the segments of its share; a segment that
// is a whole pair is written out directly, parts go to a workspace of two parts per CTA, and the CTA that finishes a
// pair's last part joins them in the order of the line, whichever CTA that is: results do not depend on timing, and
// no CTA waits for another.
//
// Streams.  Each of the four warps owns every fourth tile and a ring of its own in shared memory, filled by 16-byte
// asynchronous copies two tiles ahead and across segment borders; nothing waits for another warp but the start and the
// end of a segment.  Page numbers are fetched before the copies that need them.  HBM bounds it: two CTAs an SM keep
// 128 KB in flight each SM.
//
// Arithmetic.  Matrix units with fp32 accumulators, as on the CUDA cores the multiply-adds, and for 16-bit rows the
// widening, would take more issue slots than the rows take to arrive.
//  * 16-bit rows (m16n8k16): q and the softmax weights are fp32 and enter as three bfloat16 planes each, x = hi + mid + lo
//    exactly (24 bits cut into 8 + 8 + 8): no operand is rounded.  The planes lie side by side in the 16 rows of one
//    multiplication: four heads' three planes in one, eight heads' in two, sixteen heads' in three.
//  * fp32 rows (m16n8k8, TF32): every operand enters as two planes of 11 bits, hi + lo, so an operand keeps 22 of its 24
//    bits, rounded: of x in [1, 2) the upper plane leaves less than 2^-10, whose 11 bits end at 2^-21, so 2^-22 is lost at
//    most.  The sum of head_dim products of it is about as exact as the fp32 sum of a plain loop, whose own roundings are of
//    that size.  Eight heads' planes take one multiplication with each plane of the rows.  Sixteen heads take three, and
//    leave out the product of the two lower planes: 2^-20 of a product at most, 2^-23 on average.
// P.V of each tile starts from zero and is added to the running sum in fp32 with the rescaling, so that sums that the
// matrix units cut off stay one tile long.
//
// Measured.  64 ragged requests, 8 kv heads x 128, bfloat16, 2.2 GB of rows: 342 us, a copy's rate.  One request of 4097 positions: 11.0 us,
// a chain of latencies (lengths, table and rows 3.4, two tiles a warp 2.1, counting and joining 37 parts 3.5, launch 1).
// Sixteen heads a kv head: two thirds of a copy's rate, 96 multiplications of 8.5 cycles a tile, and parts of 8 KB to join
// (38 us for 73 MB).  Instructions that a CTA executes once arrive at five cycles each: with rolled loops instead of
// unrolled code in the join the kernel shrank from 107 to 67 KB and the request of 4097 positions from 15.0 to 11.0 us.
#include <cuda_bf16.h>
#include <math.h>
#include <algorithm>
#include <atomic>
#include "kernels.h"
#include "paged_index.h"

namespace shainet {

namespace {

constexpr unsigned FULL = 0xffffffffu;
constexpr float LOG2E = 1.4426950408889634f;
constexpr int NW = 4;                    // warps of a CTA
constexpr int THREADS = NW * 32;
constexpr int STAGES = 3;                // tiles of a warp's ring: two in flight, one in use
constexpr int STAGE_BYTES = 8192;        // K and V of one tile
constexpr int HALF = STAGE_BYTES / 2;
constexpr int MIN_TILES = 4;             // tiles a CTA takes at least, on average
constexpr int PAIR_COST = 8;             // places of the line that the start and end of a pair stand for
constexpr int CTAS_PER_SM = 2;
constexpr int LINE_PLACES = 1 << 30;        // places of the line: 8 TB of K and V, more than a device holds

// 16 bytes global -> shared
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// d += a b, or d = a b with FIRST
template <bool FIRST = false>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(FIRST ? 0.f : d[0]), "f"(FIRST ? 0.f : d[1]),
                   "f"(FIRST ? 0.f : d[2]), "f"(FIRST ? 0.f : d[3]));
}
template <bool FIRST = false>
__device__ __forceinline__ void mma1688(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(FIRST ? 0.f : d[0]), "f"(FIRST ? 0.f : d[1]),
                   "f"(FIRST ? 0.f : d[2]), "f"(FIRST ? 0.f : d[3]));
}

// An fp32 value as two TF32 planes: its upper 11 bits, and what is left rounded to 11 bits (the multiplication looks at
// the upper 19 bits of an operand register; half a step is added below them).
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
    hi = __float_as_uint(x) & 0xffffe000u;
    lo = __float_as_uint(x - __uint_as_float(hi)) + 0x1000u;
}

// Two fp32 values as three packed bfloat16 pairs, exactly: the upper halves, then the upper halves of what is left.
__device__ __forceinline__ void planes(float x0, float x1, uint32_t& hi, uint32_t& mid, uint32_t& lo) {
    const uint32_t u0 = __float_as_uint(x0), u1 = __float_as_uint(x1);
    hi = __byte_perm(u0, u1, 0x7632);
    const float r0 = x0 - __uint_as_float(u0 & 0xffff0000u), r1 = x1 - __uint_as_float(u1 & 0xffff0000u);
    const uint32_t v0 = __float_as_uint(r0), v1 = __float_as_uint(r1);
    mid = __byte_perm(v0, v1, 0x7632);
    const float s0 = r0 - __uint_as_float(v0 & 0xffff0000u), s1 = r1 - __uint_as_float(v1 & 0xffff0000u);
    lo = __byte_perm(__float_as_uint(s0), __float_as_uint(s1), 0x7632);
}

// HD: head_dim; ES: bytes per cache element; GT: query heads of a tile of heads, rounded up.
template <int HD_, int ES_, int GT_>
struct Cfg {
    static constexpr int HD = HD_, ES = ES_, GT = GT_;
    static constexpr int ROW = HD * ES;                  // bytes of a row
    static constexpr int CH = ROW / 16;                  // 16-byte pieces of a row
    static constexpr int TW = HALF / ROW;                // rows of a tile: 8, 16 or 32
    static constexpr int CPT = HALF / 16 / 32;           // pieces of K (and of V) a lane copies per tile
    static constexpr int QS = HD + 16;                   // floats between rotated q rows in shared memory: two rows, all banks
    static constexpr size_t RING = (size_t)NW * STAGES * STAGE_BYTES;
    static constexpr size_t SMEM = RING + (size_t)(GT * QS + 2 * HD + NW * GT * 2) * 4;
    static_assert(ES == 4 ? GT == 8 || GT == 16 : GT == 4 || GT == 8 || GT == 16, "heads of a tile");
    static_assert(GT * HD * 4 <= STAGE_BYTES, "a warp's sums are parked in a stage of its ring");
    static_assert(SMEM <= 113 * 1024, "two CTAs share an SM");
};

// Byte offset of piece c of row r inside a K or V tile.  The pieces of a row are permuted by its number so that a
// quarter-warp's 16-byte reads lie in different banks: 16-bit rows are read by ldmatrix, eight rows at one column; fp32
// rows four pieces of two neighbouring rows (K) and two pieces of four even or four odd rows (V) at a time.
template <class C>
__device__ __forceinline__ int tile_offset(int r, int c) {
    const int turn = C::ES == 2 ? r & 7 : ((r & 1) << 2) ^ (r & 6);
    return r * C::ROW + ((c ^ turn) << 4);
}

// A tile on the line.  Its pair stands at places [at, at + PAIR_COST + tiles), the tile at at + PAIR_COST + j.
struct Cursor {
    int b, hv, j;        // request, (kv head, tile of heads), tile of the request
    int tiles, len;      // of request b
    int at;
    __device__ __forceinline__ int place() const { return at + PAIR_COST + j; }
};

template <class C>
__device__ __forceinline__ int tiles_of(int len) { return (int)(((unsigned)len + C::TW - 1) / C::TW); }

// The first request with positions behind b, as (request, length); the number of requests where there is none.
__device__ __noinline__ int2 next_request(const int* lens, int b, int requests, int max_len) {
    while (++b < requests) {
        const int len = valid_len(lens[b], max_len);
        if (len != 0) return make_int2(b, len);
    }
    return make_int2(requests, 0);
}

// n tiles further; behind the last request the place is past every share.
template <class C>
__device__ __forceinline__ void advance(const PagedDecodeArgs& a, Cursor& c, int n) {
    c.j += n;
#pragma unroll 1
    while (c.j >= c.tiles) {
        c.j -= c.tiles;
        c.at += PAIR_COST + c.tiles;
        if (++c.hv == a.head_tiles * a.hs.num_kv_heads) {
            const int2 r = next_request(a.lens, c.b, a.requests, a.max_len);
            c.hv = 0;
            c.b = r.x;
            c.len = r.y;
            if (r.y == 0) {
                c.at = LINE_PLACES;
                c.j = 0;
                return;
            }
            c.tiles = tiles_of<C>(c.len);
        }
    }
}

// Lane r finds row r of a tile: the page of the position and the row in it, then the row of the pool (of one tensor, all
// kv heads counted: fits 32 bits).  Rows that are not there (behind the cached positions, or on a page that is not followed)
// are copied from the pool's first row: what stands there does not count.
struct Place {
    int page, row;
};
template <class C>
__device__ __forceinline__ Place lookup_page(const PagedDecodeArgs& a, const Cursor& c, int lane) {
    const int pos = c.j * C::TW + lane;
    Place p{0, -1};
    if (lane < C::TW && pos < c.len - 1) {               // the newest position comes from this call's inputs
        const int col = divide(pos, a.by_page);
        p.row = pos - col * a.page_rows;
        p.page = a.block_table[(size_t)c.b * a.table_width + col];
    }
    return p;
}
__device__ __forceinline__ unsigned row_of(const PagedDecodeArgs& a, int kv_h, Place p) {
    if (p.row < 0) return 0u;
    if (!page_in_pool(p.page, a.num_pages)) {
        report_bad_page(a.status, 14);
        return 0u;
    }
    return ((unsigned)p.page * a.hs.num_kv_heads + kv_h) * a.page_rows + p.row;
}

// kp, vp: the pools, at this lane's piece of a row
template <class C>
__device__ __forceinline__ void load_tile(const unsigned char* kp, const unsigned char* vp, unsigned row, uint32_t stage, int lane) {
    constexpr int RPI = 32 / C::CH;                      // rows of one warp-wide copy
    const int sub = lane / C::CH;
    const uint32_t to = stage + tile_offset<C>(sub, lane % C::CH);
#pragma unroll
    for (int i = 0; i < C::CPT; ++i) {
        const unsigned r = __shfl_sync(FULL, row, i * RPI + sub);
        const uint32_t dst = (to ^ (tile_offset<C>(i * RPI, 0) & 0x70)) + i * RPI * C::ROW;
        copy16(dst, kp + (size_t)r * C::ROW);
        copy16(dst + HALF, vp + (size_t)r * C::ROW);
    }
}

// The running sums of one warp over its tiles of one segment.  Lane (g = lane / 4, t = lane % 4) of a multiplication
// holds rows g and g + 8 of the 16 rows of heads and planes:
//   16-bit rows, GT = 4:  rows 0-3 hi, 4-7 mid, 8-11 lo of the four heads
//                GT = 8:  X: rows 0-7 hi, 8-15 mid;  Y: rows 0-7 lo
//                GT = 16: hi, mid and lo of the sixteen heads in three
//   fp32 rows,   GT = 8:  rows 0-7 hi, 8-15 lo
//                GT = 16: hi and lo in two; q stays in shared memory and is split for every tile (registers)
// and of the eight columns 2t and 2t + 1.  The order of the inner index is free as long as both operands share it: fp32
// rows of K are read four neighbouring columns at a time, rows of V in the order in which the weights lie in the lanes.
template <class C>
struct State {
    static constexpr int HD = C::HD, ES = C::ES, GT = C::GT;
    static constexpr int KS = HD / 16, N8 = HD / 8, NB = C::TW / 8;
    static constexpr bool Q_SHARED = ES == 4 && GT == 16;
    static constexpr int QR = ES == 2 ? (GT == 4 ? 4 : GT == 8 ? 6 : 12) : 8;     // q registers per 16 columns
    static constexpr int HL = GT == 16 ? 2 : 1;                                   // heads of a lane
    uint32_t q[Q_SHARED ? 1 : KS][QR];
    float o[N8][2 * HL];
    float m[HL], l[HL];       // maximum in units of log2

    __device__ __forceinline__ void start(const float* qs, int lane) {
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            if constexpr (ES == 4) {
                if constexpr (!Q_SHARED) {
                    const float4 x = *reinterpret_cast<const float4*>(qs + g * C::QS + s * 16 + 4 * t);
                    split_tf32(x.x, q[s][0], q[s][1]);
                    split_tf32(x.y, q[s][2], q[s][3]);
                    split_tf32(x.z, q[s][4], q[s][5]);
                    split_tf32(x.w, q[s][6], q[s][7]);
                }
            } else {
                const float* row = qs + (GT == 4 ? g & 3 : g) * C::QS + s * 16 + 2 * t;
                const float2 x = *reinterpret_cast<const float2*>(row), y = *reinterpret_cast<const float2*>(row + 8);
                uint32_t h0, m0, l0, h1, m1, l1;
                planes(x.x, x.y, h0, m0, l0);
                planes(y.x, y.y, h1, m1, l1);
                if constexpr (GT == 4) {
                    q[s][0] = g < 4 ? h0 : m0;
                    q[s][1] = g < 4 ? l0 : 0u;
                    q[s][2] = g < 4 ? h1 : m1;
                    q[s][3] = g < 4 ? l1 : 0u;
                } else if constexpr (GT == 8) {
                    q[s][0] = h0, q[s][1] = m0, q[s][2] = h1, q[s][3] = m1, q[s][4] = l0, q[s][5] = l1;
                } else {
                    const float2 z = *reinterpret_cast<const float2*>(row + 8 * C::QS), w = *reinterpret_cast<const float2*>(row + 8 * C::QS + 8);
                    uint32_t h2, m2, l2, h3, m3, l3;
                    planes(z.x, z.y, h2, m2, l2);
                    planes(w.x, w.y, h3, m3, l3);
                    q[s][0] = h0, q[s][1] = h2, q[s][2] = h1, q[s][3] = h3;
                    q[s][4] = m0, q[s][5] = m2, q[s][6] = m1, q[s][7] = m3;
                    q[s][8] = l0, q[s][9] = l2, q[s][10] = l1, q[s][11] = l3;
                }
            }
        }
#pragma unroll
        for (int n = 0; n < N8; ++n)
#pragma unroll
            for (int k = 0; k < 2 * HL; ++k) o[n][k] = 0.0f;
#pragma unroll
        for (int h = 0; h < HL; ++h) m[h] = -INFINITY, l[h] = 0.0f;
    }

    // s[n]: scores of rows 8n + 2t and 8n + 2t + 1, for head g and (GT = 16) head g + 8
    __device__ __forceinline__ void scores(const unsigned char* ks, const float* qs, float (&s)[NB][2 * HL], int lane) {
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            // c, d: the products with the upper and with the lower planes; two of each for fp32 rows, whose sums are longer
            float c[4] = {}, d[4] = {}, c1[4] = {};
            if constexpr (ES == 4) {
#pragma unroll
                for (int w = 0; w < KS; ++w) {
                    const float4 x = *reinterpret_cast<const float4*>(ks + tile_offset<C>(n * 8 + g, w * 4 + t));
                    const float xe[4] = {x.x, x.y, x.z, x.w};
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) split_tf32(xe[e], hi[e], lo[e]);
                    if constexpr (Q_SHARED) {
                        const float4 x0 = *reinterpret_cast<const float4*>(qs + g * C::QS + w * 16 + 4 * t);
                        const float4 x1 = *reinterpret_cast<const float4*>(qs + (g + 8) * C::QS + w * 16 + 4 * t);
                        const float qe[8] = {x0.x, x1.x, x0.y, x1.y, x0.z, x1.z, x0.w, x1.w};
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            uint32_t qh[4], ql[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) split_tf32(qe[4 * k + e], qh[e], ql[e]);
                            mma1688(k ? c1 : c, qh[0], qh[1], qh[2], qh[3], hi[2 * k], hi[2 * k + 1]);
                            mma1688(d, qh[0], qh[1], qh[2], qh[3], lo[2 * k], lo[2 * k + 1]);
                            mma1688(d, ql[0], ql[1], ql[2], ql[3], hi[2 * k], hi[2 * k + 1]);
                        }
                    } else {
                        const uint32_t(&a)[QR] = q[w];
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            mma1688(k ? c1 : c, a[4 * k], a[4 * k + 1], a[4 * k + 2], a[4 * k + 3], hi[2 * k], hi[2 * k + 1]);
                            mma1688(d, a[4 * k], a[4 * k + 1], a[4 * k + 2], a[4 * k + 3], lo[2 * k], lo[2 * k + 1]);
                        }
                    }
                }
            } else {
                const uint32_t at = smem_u32(ks);
                const int r = n * 8 + (lane & 7);
#pragma unroll
                for (int k2 = 0; k2 < KS; k2 += 2) {
                    uint32_t b[4];
                    ldsm4(b, at + tile_offset<C>(r, 2 * k2 + (lane >> 3)));
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const uint32_t(&a)[QR] = q[k2 + k];
                        mma16816(c, a[0], a[1], a[2], a[3], b[2 * k], b[2 * k + 1]);
                        if constexpr (GT == 8) mma16816(d, a[4], 0u, a[5], 0u, b[2 * k], b[2 * k + 1]);
                        if constexpr (GT == 16) {
                            mma16816(d, a[4], a[5], a[6], a[7], b[2 * k], b[2 * k + 1]);
                            mma16816(d, a[8], a[9], a[10], a[11], b[2 * k], b[2 * k + 1]);
                        }
                    }
                }
            }
            if constexpr (ES == 4) {
#pragma unroll
                for (int k = 0; k < 4; ++k) c[k] += c1[k];
            }
            if constexpr (GT == 16) {
#pragma unroll
                for (int k = 0; k < 4; ++k) s[n][k] = c[k] + d[k];
            } else {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    s[n][k] = (c[k] + d[k]) + (c[k + 2] + d[k + 2]);
                    if constexpr (GT == 4) s[n][k] += __shfl_xor_sync(FULL, s[n][k], 16);
                }
            }
        }
    }

    // o = o * alpha + P V of this tile
    __device__ __forceinline__ void values(const unsigned char* vs, const float (&s)[NB][2 * HL], const float (&alpha)[HL], int lane) {
        const int g = lane >> 2, t = lane & 3;
        auto add = [&](float(&to)[2 * HL], const float(&c)[4]) {
            if constexpr (GT == 16) {
#pragma unroll
                for (int x = 0; x < 4; ++x) to[x] = fmaf(to[x], alpha[x >> 1], c[x]);
            } else {
                to[0] = fmaf(to[0], alpha[0], c[0] + c[2]);
                to[1] = fmaf(to[1], alpha[0], c[1] + c[3]);
            }
        };
        if constexpr (ES == 4) {
            // the weights of rows 2t and 2t + 1 are at places t and t + 4 of the inner index; columns (8w + n) * 4 + e of V
            // form the eight columns n of multiplication 4w + e
            uint32_t ph[NB][2 * HL], pl[NB][2 * HL];
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
                for (int k = 0; k < 2 * HL; ++k) split_tf32(s[i][k], ph[i][k], pl[i][k]);
#pragma unroll
            for (int w = 0; w < HD / 32; ++w) {
                float c[4][4];
#pragma unroll
                for (int i = 0; i < NB; ++i) {
                    const float4 x = *reinterpret_cast<const float4*>(vs + tile_offset<C>(i * 8 + 2 * t, w * 8 + g));
                    const float4 y = *reinterpret_cast<const float4*>(vs + tile_offset<C>(i * 8 + 2 * t + 1, w * 8 + g));
                    const float xe[4] = {x.x, x.y, x.z, x.w}, ye[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        uint32_t h0, l0, h1, l1;
                        split_tf32(xe[e], h0, l0);
                        split_tf32(ye[e], h1, l1);
                        if constexpr (GT == 8) {
                            if (i == 0) mma1688<true>(c[e], ph[i][0], pl[i][0], ph[i][1], pl[i][1], l0, l1);
                            else mma1688(c[e], ph[i][0], pl[i][0], ph[i][1], pl[i][1], l0, l1);
                            mma1688(c[e], ph[i][0], pl[i][0], ph[i][1], pl[i][1], h0, h1);
                        } else {
                            if (i == 0) mma1688<true>(c[e], ph[i][0], ph[i][2], ph[i][1], ph[i][3], l0, l1);
                            else mma1688(c[e], ph[i][0], ph[i][2], ph[i][1], ph[i][3], l0, l1);
                            mma1688(c[e], pl[i][0], pl[i][2], pl[i][1], pl[i][3], h0, h1);
                            mma1688(c[e], ph[i][0], ph[i][2], ph[i][1], ph[i][3], h0, h1);
                        }
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) add(o[4 * w + e], c[e]);
            }
        } else {
            // the weights as operand rows: blocks 2i and 2i + 1 are the two halves of 16 rows of V
            uint32_t p[NB / 2][QR];
#pragma unroll
            for (int i = 0; i < NB / 2; ++i) {
                uint32_t h0, m0, l0, h1, m1, l1;
                planes(s[2 * i][0], s[2 * i][1], h0, m0, l0);
                planes(s[2 * i + 1][0], s[2 * i + 1][1], h1, m1, l1);
                if constexpr (GT == 4) {
                    const bool up = lane >= 16;
                    p[i][0] = up ? m0 : h0, p[i][1] = up ? 0u : l0, p[i][2] = up ? m1 : h1, p[i][3] = up ? 0u : l1;
                } else if constexpr (GT == 8) {
                    p[i][0] = h0, p[i][1] = m0, p[i][2] = h1, p[i][3] = m1, p[i][4] = l0, p[i][5] = l1;
                } else {
                    uint32_t h2, m2, l2, h3, m3, l3;
                    planes(s[2 * i][2], s[2 * i][3], h2, m2, l2);
                    planes(s[2 * i + 1][2], s[2 * i + 1][3], h3, m3, l3);
                    p[i][0] = h0, p[i][1] = h2, p[i][2] = h1, p[i][3] = h3;
                    p[i][4] = m0, p[i][5] = m2, p[i][6] = m1, p[i][7] = m3;
                    p[i][8] = l0, p[i][9] = l2, p[i][10] = l1, p[i][11] = l3;
                }
            }
            const uint32_t at = smem_u32(vs);
#pragma unroll
            for (int n = 0; n < N8; n += 2) {
                float c[2][4];
#pragma unroll
                for (int i = 0; i < NB / 2; ++i) {
                    uint32_t b[4];
                    ldsm4t(b, at + tile_offset<C>(i * 16 + (lane & 15), n + (lane >> 4)));
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        if (i == 0) mma16816<true>(c[k], p[i][0], p[i][1], p[i][2], p[i][3], b[2 * k], b[2 * k + 1]);
                        else mma16816(c[k], p[i][0], p[i][1], p[i][2], p[i][3], b[2 * k], b[2 * k + 1]);
                        if constexpr (GT == 8) mma16816(c[k], p[i][4], 0u, p[i][5], 0u, b[2 * k], b[2 * k + 1]);
                        if constexpr (GT == 16) {
                            mma16816(c[k], p[i][4], p[i][5], p[i][6], p[i][7], b[2 * k], b[2 * k + 1]);
                            mma16816(c[k], p[i][8], p[i][9], p[i][10], p[i][11], b[2 * k], b[2 * k + 1]);
                        }
                    }
                }
#pragma unroll
                for (int k = 0; k < 2; ++k) add(o[n + k], c[k]);
            }
        }
    }

    __device__ __forceinline__ void tile(const unsigned char* st, const float* qs, int nrows, float to2, int lane) {
        const int t = lane & 3;
        float s[NB][2 * HL], alpha[HL];
        scores(st, qs, s, lane);
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int k = 0; k < 2 * HL; ++k) s[n][k] *= to2;
        if (nrows < C::TW) {
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int k = 0; k < 2 * HL; ++k)
                    if (n * 8 + 2 * t + (k & 1) >= nrows) s[n][k] = -INFINITY;
        }
#pragma unroll
        for (int h = 0; h < HL; ++h) {
            float top = -INFINITY;
#pragma unroll
            for (int n = 0; n < NB; ++n) top = fmaxf(top, fmaxf(s[n][2 * h], s[n][2 * h + 1]));
            top = fmaxf(top, __shfl_xor_sync(FULL, top, 1));
            top = fmaxf(top, __shfl_xor_sync(FULL, top, 2));
            const float mn = fmaxf(m[h], top);
            alpha[h] = exp2f(m[h] - mn);
            m[h] = mn;
            float sum = 0.0f;
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    s[n][2 * h + k] = exp2f(s[n][2 * h + k] - mn);
                    sum += s[n][2 * h + k];
                }
            l[h] = fmaf(l[h], alpha[h], sum);
        }
        values(st + HALF, s, alpha, lane);
    }

    // sums to [GT][HD] floats, maxima and weight sums to ml [GT][2]
    __device__ __forceinline__ void park(float* to, float* ml, int lane) {
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int h = 0; h < HL; ++h) {
            l[h] += __shfl_xor_sync(FULL, l[h], 1);
            l[h] += __shfl_xor_sync(FULL, l[h], 2);
            if (t == 0 && g < GT) {
                ml[2 * (g + 8 * h)] = m[h];
                ml[2 * (g + 8 * h) + 1] = l[h];
            }
        }
        if constexpr (ES == 4) {
#pragma unroll
            for (int w = 0; w < HD / 32; ++w)
#pragma unroll
                for (int h = 0; h < HL; ++h)
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        *reinterpret_cast<float4*>(to + (g + 8 * h) * HD + (8 * w + 2 * t + k) * 4) =
                            make_float4(o[4 * w][2 * h + k], o[4 * w + 1][2 * h + k], o[4 * w + 2][2 * h + k], o[4 * w + 3][2 * h + k]);
        } else {
#pragma unroll
            for (int n = 0; n < N8; ++n)
#pragma unroll
                for (int h = 0; h < HL; ++h) {
                    float2 x = make_float2(o[n][2 * h], o[n][2 * h + 1]);
                    if constexpr (GT == 4) {
                        x.x += __shfl_xor_sync(FULL, x.x, 16);
                        x.y += __shfl_xor_sync(FULL, x.y, 16);
                    }
                    if (g < GT) *reinterpret_cast<float2*>(to + (g + 8 * h) * HD + n * 8 + 2 * t) = x;
                }
        }
    }
};

// The weight of a part with maximum m (scores times log2 e) under a maximum of all parts; 0 for a part that saw nothing.
__device__ __forceinline__ float part_weight(float m, float top) { return m == -INFINITY ? 0.0f : exp2f(m - top); }

// (one copy of each in the kernel: its code is long, and instructions that run once per call arrive at the pace of L2)
__device__ __noinline__ float2 angle(float position, float freq) {
    float2 r;
    sincosf(__fmul_rn(position, freq), &r.y, &r.x);
    return r;
}
__device__ __noinline__ float inverse_rms(float mean_square, double eps) { return (float)(1.0 / sqrt((double)mean_square + eps)); }

// What a segment works on.
struct Segment {
    int b, len, kv_h, head0, heads;
    bool owns_new, stores;     // it ends with the new position; it writes the new rows into their page
};

// The projections that a segment starts from: its q rows into qs and, where it ends with the new position, the new k and
// v rows into xk and xv, by asynchronous copies; then bias, norm and rotation in place, in the order and with the roundings
// of the other decode kernels, the new rows into their page too.  A warp takes every fourth row.
template <class C>
__device__ __forceinline__ void request_rows(const PagedDecodeArgs& a, const Segment& s, float* qs, float* xk, float* xv, int warp, int lane) {
    constexpr int HD = C::HD;
    const int items = s.heads + (s.owns_new ? 2 : 0);
#pragma unroll 1
    for (int it = warp; it < items; it += NW) {
        const bool is_q = it < s.heads, is_k = it == s.heads;
        const float* src = is_q ? a.q + ((size_t)s.b * a.hs.num_heads + s.head0 + it) * HD : (is_k ? a.k_new : a.v_new) + ((size_t)s.b * a.hs.num_kv_heads + s.kv_h) * HD;
        float* to = is_q ? qs + it * C::QS : is_k ? xk : xv;
        if (lane < HD / 4) copy16(smem_u32(to + lane * 4), src + lane * 4);
    }
}
template <class C>
__device__ __forceinline__ void prepare_rows(const PagedDecodeArgs& a, const Segment& s, float* qs, float* xk, float* xv, int warp, int lane) {
    constexpr int HD = C::HD, PL = HD / 64;
    const int pos = s.len - 1, items = s.heads + (s.owns_new ? 2 : 0);
    float2 turn[PL];
#pragma unroll
    for (int k = 0; k < PL; ++k) turn[k] = angle((float)pos, __ldg(a.inv_freq + lane + 32 * k));
    size_t at = 0;
    bool stores = s.owns_new && s.stores;
    if (stores) {
        const int col = divide(pos, a.by_page), page = a.block_table[(size_t)s.b * a.table_width + col];
        stores = page_in_pool(page, a.num_pages);
        if (stores) at = pool_row(page, a.hs.num_kv_heads, s.kv_h, a.page_rows, pos - col * a.page_rows) * HD;
        else if (warp == 0 && lane == 0) report_bad_page(a.status, 15);
    }
#pragma unroll 1
    for (int it = warp; it < items; it += NW) {      // the rows this warp requested
        const bool is_q = it < s.heads, is_k = it == s.heads;
        float* row = is_q ? qs + it * C::QS : is_k ? xk : xv;
        const float* bias = is_q ? a.b_q : is_k ? a.b_k : a.b_v;
        const float* w = is_q ? a.q_norm : is_k ? a.k_norm : nullptr;
        float x[2 * PL];
#pragma unroll
        for (int c = 0; c < 2 * PL; ++c) x[c] = row[lane + 32 * c];
        if (bias) {
            bias += (size_t)(is_q ? s.head0 + it : s.kv_h) * HD;
#pragma unroll
            for (int c = 0; c < 2 * PL; ++c) x[c] = __fadd_rn(x[c], __ldg(bias + lane + 32 * c));
        }
        if (w) {
            float ss = 0.0f;
#pragma unroll
            for (int c = 0; c < 2 * PL; ++c) ss = fmaf(x[c], x[c], ss);
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) ss += __shfl_xor_sync(FULL, ss, off);
            const float inv = inverse_rms(ss / (float)HD, a.eps);
#pragma unroll
            for (int c = 0; c < 2 * PL; ++c) x[c] = __fmul_rn(__fmul_rn(x[c], inv), __ldg(w + lane + 32 * c));
        }
        if (is_q || is_k) {
#pragma unroll
            for (int k = 0; k < PL; ++k) {
                const float x0 = x[k], x1 = x[k + PL];
                x[k] = __fsub_rn(__fmul_rn(x0, turn[k].x), __fmul_rn(x1, turn[k].y));
                x[k + PL] = __fadd_rn(__fmul_rn(x1, turn[k].x), __fmul_rn(x0, turn[k].y));
            }
        }
#pragma unroll
        for (int c = 0; c < 2 * PL; ++c) row[lane + 32 * c] = x[c];
        if (!is_q && stores) {
            void* dst = is_k ? a.k_pages : a.v_pages;
#pragma unroll
            for (int c = 0; c < 2 * PL; ++c) {
                if constexpr (C::ES == 4) static_cast<float*>(dst)[at + lane + 32 * c] = x[c];
                else static_cast<__nv_bfloat16*>(dst)[at + lane + 32 * c] = __float2bfloat16_rn(x[c]);
            }
        }
    }
#pragma unroll 1
    for (int it = s.heads + warp; it < C::GT; it += NW)      // heads that fill up the tile
#pragma unroll
        for (int c = 0; c < 2 * PL; ++c) qs[it * C::QS + lane + 32 * c] = 0.0f;
}

// The last tile of a request: the new k and v rows, as the pages hold them, into row r; v rows behind it are zeros (their
// weights are, but what was copied there may not be finite).
template <class C>
__device__ __forceinline__ void patch_tile(unsigned char* st, int r, const float* xk, const float* xv, int lane) {
#pragma unroll
    for (int c = 0; c < C::HD / 32; ++c) {
        const int d = lane + 32 * c, at = tile_offset<C>(r, d * C::ES / 16) + d * C::ES % 16;
        if constexpr (C::ES == 4) {
            *reinterpret_cast<float*>(st + at) = xk[d];
            *reinterpret_cast<float*>(st + HALF + at) = xv[d];
        } else {
            *reinterpret_cast<__nv_bfloat16*>(st + at) = __float2bfloat16_rn(xk[d]);
            *reinterpret_cast<__nv_bfloat16*>(st + HALF + at) = __float2bfloat16_rn(xv[d]);
        }
    }
#pragma unroll 1
    for (int i = (r + 1) * C::CH + lane; i < C::TW * C::CH; i += 32) *reinterpret_cast<uint4*>(st + HALF + i * 16) = make_uint4(0u, 0u, 0u, 0u);
    __syncwarp();
}

// A pair that several CTAs share: the parts of CTAs c0 .. c0 + n - 1.  A CTA has two places for parts: of a pair that
// began before it (0) and of one that begins in it (1).
struct Shared {
    int c0, n, fan, heads;     // fan: parts that are joined at once
    bool mine;                 // this CTA joins
    float* out;
};

// Parts added from the workspace: staged in the rings by asynchronous copies, all requested before the first is waited
// for, then four columns of TPT heads a thread; where the heads leave threads over, up to four threads share a column's
// parts.  Loops and not unrolled code: a CTA works alone here, once a call, and cold instructions arrive more slowly than
// they are executed.
template <class C>
struct Join {
    static constexpr int HD = C::HD, GT = C::GT, TPT = (GT * HD / 4 + THREADS - 1) / THREADS, HPW = GT / NW;
    static constexpr int MOST = 64;                          // parts of one call; a lane brings the maxima of two a head
    static constexpr int META = GT * 8 + MOST * GT * 4;      // bytes: sums, then weights [part][head]
    static constexpr int SHARES = THREADS * 16;
    float4 acc[TPT];

    __device__ __forceinline__ static int groups_of(int heads) {
        const int tasks = heads * (HD / 4);
        return tasks <= THREADS / 4 ? 4 : tasks <= THREADS / 2 ? 2 : 1;
    }
    // All parts at once where they fit; more in groups of about the root of their number, each by its last CTA into a second
    // table, then the groups.
    __device__ __forceinline__ static int fan_of(int n, int heads) {
        return n <= MOST && n * heads * HD * 4 <= (int)C::RING - META - SHARES ? n : (int)ceilf(sqrtf((float)n));
    }
    static_assert(GT % NW == 0, "a warp weighs the parts of every fourth head");

    __device__ __forceinline__ static float2* sums(unsigned char* smem) { return reinterpret_cast<float2*>(smem); }

    // n parts at places at0, at0 + step, ...; the first one place further where `odd`.  Maxima and weight sums in sums().
    __device__ __forceinline__ void run(const float* po, const float2* pml, int at0, int step, int n, int odd, int heads, unsigned char* smem, int tid) {
        const int warp = tid >> 5, lane = tid & 31;
        const int tasks = heads * (HD / 4), groups = groups_of(heads), wide = THREADS / groups, sub = tid / wide, e0 = tid - sub * wide;
        float2* total = sums(smem);
        float* weight = reinterpret_cast<float*>(total + GT);
        float4* share = reinterpret_cast<float4*>(smem + META);
        unsigned char* stage = smem + META + SHARES;
        const int room = ((int)C::RING - META - SHARES) / (tasks * 16);
        float2 ml[HPW][2];
#pragma unroll
        for (int x = 0; x < HPW; ++x)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int g = warp + x * NW, i = lane + 32 * k;
                ml[x][k] = make_float2(-INFINITY, 0.f);
                if (g < heads && i < n) ml[x][k] = __ldcg(pml + (at0 + i * step + (i == 0 ? odd : 0)) * GT + g);
            }
        auto request = [&](int i0, int cnt) {
            const float* src = po + (size_t)((at0 + (i0 + sub) * step) * (GT * HD)) + e0 * 4;
            uint32_t to = smem_u32(stage) + (sub * tasks + e0) * 16;
            int skip = i0 + sub == 0 ? odd * (GT * HD) : 0;
#pragma unroll 1
            for (int i = sub; i < cnt; i += groups) {
#pragma unroll
                for (int x = 0; x < TPT; ++x)
                    if (e0 + x * THREADS < tasks) copy16(to + x * (THREADS * 16), src + skip + x * (THREADS * 4));
                skip = 0;
                src += groups * step * (GT * HD);
                to += groups * tasks * 16;
            }
            copy_commit();
        };
        int cnt = min(n, room);
        request(0, cnt);
#pragma unroll
        for (int x = 0; x < HPW; ++x) {
            const int g = warp + x * NW;
            float top = fmaxf(ml[x][0].x, ml[x][1].x);
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(FULL, top, off));
            const float w0 = part_weight(ml[x][0].x, top), w1 = part_weight(ml[x][1].x, top);
            float L = fmaf(w0, ml[x][0].y, w1 * ml[x][1].y);
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) L += __shfl_xor_sync(FULL, L, off);
            if (g < heads) {
                if (lane < n) weight[lane * heads + g] = w0;
                if (lane + 32 < n) weight[(lane + 32) * heads + g] = w1;
                if (lane == 0) total[g] = make_float2(top, L);
            }
        }
#pragma unroll
        for (int x = 0; x < TPT; ++x) acc[x] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
        for (int i0 = 0;;) {
            copy_wait<0>();
            __syncthreads();
#pragma unroll
            for (int x = 0; x < TPT; ++x) {
                const int e = e0 + x * THREADS;
                if (e < tasks) {
                    const float* w = weight + (i0 + sub) * heads + e / (HD / 4);
                    const float4* v = reinterpret_cast<const float4*>(stage) + sub * tasks + e;
#pragma unroll 4
                    for (int i = sub; i < cnt; i += groups) {
                        const float wt = *w;
                        const float4 y = *v;
                        acc[x].x = fmaf(wt, y.x, acc[x].x);
                        acc[x].y = fmaf(wt, y.y, acc[x].y);
                        acc[x].z = fmaf(wt, y.z, acc[x].z);
                        acc[x].w = fmaf(wt, y.w, acc[x].w);
                        w += groups * heads;
                        v += groups * tasks;
                    }
                }
            }
            i0 += cnt;
            if (i0 >= n) break;
            __syncthreads();
            cnt = min(n - i0, room);
            request(i0, cnt);
        }
        if (groups > 1) {        // one task a thread
            share[tid] = acc[0];
            __syncthreads();
            if (sub == 0)
#pragma unroll 1
                for (int k = 1; k < groups; ++k) {
                    const float4 o = share[tid + k * wide];
                    acc[0].x += o.x, acc[0].y += o.y, acc[0].z += o.z, acc[0].w += o.w;
                }
        }
    }
    __device__ __forceinline__ void store(float* po, float2* pml, int at, int heads, unsigned char* smem, int tid) {
#pragma unroll
        for (int x = 0; x < TPT; ++x) {
            const int e = tid + x * THREADS;
            if (e < heads * (HD / 4)) *(reinterpret_cast<float4*>(po) + at * (GT * HD / 4) + e) = acc[x];
        }
        if (tid < heads) pml[at * GT + tid] = sums(smem)[tid];
    }
    __device__ __forceinline__ void finish(float* out, int heads, unsigned char* smem, int tid) {
#pragma unroll
        for (int x = 0; x < TPT; ++x) {
            const int e = tid + x * THREADS;
            if (e < heads * (HD / 4)) {
                const float inv = 1.0f / sums(smem)[e / (HD / 4)].y;
                *reinterpret_cast<float4*>(out + e * 4) = make_float4(acc[x].x * inv, acc[x].y * inv, acc[x].z * inv, acc[x].w * inv);
            }
        }
    }
};

template <class C>
__global__ void __launch_bounds__(THREADS, CTAS_PER_SM) paged_decode_kernel(PagedDecodeArgs a) {
    constexpr int HD = C::HD, GT = C::GT, EACH = 4;
    extern __shared__ __align__(1024) unsigned char pd_smem[];
    float* qs = reinterpret_cast<float*>(pd_smem + C::RING);
    float* xk = qs + GT * C::QS;
    float* xv = xk + HD;
    float* wml = xv + HD;                                          // [NW][GT][2]
    __shared__ int s_last, s_park[NW];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int H = a.hs.num_heads, KV = a.hs.num_kv_heads, G = H / KV;
    const int HV = KV * a.head_tiles, per = (G + a.head_tiles - 1) / a.head_tiles;
    unsigned char* ring = pd_smem + (size_t)warp * STAGES * STAGE_BYTES;

    // Everything this kernel reads may come from the kernel ahead in the stream.  The next one may start its own launch
    // now: it waits for this one's end before it touches anything, as this one has waited.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    // ---- the line: its length, then the request in which this CTA's share starts.  Every warp for itself, 128 requests
    // at a time, EACH a lane ----
    int lens[EACH];
    auto places = [&](int len) { return len > 0 ? (tiles_of<C>(len) + PAIR_COST) * HV : 0; };
    auto scan = [&](int b0, int& upto) {             // places of this lane's requests and all before them
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int b = b0 + lane * EACH + i;
            lens[i] = b < a.requests ? valid_len(a.lens[b], a.max_len) : 0;
        }
        upto = 0;
#pragma unroll
        for (int i = 0; i < EACH; ++i) upto += places(lens[i]);
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int up = __shfl_up_sync(FULL, upto, off);
            if (lane >= off) upto += up;
        }
        return __shfl_sync(FULL, upto, 31);
    };
    int total = 0, upto = 0, live = 0;
    float size = 0.0f;                               // of the line, in numbers that cannot overflow
#pragma unroll 1
    for (int b0 = 0; b0 < a.requests; b0 += 32 * EACH) {
        total += scan(b0, upto);
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            live += __popc(__ballot_sync(FULL, lens[i] > 0));
            size += (float)lens[i];
        }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) size += __shfl_xor_sync(FULL, size, off);
    const bool too_long = (size / C::TW + (PAIR_COST + 2) * (float)live) * HV > 0.99f * LINE_PLACES;
    const int pairs = live * HV, tiles = total - pairs * PAIR_COST;
    const int ctas = min((int)gridDim.x, max(1, max(pairs, tiles / MIN_TILES)));
    const int cta = blockIdx.x;
    // equal shares, the first `rest` of them a place longer
    const int each = total / ctas, rest = total - each * ctas;
    auto share = [&](int c) { return c * each + min(c, rest); };
    auto owner = [&](int place) {
        const int longer = rest * (each + 1);
        return place < longer ? place / (each + 1) : rest + (place - longer) / each;
    };

    // padded rows, and lengths that do not fit: zeros
#pragma unroll 1
    for (int b = cta; b < a.requests; b += gridDim.x) {
        const int len = a.lens[b];
        if (valid_len(len, a.max_len) > 0 && !too_long) continue;
        if (len != 0 && tid == 0) report_bad_page(a.status, 13);
#pragma unroll 1
        for (int d = tid; d < H * HD / 4; d += THREADS) reinterpret_cast<float4*>(a.out)[(size_t)b * (H * HD / 4) + d] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    if (cta >= ctas || total == 0 || too_long) return;
    const int s0 = share(cta), s1 = share(cta + 1);

    Cursor seg{};    // the first tile of this share
    {
        int base = 0;
#pragma unroll 1
        for (int b0 = 0; b0 < a.requests; b0 += 32 * EACH) {
            const int all = a.requests <= 32 * EACH ? total : scan(b0, upto);
            if (s0 < base + all) {
                const int at = __ffs(__ballot_sync(FULL, base + upto > s0)) - 1;      // the lane that holds the request
                int from = base + upto, b = 0, len = 0, first = 0;
#pragma unroll
                for (int i = 0; i < EACH; ++i) from -= places(lens[i]);
#pragma unroll
                for (int i = 0; i < EACH; ++i) {
                    if (lens[i] > 0 && from <= s0) b = b0 + lane * EACH + i, len = lens[i], first = from;
                    from += places(lens[i]);
                }
                seg.b = __shfl_sync(FULL, b, at);
                seg.len = __shfl_sync(FULL, len, at);
                seg.at = __shfl_sync(FULL, first, at);
                break;
            }
            base += all;
        }
    }
    seg.tiles = tiles_of<C>(seg.len);
    seg.hv = (s0 - seg.at) / (seg.tiles + PAIR_COST);
    seg.at += seg.hv * (seg.tiles + PAIR_COST);
    seg.j = max(0, s0 - seg.at - PAIR_COST);
    if (seg.place() >= s1) return;                   // the share lies before the pair's first tile

    auto seg_head = [&](const Cursor& c) { return divide(c.hv, a.by_tiles); };
    // Segment of the pair at the cursor, up to jend
    auto segment_of = [&](const Cursor& c, int& jend) {
        jend = min(c.tiles, s1 - c.at - PAIR_COST);
        Segment s;
        s.b = c.b;
        s.len = c.len;
        s.kv_h = seg_head(c);
        const int ht = c.hv - s.kv_h * a.head_tiles;
        s.head0 = s.kv_h * G + ht * per;
        s.heads = min(per, G - ht * per);
        s.owns_new = jend == c.tiles;
        s.stores = ht == 0;
        return s;
    };

    // ---- this warp's copies: the share's tiles warp, warp + NW, ...; page numbers two tiles ahead ----
    Cursor ld = seg;
    if (warp > 0) advance<C>(a, ld, warp);
    Cursor ahead = ld;
    Place place0{-1, -1}, place1{-1, -1};
    if (ahead.place() < s1) {
        place0 = lookup_page<C>(a, ahead, lane);
        advance<C>(a, ahead, NW);
        if (ahead.place() < s1) place1 = lookup_page<C>(a, ahead, lane);
    }
    int ld_head = seg_head(ld);
    int ld_place = ld.place();
    const unsigned char* kp = static_cast<const unsigned char*>(a.k_pages) + lane % C::CH * 16;
    const unsigned char* vp = static_cast<const unsigned char*>(a.v_pages) + lane % C::CH * 16;
    const uint32_t ring_at = smem_u32(ring);
    uint32_t fill = 0, take = 0;                     // byte offsets in the ring: the next tile's, the next that is used
    auto fetch = [&]() {                             // one group of copies, empty behind the last tile
        if (ld_place < s1) {
            load_tile<C>(kp, vp, row_of(a, ld_head, place0), ring_at + fill, lane);
            fill = fill == (STAGES - 1) * STAGE_BYTES ? 0 : fill + STAGE_BYTES;
            ld_place = ahead.place();
            ld_head = seg_head(ahead);
            place0 = place1;
            if (ld_place < s1) {
                advance<C>(a, ahead, NW);
                if (ahead.place() < s1) place1 = lookup_page<C>(a, ahead, lane);
            }
        }
        copy_commit();
    };

    int jend;
    Segment sg = segment_of(seg, jend);
    request_rows<C>(a, sg, qs, xk, xv, warp, lane);
    copy_commit();
#pragma unroll 1
    for (int i = 0; i < STAGES - 1; ++i) fetch();
    copy_wait<STAGES - 1>();          // the rows

    State<C> st;
    const float to2 = a.scale * LOG2E;
    int done = 0;                                    // tiles of the share in the segments before
    Shared pend[2];                                  // the pairs this CTA shares: its first segment's and its last one's
    pend[0].mine = pend[1].mine = false;
    // Parts are counted when they are complete: the CTA's barrier, then one acquire-release addition.  True for the CTA that
    // counts the last of n.
    auto last_of = [&](unsigned* counter, int n) {
        __syncthreads();
        if (tid == 0) {
            unsigned before;
            asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
            s_last = before == (unsigned)(n - 1);
            if (s_last) *counter = 0u;
        }
        __syncthreads();
        return s_last != 0;
    };
#pragma unroll 1
    while (true) {
        __syncwarp();
        prepare_rows<C>(a, sg, qs, xk, xv, warp, lane);
        __syncthreads();
        st.start(qs, lane);
#pragma unroll 1
        for (int j = seg.j + ((warp - done) & (NW - 1)); j < jend; j += NW) {     // this warp's tiles
            copy_wait<STAGES - 2>();
            __syncwarp();
            unsigned char* stage = ring + take;
            const int nrows = min(C::TW, seg.len - j * C::TW);
            if (j == seg.tiles - 1) patch_tile<C>(stage, nrows - 1, xk, xv, lane);
            fetch();
            st.tile(stage, qs, nrows, to2, lane);
            __syncwarp();
            take = take == (STAGES - 1) * STAGE_BYTES ? 0 : take + STAGE_BYTES;
        }
        // the stage that was used last is not filled again before the next tile: the sums wait there to be joined
        const uint32_t parked = take == 0 ? (STAGES - 1) * STAGE_BYTES : take - STAGE_BYTES;
        st.park(reinterpret_cast<float*>(ring + parked), wml + warp * GT * 2, lane);
        if (lane == 0) s_park[warp] = warp * STAGES * STAGE_BYTES + (int)parked;

        const Segment cur = sg;
        const int j0 = seg.j, jn = jend, whole = seg.tiles;
        const int pair_at = seg.at;
        done += jn - j0;
        advance<C>(a, seg, jn - j0);
        const bool more = jn == whole && seg.place() < s1;
        __syncthreads();
        if (more) {
            sg = segment_of(seg, jend);
            request_rows<C>(a, sg, qs, xk, xv, warp, lane);      // arrive while the sums are joined
            copy_commit();
        }

        // ---- the four warps' sums, to the output or to the workspace ----
        const bool complete = j0 == 0 && jn == whole;
        const size_t part = (size_t)cta * 2 + (j0 == 0 ? 1 : 0);
        float* out = a.out + ((size_t)cur.b * H + cur.head0) * HD;
        const int tasks = cur.heads * (HD / 4);      // four columns of a head
#pragma unroll 1
        for (int e = tid; e < tasks; e += THREADS) {
            const int g = e / (HD / 4), d = (e - g * (HD / 4)) * 4;
            float top = -INFINITY, L = 0.0f;
#pragma unroll
            for (int w = 0; w < NW; ++w) top = fmaxf(top, wml[(w * GT + g) * 2]);
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const float wt = part_weight(wml[(w * GT + g) * 2], top);
                const float4 v = *reinterpret_cast<const float4*>(pd_smem + s_park[w] + e * 16);
                L = fmaf(wt, wml[(w * GT + g) * 2 + 1], L);
                acc.x = fmaf(wt, v.x, acc.x);
                acc.y = fmaf(wt, v.y, acc.y);
                acc.z = fmaf(wt, v.z, acc.z);
                acc.w = fmaf(wt, v.w, acc.w);
            }
            if (complete) {
                const float inv = 1.0f / L;
                *reinterpret_cast<float4*>(out + e * 4) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
            } else {
                *reinterpret_cast<float4*>(a.part_o + part * GT * HD + e * 4) = acc;
                if (d == 0) *reinterpret_cast<float2*>(a.part_ml + (part * GT + g) * 2) = make_float2(top, L);
            }
        }
        if (!complete) {
            Shared p;
            p.c0 = owner(pair_at + PAIR_COST);
            p.n = owner(pair_at + PAIR_COST + whole - 1) - p.c0 + 1;
            p.fan = Join<C>::fan_of(p.n, cur.heads);
            p.heads = cur.heads;
            p.out = out;
            // The groups' counters: a group may begin with the CTA in which another pair begins.
            const int g0 = p.c0 + (cta - p.c0) / p.fan * p.fan;
            p.mine = last_of(p.n <= p.fan ? a.counters + p.c0 : a.counters + gridDim.x + 2 * g0 + (g0 == p.c0 ? 1 : 0),
                             min(p.fan, p.c0 + p.n - g0));
            pend[j0 == 0 ? 1 : 0] = p;
        }
        if (!more) break;
        copy_wait<0>();
        __syncthreads();      // the parked sums have been read
    }
    copy_wait<0>();
    __syncthreads();

    // ---- the pairs whose last part was this CTA's; the rings are free now ----
#pragma unroll 1
    for (int i = 0; i < 2; ++i) {
        const Shared p = pend[i];
        if (!p.mine) continue;
        __syncthreads();
        Join<C> join;
        float2* ml = reinterpret_cast<float2*>(a.part_ml);
        const int g0 = p.c0 + (cta - p.c0) / p.fan * p.fan;
        int at = 2 * g0, step = 2, n = min(p.fan, p.c0 + p.n - g0), odd = g0 == p.c0 ? 1 : 0;
        bool last = true;
#pragma unroll 1
        while (true) {
            join.run(a.part_o, ml, at, step, n, odd, p.heads, pd_smem, tid);
            if (p.n <= p.fan || step == 1) break;
            // the second table lies behind the parts; a pair's groups take the places of its first CTAs there
            const int second = 2 * gridDim.x + p.c0;
            n = (p.n + p.fan - 1) / p.fan;
            join.store(a.part_o, ml, second + (g0 - p.c0) / p.fan, p.heads, pd_smem, tid);
            last = last_of(a.counters + p.c0, n);
            if (!last) break;
            at = second, step = 1, odd = 0;
        }
        if (!last) continue;
        join.finish(p.out, p.heads, pd_smem, tid);
    }
}

template <int HD, int ES, int GT>
cudaError_t launch(const PagedDecodeArgs& a, int ctas, cudaStream_t s) {
    using C = Cfg<HD, ES, GT>;
    static std::atomic<unsigned long long> configured{0};   // bit per device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !(configured.load(std::memory_order_acquire) >> dev & 1ull)) {
        e = cudaFuncSetAttribute(paged_decode_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::SMEM);
        if (e != cudaSuccess) return e;
        if (dev < 64) configured.fetch_or(1ull << dev, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, paged_decode_kernel<C>, a);
}

template <int HD, int ES>
cudaError_t launch_heads(const PagedDecodeArgs& a, int gt, int ctas, cudaStream_t s) {
    if constexpr (ES == 2)
        if (gt == 4) return launch<HD, ES, 4>(a, ctas, s);
    if (gt == 8) return launch<HD, ES, 8>(a, ctas, s);
    return launch<HD, ES, 16>(a, ctas, s);
}

}  // namespace

PagedPlan paged_decode_plan(const HeadShape& hs, int kv_elem_bytes, int sm_count) {
    const int G = hs.num_heads / hs.num_kv_heads, most = 16;
    PagedPlan p;
    p.head_tiles = (G + most - 1) / most;
    const int per = (G + p.head_tiles - 1) / p.head_tiles;
    p.gt = kv_elem_bytes == 4 ? 8 : 4;
    while (p.gt < per) p.gt *= 2;
    p.ctas = sm_count * CTAS_PER_SM;
    p.part_floats = (size_t)p.ctas * 3 * p.gt * (hs.head_dim + 2);
    return p;
}

cudaError_t launch_paged_decode(PagedDecodeArgs a, const PagedPlan& p, float* workspace, unsigned* counters, cudaStream_t s) {
    a.max_len = max_len_of(a.table_width, a.page_rows);
    a.by_page = fast_div(a.page_rows);
    a.by_tiles = fast_div(p.head_tiles);
    a.head_tiles = p.head_tiles;
    a.part_o = workspace;
    a.part_ml = workspace + (size_t)p.ctas * 3 * p.gt * a.hs.head_dim;
    a.counters = counters;
    const long long most = (long long)a.table_width * a.page_rows * a.hs.num_kv_heads * p.head_tiles;   // tiles, at one row each
    const int ctas = (int)std::min<long long>(p.ctas, std::max<long long>(1, std::min<long long>(most, 0x7fffffff) * a.requests));
    if (a.hs.head_dim == 128) return a.kv_elem_bytes == 4 ? launch_heads<128, 4>(a, p.gt, ctas, s) : launch_heads<128, 2>(a, p.gt, ctas, s);
    return a.kv_elem_bytes == 4 ? launch_heads<64, 4>(a, p.gt, ctas, s) : launch_heads<64, 2>(a, p.gt, ctas, s);
}

}  // namespace shainet
