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
// and a captured call follows them.  A CTA walks the segments of its share; a segment that is a whole (request, kv head)
// is written out directly, parts go to a workspace of two parts per CTA, and the CTA that finishes a pair's last part
// joins them in the order of the line, whichever CTA that is: results do not depend on timing.
//
// Streams.  Each of the four warps owns every fourth tile and a ring of its own in shared memory, filled by 16-byte
// asynchronous copies two tiles ahead and across segment borders; nothing waits for another warp but the start and the
// end of a segment.  Page numbers are fetched one tile before they are needed.  HBM bounds it: two CTAs an SM keep
// 128 KB in flight each SM.
//
// Arithmetic.  fp32 rows: sixteen lanes to a k row, packed fp32 multiply-adds, scores summed over the lanes by halving
// exchanges.  16-bit rows: the matrix units (m16n8k16, fp32 accumulators), where the CUDA cores would need more issue
// slots than the rows take to arrive (eight heads a group: 256 multiply-adds per 2 bytes of K and V).  q and the softmax
// weights are fp32 and enter as three bfloat16 planes each, x = hi + mid + lo exactly (24 bits cut into 8 + 8 + 8), so
// no operand is rounded.  The planes lie side by side in the 16 rows of one multiplication: four heads' three planes
// in one, eight heads' in two, sixteen in three.  P.V of each tile starts from zero and is added to the running sum in
// fp32 with the rescaling, so that the matrix units' cut-off sums stay one tile long.
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
constexpr int MIN_TILES = 4;             // tiles a CTA takes at least
constexpr int CTAS_PER_SM = 2;

typedef unsigned long long f32x2;

__device__ __forceinline__ f32x2 pack2(float lo, float hi) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void unpack2(f32x2 v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ f32x2 ffma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ f32x2 fmul2(f32x2 a, f32x2 b) {
    f32x2 d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// 16 bytes global -> shared, zeros where !valid (nothing is read then).
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool valid) {
    const int n = valid ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
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
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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
    static constexpr int QS = HD + 4;                    // floats between rotated q rows in shared memory
    // fp32 rows: R rows of a half-warp give R * GT scores, at most 16, summed over its lanes
    static constexpr int R = (16 / (GT > 16 ? 16 : GT)) < TW / 2 ? 16 / (GT > 16 ? 16 : GT) : TW / 2;
    static constexpr int NS = R * GT;
    static constexpr int BR = 2 * R;
    static constexpr int PS = 2 * R * GT + GT;           // packed pairs of a warp: weights of a batch, rescaling factors
    static constexpr size_t RING = (size_t)NW * STAGES * STAGE_BYTES;
    static constexpr size_t SMEM = RING + (size_t)(GT * QS + 2 * HD + NW * GT * 2) * 4 + (ES == 4 ? (size_t)NW * PS * 8 : 0);
    static_assert(GT * HD * 4 <= STAGE_BYTES, "a warp's sums are parked in a stage of its ring");
    static_assert(SMEM <= 113 * 1024, "two CTAs share an SM");
};

// Byte offset of piece c of row r inside a K or V tile.  16-bit rows are read by ldmatrix, eight rows at one column: the
// pieces of a row are permuted by its number so that the eight lie in different banks.
template <class C>
__device__ __forceinline__ int tile_offset(int r, int c) {
    return r * C::ROW + ((C::ES == 2 ? c ^ (r & 7) : c) << 4);
}

// A place on the line of tiles.
struct Cursor {
    int b, hv, j;        // request, (kv head, tile of heads), tile of the request
    int tiles, len;      // of request b
};

template <class C>
__device__ __forceinline__ int valid_len(const PagedDecodeArgs& a, int b) {
    const int len = a.lens[b];
    return length_fits(len, a.table_width, a.page_rows) ? len : 0;
}
template <class C>
__device__ __forceinline__ int tiles_of(int len) { return (int)(((long long)len + C::TW - 1) / C::TW); }

// The next request with positions at or behind b (there is one).
template <class C>
__device__ __forceinline__ void enter_request(const PagedDecodeArgs& a, Cursor& c) {
    while (c.b < a.requests) {
        c.len = valid_len<C>(a, c.b);
        if (c.len > 0) break;
        ++c.b;
    }
    c.tiles = tiles_of<C>(c.len);
}
template <class C>
__device__ __forceinline__ void advance(const PagedDecodeArgs& a, Cursor& c, int n) {
    c.j += n;
    while (c.j >= c.tiles) {
        c.j -= c.tiles;
        if (++c.hv == a.head_tiles * a.hs.num_kv_heads) {
            c.hv = 0;
            ++c.b;
            enter_request<C>(a, c);
            if (c.b >= a.requests) return;
        }
    }
}

// Where lane r finds row r of a tile: its byte offset in the pool, or -1 (no such cached row, or a bad page).
template <class C>
__device__ __forceinline__ int lookup_page(const PagedDecodeArgs& a, const Cursor& c, int lane) {
    const int pos = c.j * C::TW + lane;
    if (lane >= C::TW || pos >= c.len - 1) return -1;     // the newest position comes from this call's inputs
    return a.block_table[(size_t)c.b * a.table_width + pos / a.page_rows];
}
template <class C>
__device__ __forceinline__ long long row_offset(const PagedDecodeArgs& a, const Cursor& c, int page, int lane) {
    const int pos = c.j * C::TW + lane;
    if (lane >= C::TW || pos >= c.len - 1) return -1;
    if (!page_in_pool(page, a.num_pages)) {
        report_status(a.status, DEV_BAD_PAGE, 14);
        return -1;
    }
    return (long long)(pool_row(page, a.hs.num_kv_heads, c.hv / a.head_tiles, a.page_rows, pos % a.page_rows) * C::ROW);
}

template <class C>
__device__ __forceinline__ void load_tile(const PagedDecodeArgs& a, long long off, uint32_t stage, int lane) {
    const unsigned char* kp = static_cast<const unsigned char*>(a.k_pages);
    const unsigned char* vp = static_cast<const unsigned char*>(a.v_pages);
#pragma unroll
    for (int i = 0; i < C::CPT; ++i) {
        const int piece = i * 32 + lane, r = piece / C::CH, c = piece % C::CH;
        const long long at = __shfl_sync(FULL, off, r);
        const bool valid = at >= 0;
        const size_t from = (valid ? (size_t)at : 0) + c * 16;
        const uint32_t to = stage + tile_offset<C>(r, c);
        copy16(to, kp + from, valid);
        copy16(to + HALF, vp + from, valid);
    }
}

// ---- fp32 rows ----
template <class C>
struct StateF {
    f32x2 o[C::GT][2];     // four output columns of every head
    float m, l;            // of the head of this lane's score
    ulonglong2 q[C::GT][C::HD / 64];

    __device__ __forceinline__ void start(const float* qs, int lane) {
        const int i16 = lane & 15;
#pragma unroll
        for (int g = 0; g < C::GT; ++g) {
            o[g][0] = o[g][1] = 0ull;
#pragma unroll
            for (int c = 0; c < C::HD / 64; ++c) q[g][c] = *reinterpret_cast<const ulonglong2*>(qs + g * C::QS + (c * 16 + i16) * 4);
        }
        m = -INFINITY;
        l = 0.0f;
    }

    // Sum over the 16 lanes of a half-warp of each of NS values; lane i ends with value i % NS in acc[0].
    __device__ __forceinline__ static void sum16(float (&acc)[C::NS], int lane) {
#pragma unroll
        for (int off = 8; off >= 1; off >>= 1) {
            if (off < C::NS) {
                const bool up = (lane & off) != 0;
#pragma unroll
                for (int k = 0; k < C::NS; ++k)
                    if (k < off) {
                        const float send = up ? acc[k] : acc[k + off], keep = up ? acc[k + off] : acc[k];
                        acc[k] = keep + __shfl_xor_sync(FULL, send, off);
                    }
            } else {
#pragma unroll
                for (int k = 0; k < C::NS; ++k) acc[k] += __shfl_xor_sync(FULL, acc[k], off);
            }
        }
    }

    __device__ __forceinline__ void tile(const unsigned char* st, int nrows, float scale, f32x2* ps, int lane) {
        constexpr int HD = C::HD, GT = C::GT, R = C::R, NS = C::NS;
        const float* ks = reinterpret_cast<const float*>(st);
        const float* vs = reinterpret_cast<const float*>(st + HALF);
        const int i16 = lane & 15, hw = lane >> 4, e = i16 % NS, row_of = hw * R + e / GT;
        f32x2* as = ps + 2 * NS;
#pragma unroll
        for (int base = 0; base < C::TW; base += C::BR) {
            if (base >= nrows) break;
            f32x2 acc2[NS];
#pragma unroll
            for (int k = 0; k < NS; ++k) acc2[k] = 0ull;
#pragma unroll
            for (int rr = 0; rr < R; ++rr)
#pragma unroll
                for (int c = 0; c < HD / 64; ++c) {
                    const ulonglong2 kk = *reinterpret_cast<const ulonglong2*>(ks + (base + hw * R + rr) * HD + (c * 16 + i16) * 4);
#pragma unroll
                    for (int g = 0; g < GT; ++g) {
                        acc2[rr * GT + g] = ffma2(q[g][c].x, kk.x, acc2[rr * GT + g]);
                        acc2[rr * GT + g] = ffma2(q[g][c].y, kk.y, acc2[rr * GT + g]);
                    }
                }
            float acc[NS];
#pragma unroll
            for (int k = 0; k < NS; ++k) {
                float lo, hi;
                unpack2(acc2[k], lo, hi);
                acc[k] = lo + hi;
            }
            sum16(acc, lane);
            const float sc = base + row_of < nrows ? acc[0] * scale : -INFINITY;
            float top = sc;
#pragma unroll
            for (int off = GT; off < 32; off <<= 1)
                if (off < NS || off == 16) top = fmaxf(top, __shfl_xor_sync(FULL, top, off));
            const float mn = fmaxf(m, top), alpha = exp2f((m - mn) * LOG2E), p = exp2f((sc - mn) * LOG2E);
            l = fmaf(l, alpha, p);
            m = mn;
            __syncwarp();
            if (i16 < NS) ps[hw * NS + e] = pack2(p, p);     // row_of * GT + head
            if (lane < GT) as[lane] = pack2(alpha, alpha);
            __syncwarp();
#pragma unroll
            for (int g = 0; g < GT; ++g) {
                const f32x2 al = as[g];
                o[g][0] = fmul2(o[g][0], al);
                o[g][1] = fmul2(o[g][1], al);
            }
            constexpr int RPI = 128 / HD;     // v rows of one warp-wide load
#pragma unroll
            for (int rr = 0; rr < C::BR; rr += RPI) {
                const int rb = rr + (RPI == 2 ? hw : 0);
                const ulonglong2 vv = *reinterpret_cast<const ulonglong2*>(vs + (base + rb) * HD + (RPI == 2 ? i16 : lane) * 4);
#pragma unroll
                for (int g = 0; g < GT; ++g) {
                    const f32x2 pg = ps[rb * GT + g];
                    o[g][0] = ffma2(pg, vv.x, o[g][0]);
                    o[g][1] = ffma2(pg, vv.y, o[g][1]);
                }
            }
        }
    }

    __device__ __forceinline__ void park(float* to, float* ml, int lane) {
        // lanes that hold the same score twice (NS < 16) each summed it: only the first NS lanes of a half-warp count
        float sum = (lane & 15) < C::NS ? l : 0.0f;
#pragma unroll
        for (int off = C::GT; off < 32; off <<= 1) sum += __shfl_xor_sync(FULL, sum, off);
        if (lane < C::GT) {
            ml[2 * lane] = m;
            ml[2 * lane + 1] = sum;
        }
#pragma unroll
        for (int g = 0; g < C::GT; ++g) {
            float x[4];
            unpack2(o[g][0], x[0], x[1]);
            unpack2(o[g][1], x[2], x[3]);
            if constexpr (C::HD == 64) {      // the half-warps took every other v row
#pragma unroll
                for (int k = 0; k < 4; ++k) x[k] += __shfl_xor_sync(FULL, x[k], 16);
                if (lane < 16) *reinterpret_cast<float4*>(to + g * C::HD + lane * 4) = make_float4(x[0], x[1], x[2], x[3]);
            } else {
                *reinterpret_cast<float4*>(to + g * C::HD + lane * 4) = make_float4(x[0], x[1], x[2], x[3]);
            }
        }
    }
};

// ---- 16-bit rows ----
// Lane (g = lane / 4, t = lane % 4) of a multiplication holds rows g and g + 8 of the 16.
//   GT = 4:  rows 0-3 hi, 4-7 mid, 8-11 lo of the four heads
//   GT = 8:  X: rows 0-7 hi, 8-15 mid;  Y: rows 0-7 lo
//   GT = 16: hi, mid and lo of the sixteen heads in three
template <class C>
struct StateM {
    static constexpr int GT = C::GT, KS = C::HD / 16, N8 = C::HD / 8;
    static constexpr int QR = GT == 4 ? 4 : GT == 8 ? 6 : 12;     // q registers per 16 columns
    static constexpr int HL = GT == 16 ? 2 : 1;                   // heads of a lane
    uint32_t q[KS][QR];
    float o[N8][2 * HL];
    float m[HL], l[HL];

    __device__ __forceinline__ void start(const float* qs, int lane) {
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
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
#pragma unroll
        for (int n = 0; n < N8; ++n)
#pragma unroll
            for (int k = 0; k < 2 * HL; ++k) o[n][k] = 0.0f;
#pragma unroll
        for (int h = 0; h < HL; ++h) m[h] = -INFINITY, l[h] = 0.0f;
    }

    __device__ __forceinline__ void tile(const unsigned char* st, int nrows, float scale, f32x2*, int lane) {
        constexpr int NB = C::TW / 8;         // blocks of eight rows
        const uint32_t ks = smem_u32(st), vs = ks + HALF;
        const int t = lane & 3;
        float s[NB][2 * HL];
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            float c[4] = {0.f, 0.f, 0.f, 0.f}, d[4] = {0.f, 0.f, 0.f, 0.f};
            const int r = n * 8 + (lane & 7);
#pragma unroll
            for (int k2 = 0; k2 < KS; k2 += 2) {
                uint32_t b[4];
                ldsm4(b, ks + tile_offset<C>(r, 2 * k2 + (lane >> 3)));
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
            if constexpr (GT == 16) {
#pragma unroll
                for (int k = 0; k < 4; ++k) s[n][k] = c[k] + d[k];
            } else {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    s[n][k] = c[k] + (c[k + 2] + d[k]);
                    if constexpr (GT == 4) s[n][k] += __shfl_xor_sync(FULL, s[n][k], 16);
                }
            }
        }
        const float to2 = scale * LOG2E;
        if (nrows < C::TW) {
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int k = 0; k < 2 * HL; ++k)
                    if (n * 8 + 2 * t + (k & 1) >= nrows) s[n][k] = -INFINITY;
        }
        float alpha[HL];
#pragma unroll
        for (int h = 0; h < HL; ++h) {
            float top = -INFINITY;
#pragma unroll
            for (int n = 0; n < NB; ++n) top = fmaxf(top, fmaxf(s[n][2 * h], s[n][2 * h + 1]));
            top = fmaxf(top, __shfl_xor_sync(FULL, top, 1));
            top = fmaxf(top, __shfl_xor_sync(FULL, top, 2)) * to2;
            const float mn = fmaxf(m[h], top);
            alpha[h] = exp2f(m[h] - mn);
            m[h] = mn;
            float sum = 0.0f;
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    s[n][2 * h + k] = exp2f(fmaf(s[n][2 * h + k], to2, -mn));
                    sum += s[n][2 * h + k];
                }
            l[h] = fmaf(l[h], alpha[h], sum);
        }
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
#pragma unroll
        for (int n = 0; n < N8; n += 2) {
            float c[2][4] = {};
#pragma unroll
            for (int i = 0; i < NB / 2; ++i) {
                uint32_t b[4];
                const int r = i * 16 + (lane & 15);
                ldsm4t(b, vs + tile_offset<C>(r, n + (lane >> 4)));
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    mma16816(c[k], p[i][0], p[i][1], p[i][2], p[i][3], b[2 * k], b[2 * k + 1]);
                    if constexpr (GT == 8) mma16816(c[k], p[i][4], 0u, p[i][5], 0u, b[2 * k], b[2 * k + 1]);
                    if constexpr (GT == 16) {
                        mma16816(c[k], p[i][4], p[i][5], p[i][6], p[i][7], b[2 * k], b[2 * k + 1]);
                        mma16816(c[k], p[i][8], p[i][9], p[i][10], p[i][11], b[2 * k], b[2 * k + 1]);
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                if constexpr (GT == 16) {
#pragma unroll
                    for (int x = 0; x < 4; ++x) o[n + k][x] = fmaf(o[n + k][x], alpha[x >> 1], c[k][x]);
                } else {
                    o[n + k][0] = fmaf(o[n + k][0], alpha[0], c[k][0] + c[k][2]);
                    o[n + k][1] = fmaf(o[n + k][1], alpha[0], c[k][1] + c[k][3]);
                }
            }
        }
    }

    __device__ __forceinline__ void park(float* to, float* ml, int lane) {
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int h = 0; h < HL; ++h) {
            l[h] += __shfl_xor_sync(FULL, l[h], 1);
            l[h] += __shfl_xor_sync(FULL, l[h], 2);
            if (t == 0 && (GT != 4 || g < 4)) {
                ml[2 * (g + 8 * h)] = m[h];
                ml[2 * (g + 8 * h) + 1] = l[h];
            }
        }
#pragma unroll
        for (int n = 0; n < N8; ++n)
#pragma unroll
            for (int h = 0; h < HL; ++h) {
                float2 x = make_float2(o[n][2 * h], o[n][2 * h + 1]);
                if constexpr (GT == 4) {
                    x.x += __shfl_xor_sync(FULL, x.x, 16);
                    x.y += __shfl_xor_sync(FULL, x.y, 16);
                }
                if (GT != 4 || g < 4) *reinterpret_cast<float2*>(to + (g + 8 * h) * C::HD + n * 8 + 2 * t) = x;
            }
    }
};

// exp2 of a difference of maxima in the state's units (fp32 rows keep scores, 16-bit rows scores times log2 e); weight 0
// for a part that saw nothing.
template <class C>
__device__ __forceinline__ float part_weight(float m, float top) {
    if (m == -INFINITY) return 0.0f;
    return C::ES == 4 ? exp2f((m - top) * LOG2E) : exp2f(m - top);
}

template <class C>
struct StateOf {
    using type = StateM<C>;
};
template <int HD, int GT>
struct StateOf<Cfg<HD, 4, GT>> {
    using type = StateF<Cfg<HD, 4, GT>>;
};

// The bias, norm and rotation of this segment's q rows (into qs) and, where it ends with the new position, of the new k
// row and the v row (into xk and xv, and, by the first tile of heads, into their page).  A warp takes every fourth row.
template <class C>
__device__ __forceinline__ void prepare_rows(const PagedDecodeArgs& a, int b, int kv_h, int head0, int heads, int len, bool owns_new, bool stores,
                                             float* qs, float* xk, float* xv, int warp, int lane) {
    constexpr int HD = C::HD, PL = HD / 64, MAXIT = (C::GT + 2 + NW - 1) / NW;
    const int H = a.hs.num_heads, KV = a.hs.num_kv_heads, pos = len - 1;
    const int items = C::GT + (owns_new ? 2 : 0);
    float x[MAXIT][2 * PL];
#pragma unroll
    for (int n = 0; n < MAXIT; ++n) {
        const int it = warp + n * NW;
#pragma unroll
        for (int c = 0; c < 2 * PL; ++c) x[n][c] = 0.0f;
        if (it >= items || (it < C::GT && it >= heads)) continue;
        const int row = it < C::GT ? head0 + it : kv_h;
        const float* src = it < C::GT ? a.q + ((size_t)b * H + row) * HD : (it == C::GT ? a.k_new : a.v_new) + ((size_t)b * KV + row) * HD;
        const float* bias = it < C::GT ? a.b_q : it == C::GT ? a.b_k : a.b_v;
#pragma unroll
        for (int c = 0; c < 2 * PL; ++c) {
            x[n][c] = src[lane + 32 * c];
            if (bias) x[n][c] = __fadd_rn(x[n][c], bias[(size_t)row * HD + lane + 32 * c]);
        }
    }
    float rs[PL], rc[PL];
#pragma unroll
    for (int k = 0; k < PL; ++k) sincosf(__fmul_rn((float)pos, a.inv_freq[lane + 32 * k]), &rs[k], &rc[k]);
    float inv[MAXIT];
    if (a.q_norm != nullptr || a.k_norm != nullptr) {
#pragma unroll
        for (int n = 0; n < MAXIT; ++n) {
            inv[n] = 0.0f;
#pragma unroll
            for (int c = 0; c < 2 * PL; ++c) inv[n] = fmaf(x[n][c], x[n][c], inv[n]);
        }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1)
#pragma unroll
            for (int n = 0; n < MAXIT; ++n) inv[n] += __shfl_xor_sync(FULL, inv[n], off);
#pragma unroll
        for (int n = 0; n < MAXIT; ++n) inv[n] = (float)(1.0 / sqrt((double)(inv[n] / (float)HD) + a.eps));
    }
    int page = 0;
    if (owns_new && stores) {
        page = a.block_table[(size_t)b * a.table_width + pos / a.page_rows];
        if (!page_in_pool(page, a.num_pages)) {
            if (warp == 0 && lane == 0) report_status(a.status, DEV_BAD_PAGE, 15);
            stores = false;
        }
    }
    const size_t at = pool_row(stores ? page : 0, KV, kv_h, a.page_rows, pos % a.page_rows) * HD;
#pragma unroll
    for (int n = 0; n < MAXIT; ++n) {
        const int it = warp + n * NW;
        if (it >= items) break;
        float* to = it < C::GT ? qs + it * C::QS : it == C::GT ? xk : xv;
        if (it <= C::GT) {
            const float* w = it < C::GT ? a.q_norm : a.k_norm;
#pragma unroll
            for (int k = 0; k < PL; ++k) {
                float x0 = x[n][k], x1 = x[n][k + PL];
                if (w) {
                    x0 = __fmul_rn(__fmul_rn(x0, inv[n]), w[lane + 32 * k]);
                    x1 = __fmul_rn(__fmul_rn(x1, inv[n]), w[lane + 32 * k + HD / 2]);
                }
                x[n][k] = __fsub_rn(__fmul_rn(x0, rc[k]), __fmul_rn(x1, rs[k]));
                x[n][k + PL] = __fadd_rn(__fmul_rn(x1, rc[k]), __fmul_rn(x0, rs[k]));
            }
        }
#pragma unroll
        for (int c = 0; c < 2 * PL; ++c) {
            to[lane + 32 * c] = x[n][c];
            if (it >= C::GT && stores) {
                void* dst = it == C::GT ? a.k_pages : a.v_pages;
                if constexpr (C::ES == 4) static_cast<float*>(dst)[at + lane + 32 * c] = x[n][c];
                else static_cast<__nv_bfloat16*>(dst)[at + lane + 32 * c] = __float2bfloat16_rn(x[n][c]);
            }
        }
    }
}

// The new k and v rows into row r of a tile, as the pages hold them.
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
    __syncwarp();
}

template <class C>
__global__ void __launch_bounds__(THREADS, CTAS_PER_SM) paged_decode_kernel(PagedDecodeArgs a) {
    constexpr int HD = C::HD, GT = C::GT;
    extern __shared__ __align__(1024) unsigned char pd_smem[];
    float* qs = reinterpret_cast<float*>(pd_smem + C::RING);
    float* xk = qs + GT * C::QS;
    float* xv = xk + HD;
    float* wml = xv + HD;                                          // [NW][GT][2]
    f32x2* scratch = reinterpret_cast<f32x2*>(wml + NW * GT * 2);  // [NW][PS], fp32 rows only
    __shared__ long long sums[NW];
    __shared__ int s_b, s_last;
    __shared__ long long s_off;
    __shared__ int s_park[NW];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int H = a.hs.num_heads, KV = a.hs.num_kv_heads, G = H / KV;
    const int HV = KV * a.head_tiles;
    unsigned char* ring = pd_smem + (size_t)warp * STAGES * STAGE_BYTES;

    // ---- the line of tiles: its length, then the request in which this CTA's share starts ----
    auto scan = [&](int b0, long long& mine, long long& upto) {    // tiles of request b0 + tid and of all from b0 to it
        const int b = b0 + tid;
        mine = b < a.requests ? (long long)tiles_of<C>(valid_len<C>(a, b)) * HV : 0;
        upto = mine;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const long long up = __shfl_up_sync(FULL, upto, off);
            if (lane >= off) upto += up;
        }
        if (lane == 31) sums[warp] = upto;
        __syncthreads();
        long long all = 0;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            if (w < warp) upto += sums[w];
            all += sums[w];
        }
        __syncthreads();
        return all;
    };
    long long total = 0, mine, upto, t0 = 0, t1 = 0;
    for (int b0 = 0; b0 < a.requests; b0 += THREADS) total += scan(b0, mine, upto);
    const int ctas = (int)max(1ll, min((long long)gridDim.x, total / MIN_TILES));
    const int cta = blockIdx.x;
    auto share = [&](int c) { return total * c / ctas; };
    auto owner = [&](long long f) { return (int)(((f + 1) * ctas - 1) / total); };
    if (cta < ctas) t0 = share(cta), t1 = share(cta + 1);
    if (t0 < t1) {
        long long base = 0;
        for (int b0 = 0; b0 < a.requests; b0 += THREADS) {
            const long long all = a.requests <= THREADS ? total : scan(b0, mine, upto);
            if (mine > 0 && base + upto - mine <= t0 && t0 < base + upto) {
                s_b = b0 + tid;
                s_off = t0 - (base + upto - mine);
            }
            base += all;
        }
    }
    // padded rows, and lengths that do not fit: zeros
    for (int b = cta; b < a.requests; b += gridDim.x) {
        const int len = a.lens[b];
        if (valid_len<C>(a, b) > 0) continue;
        if (len != 0 && tid == 0) report_status(a.status, DEV_BAD_PAGE, 13);
        for (int d = tid; d < H * HD / 4; d += THREADS) reinterpret_cast<float4*>(a.out)[(size_t)b * (H * HD / 4) + d] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    __syncthreads();
    if (t0 >= t1) return;

    Cursor seg;      // the segment under way, at its first tile in this share
    seg.b = s_b;
    seg.len = valid_len<C>(a, seg.b);
    seg.tiles = tiles_of<C>(seg.len);
    seg.hv = (int)(s_off / seg.tiles);
    seg.j = (int)(s_off - (long long)seg.hv * seg.tiles);

    // ---- this warp's copies: tiles t0 + warp, t0 + warp + NW, ... ----
    Cursor ld = seg;
    long long next = t0 + warp;                      // tile the next copy is for
    int page = -1;
    if (next < t1) {
        advance<C>(a, ld, warp);
        page = lookup_page<C>(a, ld, lane);
    }
    int filled = 0, used = 0;                        // tiles copied into, and taken from, the ring so far
    auto fetch = [&]() {                             // one group of copies, empty behind the last tile
        if (next < t1) {
            const long long off = row_offset<C>(a, ld, page, lane);
            load_tile<C>(a, off, smem_u32(ring + (filled % STAGES) * STAGE_BYTES), lane);
            ++filled;
            next += NW;
            if (next < t1) {
                advance<C>(a, ld, NW);
                page = lookup_page<C>(a, ld, lane);
            }
        }
        copy_commit();
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) fetch();

    typename StateOf<C>::type st;
    long long at = t0;                               // line position of seg
    while (true) {
        const int jend = (int)min((long long)seg.tiles, seg.j + (t1 - at));
        const long long end = at + (jend - seg.j), whole0 = at - seg.j, whole1 = whole0 + seg.tiles;
        const int kv_h = seg.hv / a.head_tiles, ht = seg.hv - kv_h * a.head_tiles;
        const int per = (G + a.head_tiles - 1) / a.head_tiles;
        const int head0 = kv_h * G + ht * per, heads = min(per, G - ht * per);
        const bool owns_new = jend == seg.tiles;
        prepare_rows<C>(a, seg.b, kv_h, head0, heads, seg.len, owns_new, ht == 0, qs, xk, xv, warp, lane);
        __syncthreads();
        st.start(qs, lane);
        // the first tile of this segment that is this warp's
        for (int j = seg.j + (int)((warp - (at - t0)) & (NW - 1)); j < jend; j += NW) {
            copy_wait<STAGES - 2>();
            __syncwarp();
            unsigned char* stage = ring + (used % STAGES) * STAGE_BYTES;
            const int nrows = min(C::TW, seg.len - j * C::TW);
            if (j == seg.tiles - 1) patch_tile<C>(stage, nrows - 1, xk, xv, lane);
            fetch();
            st.tile(stage, nrows, a.scale, scratch + warp * C::PS, lane);
            __syncwarp();
            ++used;
        }
        // the stage that was used last is not filled again before the next tile: the sums wait there for the join
        const int free_stage = (used + STAGES - 1) % STAGES;
        st.park(reinterpret_cast<float*>(ring + free_stage * STAGE_BYTES), wml + warp * GT * 2, lane);
        if (lane == 0) s_park[warp] = free_stage;
        __syncthreads();

        // ---- the four warps' sums, to the output or to the workspace ----
        const bool complete = at == whole0 && end == whole1;
        const size_t part = (size_t)cta * 2 + (at == t0 ? 0 : 1);
        for (int e = tid; e < GT * HD / 4; e += THREADS) {
            const int g = e / (HD / 4), d = (e - g * (HD / 4)) * 4;
            if (g >= heads) break;
            float top = -INFINITY, L = 0.0f;
#pragma unroll
            for (int w = 0; w < NW; ++w) top = fmaxf(top, wml[(w * GT + g) * 2]);
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const float wt = part_weight<C>(wml[(w * GT + g) * 2], top);
                const float4 v = *reinterpret_cast<const float4*>(pd_smem + (size_t)(w * STAGES + s_park[w]) * STAGE_BYTES + (g * HD + d) * 4);
                L = fmaf(wt, wml[(w * GT + g) * 2 + 1], L);
                acc.x = fmaf(wt, v.x, acc.x);
                acc.y = fmaf(wt, v.y, acc.y);
                acc.z = fmaf(wt, v.z, acc.z);
                acc.w = fmaf(wt, v.w, acc.w);
            }
            if (complete) {
                const float inv = 1.0f / L;
                *reinterpret_cast<float4*>(a.out + ((size_t)seg.b * H + head0 + g) * HD + d) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
            } else {
                *reinterpret_cast<float4*>(a.part_o + (part * GT + g) * HD + d) = acc;
                if (d == 0) *reinterpret_cast<float2*>(a.part_ml + (part * GT + g) * 2) = make_float2(top, L);
            }
        }
        if (!complete) {
            const int c0 = owner(whole0), c1 = owner(whole1 - 1);
            __syncthreads();
            if (tid == 0) {      // the barrier, then one acquire-release addition: parts are complete before they are counted
                unsigned n;
                asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(n) : "l"(a.counters + c0) : "memory");
                s_last = n == (unsigned)(c1 - c0);
                if (s_last) a.counters[c0] = 0u;
            }
            __syncthreads();
            if (s_last) {
                for (int e = tid; e < GT * HD / 4; e += THREADS) {
                    const int g = e / (HD / 4), d = (e - g * (HD / 4)) * 4;
                    if (g >= heads) break;
                    float top = -INFINITY, L = 0.0f;
                    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
                    constexpr int RND = 8;       // parts requested before the first is used
                    for (int c = c0; c <= c1; c += RND) {
                        float2 ml[RND];
                        float4 v[RND];
#pragma unroll
                        for (int k = 0; k < RND; ++k) {
                            ml[k] = make_float2(-INFINITY, 0.f);
                            v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                            if (c + k <= c1) {
                                const size_t p = ((size_t)(c + k) * 2 + (c + k == c0 && share(c0) < whole0 ? 1 : 0)) * GT + g;
                                ml[k] = __ldcg(reinterpret_cast<const float2*>(a.part_ml) + p);
                                v[k] = __ldcg(reinterpret_cast<const float4*>(a.part_o + p * HD + d));
                            }
                        }
                        float mn = top;
#pragma unroll
                        for (int k = 0; k < RND; ++k) mn = fmaxf(mn, ml[k].x);
                        const float old = part_weight<C>(top, mn);
                        L *= old;
                        acc.x *= old, acc.y *= old, acc.z *= old, acc.w *= old;
                        top = mn;
#pragma unroll
                        for (int k = 0; k < RND; ++k) {
                            const float wt = part_weight<C>(ml[k].x, mn);
                            L = fmaf(wt, ml[k].y, L);
                            acc.x = fmaf(wt, v[k].x, acc.x);
                            acc.y = fmaf(wt, v[k].y, acc.y);
                            acc.z = fmaf(wt, v[k].z, acc.z);
                            acc.w = fmaf(wt, v[k].w, acc.w);
                        }
                    }
                    const float inv = 1.0f / L;
                    *reinterpret_cast<float4*>(a.out + ((size_t)seg.b * H + head0 + g) * HD + d) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
                }
            }
        }
        at = end;
        if (at >= t1) break;
        __syncthreads();      // parked sums, q rows and new rows have been read
        advance<C>(a, seg, jend - seg.j);
    }
    copy_wait<0>();
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
    paged_decode_kernel<C><<<ctas, THREADS, C::SMEM, s>>>(a);
    return cudaGetLastError();
}

template <int HD, int ES>
cudaError_t launch_heads(const PagedDecodeArgs& a, int gt, int ctas, cudaStream_t s) {
    if constexpr (ES == 4) {
        if (gt == 1) return launch<HD, ES, 1>(a, ctas, s);
        if (gt == 2) return launch<HD, ES, 2>(a, ctas, s);
        if (gt == 4) return launch<HD, ES, 4>(a, ctas, s);
        return launch<HD, ES, 8>(a, ctas, s);
    } else {
        if (gt == 4) return launch<HD, ES, 4>(a, ctas, s);
        if (gt == 8) return launch<HD, ES, 8>(a, ctas, s);
        return launch<HD, ES, 16>(a, ctas, s);
    }
}

}  // namespace

PagedPlan paged_decode_plan(const HeadShape& hs, int kv_elem_bytes, int sm_count) {
    const int G = hs.num_heads / hs.num_kv_heads, most = kv_elem_bytes == 4 ? 8 : 16;
    PagedPlan p;
    p.head_tiles = (G + most - 1) / most;
    const int per = (G + p.head_tiles - 1) / p.head_tiles;
    p.gt = kv_elem_bytes == 4 ? 1 : 4;
    while (p.gt < per) p.gt *= 2;
    p.ctas = sm_count * CTAS_PER_SM;
    p.part_floats = (size_t)p.ctas * 2 * p.gt * (hs.head_dim + 2);
    return p;
}

cudaError_t launch_paged_decode(PagedDecodeArgs a, const PagedPlan& p, float* workspace, unsigned* counters, cudaStream_t s) {
    a.head_tiles = p.head_tiles;
    a.part_o = workspace;
    a.part_ml = workspace + (size_t)p.ctas * 2 * p.gt * a.hs.head_dim;
    a.counters = counters;
    const long long most = (long long)a.table_width * a.page_rows * a.hs.num_kv_heads * p.head_tiles;   // tiles, at one row each
    const int ctas = (int)std::min<long long>(p.ctas, std::max<long long>(1, std::min<long long>(most, 0x7fffffff) * a.requests));
    if (a.hs.head_dim == 128) return a.kv_elem_bytes == 4 ? launch_heads<128, 4>(a, p.gt, ctas, s) : launch_heads<128, 2>(a, p.gt, ctas, s);
    return a.kv_elem_bytes == 4 ? launch_heads<64, 4>(a, p.gt, ctas, s) : launch_heads<64, 2>(a, p.gt, ctas, s);
}

}  // namespace shainet
