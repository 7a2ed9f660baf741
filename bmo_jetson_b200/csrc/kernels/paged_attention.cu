// paged_attention.cu -- attention of single tokens over the paged key-value
// cache, the work of all rows split evenly over the GPU's warps and joined.
//
//   s_j = scale * q . k_j,  out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m)
//
// over the last `window` positions of a row.  One pass over the keys and
// values: each warp keeps a running maximum, the sum of the weights and the
// weighted sum of the values, and rescales them when the maximum grows.
//
// Every key and value is read once and used for a few query heads, so the
// kernel is bound by memory; what has to be avoided is anything that keeps
// loads from being in flight.  Both products are mma.sync m16n8k16 with the rows
// as its A operand.  (tcgen05.mma would need them in shared memory in its
// canonical layout, and 128 rows of B's side, of which a decode step fills 2.)
//   scores: A = 16 positions x 16 elements of K, B = q
//   values: A = 16 elements x 16 positions of V^T, B = the weights
// B has 8 columns.  An fp32 factor x, brought into fp16's range by a power of
// two, takes two of them: hi = fp16(x) and lo = fp16(2^11 (x - hi)), whose sum is
// divided by 2^11 when the two are added.  So products with fp16 keys and values
// keep 22 bits of x, relative to x itself down to 2^-14 and to 2^-36 absolute
// below (an unscaled lo would end at 2^-25: weights 2^-32 of the largest would
// count as nothing, some 2^-15 of a row of 131072).  The
// tensor core sums a tile in fp32, and tiles are added by fp32 additions.
//
// fp16 cache: columns 2t, 2t + 1 are head t of a group of 4 (or of 2 x 4).  The
// contraction runs over a permuted index, so that 16 consecutive bytes of a
// row are a lane's fragment: rows go from global memory straight into
// registers, and nothing is staged.  64 sessions of up to 3000 positions, 32
// heads of 128 (1.64 GB): 259 to 264 us, 6.2 to 6.3 TB/s, 0.97 of the measured copy.
//
// Q4_0 cache: columns 2t, 2t + 1 are block t of head_dim.  q is masked to the
// block, so the score comes out as one sum over codes a block, which the
// block's scale multiplies in fp32; and the weight of a value's block is p times that
// block's scale.  Unpacking costs two instructions per two codes, on
// half-rate pipes, and makes the kernel bound by instructions and their latencies at
// three warps a scheduler: registers go to the arithmetic, and rows arrive in a ring in
// shared memory by asynchronous copies.  64 sessions of 1500 positions (442 MB): 104 to
// 106 us, 4.2 TB/s, the issue slots 62% busy; the rows in registers took 152 us, the
// ring alone brought 111.
//
// Work: a row's window is cut into tiles of kTile positions; (row, key head,
// tile) in that order is a line of tiles of which every warp takes an equal,
// contiguous part.  A head that lies within one warp's part is written at once.
// Otherwise its pieces are joined in shared memory among the CTA's warps,
// then through global memory by the last CTA to arrive, in the order of the
// line, so the result does not depend on the order of arrival.  Nothing waits for
// another CTA.  A call of few heads is bound by latency instead (its code
// is fetched cold, then loads, two barriers and the join follow one another): there a head gets a
// CTA or a cluster of CTAs of its own, chosen in pa_launch.
#include <cuda_bf16.h>
#include <math.h>

#include <atomic>
#include <type_traits>

#include "../paged.h"
#include "common.cuh"

namespace bmo {
namespace {

constexpr int kPaWarps = 4;
constexpr int kPaThreads = 32 * kPaWarps;
constexpr float kLn2 = 0.6931471805599453f;
// Weights are e^(s - m) * 2^7 in two fp16 parts; the maximum m is raised only
// when a score passes it by more than 2^8, so a weight is below 2^15.  Of n
// weights the parts leave out 2^-22 of each and n 2^-43 of the largest.
constexpr float kSlack = 8.0f, kHead = 7.0f;
// The second part of a factor is held times kLo.
constexpr float kLo = 2048.0f, kLoInv = 1.0f / 2048.0f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint4 ldg_stream16(const void *p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
        : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
        : "l"(p));
    return v;
}

// Shared memory by 32-bit address.
__device__ __forceinline__ uint4 lds16(uint32_t p) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(p) : "memory");
    return v;
}
__device__ __forceinline__ uint2 lds8(uint32_t p) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(p) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t lds4(uint32_t p) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(p) : "memory");
    return v;
}
__device__ __forceinline__ float lds_half(uint32_t p) {
    uint16_t v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(p) : "memory");
    return __half2float(__ushort_as_half(v));
}
template <int N>
__device__ __forceinline__ void copy_async(uint32_t dst, const void *src) {
    if constexpr (N == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(N) : "memory");
}

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// c = A B if first, else c += A B (first known at compile time).
__device__ __forceinline__ void mma16816(float (&c)[4], bool first, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
    if (first)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%10, %10, %10, %10};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
    else
        mma16816(c, a0, a1, a2, a3, b0, b1);
}

__device__ __forceinline__ uint32_t word(const uint4 &x, int i) { return i == 0 ? x.x : i == 1 ? x.y : i == 2 ? x.z : x.w; }

// Transpose of an 8 x 8 matrix of 16-bit elements held two a lane.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ void split_half2(float x, float y, uint32_t &px, uint32_t &py) {  // (hi, lo) of x, of y
    const __half2 hi = __floats2half2_rn(x, y);
    const float2 f = __half22float2(hi);
    const __half2 lo = __floats2half2_rn((x - f.x) * kLo, (y - f.y) * kLo);
    const uint32_t h = *reinterpret_cast<const uint32_t *>(&hi), l = *reinterpret_cast<const uint32_t *>(&lo);
    px = __byte_perm(h, l, 0x5410);
    py = __byte_perm(h, l, 0x7632);
}
__device__ __forceinline__ uint32_t half_bits2(__half a, __half b) {
    const __half2 p = __halves2half2(a, b);
    return *reinterpret_cast<const uint32_t *>(&p);
}

// Codes 0..15 at bits 0-3 and 16-19 (or 4-7 and 20-23) of w as halves n - 8,
// by the usual way from a small integer to a float: its bits are placed in the
// mantissa of a power of two, 1024, which is taken away with the offset.
__device__ __forceinline__ uint32_t codes_lo(uint32_t w) {
    uint32_t m;
    asm("lop3.b32 %0, %1, 0x000f000f, 0x64006400, 0xea;" : "=r"(m) : "r"(w));  // (w & mask) | 1024.0
    const __half2 h = __hsub2(*reinterpret_cast<const __half2 *>(&m), __float2half2_rn(1032.0f));
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t codes_hi(uint32_t w) {
    uint32_t m;
    asm("lop3.b32 %0, %1, 0x00f000f0, 0x64006400, 0xea;" : "=r"(m) : "r"(w));
    const __half2 h =
        __hfma2(*reinterpret_cast<const __half2 *>(&m), __float2half2_rn(0.0625f), __float2half2_rn(-72.0f));
    return *reinterpret_cast<const uint32_t *>(&h);
}

// Activations are read and written an element a lane: a warp's accesses are
// whole lines whatever the rows' alignment, and the code stays short.  (These kernels
// run for a few microseconds and fetch their code cold on every SM.)
template <int ACT>
__device__ __forceinline__ float act_load(const void *p, long long i) {
    if constexpr (ACT == BMO_ACT_F32) return static_cast<const float *>(p)[i];
    else if constexpr (ACT == BMO_ACT_F16) return __half2float(static_cast<const __half *>(p)[i]);
    else return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}
template <int ACT>
__device__ __forceinline__ void act_store(void *p, long long i, float x) {
    if constexpr (ACT == BMO_ACT_F32) static_cast<float *>(p)[i] = x;
    else if constexpr (ACT == BMO_ACT_F16) static_cast<__half *>(p)[i] = __float2half_rn(x);
    else static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(x);
}

// The power of two that brings amax into [2^10, 2^11), and its inverse
// (both normal floats; amax 0, infinite or NaN gives some finite factor).
__device__ __forceinline__ void range_factor(float amax, float &mul, float &inv) {
    int ex = (__float_as_int(amax) >> 23) & 255;
    ex = min(max(ex, 11), 254);
    mul = __int_as_float((264 - ex) << 23);
    inv = __int_as_float((ex - 10) << 23);
}

// 4 elements of a query head, split: times the power of two that brings the
// head into fp16's range; inv: that power's inverse.
struct QueryPart {
    __half hi[4], lo[4];
    float inv;
};
template <int ACT, int HD>
__device__ __forceinline__ void query_load(const void *src, long long at, int lane, float (&x)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = 4 * lane < HD ? act_load<ACT>(src, at + 4 * lane + i) : 0.0f;
}
__device__ __forceinline__ QueryPart query_part(const float (&x)[4]) {
    const float amax = warp_max(fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))));
    QueryPart p;
    float mul;
    range_factor(amax, mul, p.inv);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float y = x[i] * mul;
        p.hi[i] = __float2half_rn(y);
        p.lo[i] = __float2half_rn((y - __half2float(p.hi[i])) * kLo);
    }
    return p;
}

// Rows of 16 consecutive positions of a layer, numbered from 0 (fewer than
// 2^32, checked by the entry point).  Pages of a multiple of 16 positions:
// one number, of position 0.  Other page sizes: each lane's own rows, each
// less the position's number, so that the addresses are formed the same way.
template <bool kAligned>
struct Pos16;
template <>
struct Pos16<true> {
    uint32_t first;
    __device__ __forceinline__ long long row(int) const { return first; }
    __device__ __forceinline__ long long key(int) const { return first; }
    __device__ __forceinline__ long long value(int) const { return first; }
};
template <>
struct Pos16<false> {
    long long k[2], v[4];
    uint32_t mine;  // row of position lane % 16
    __device__ __forceinline__ long long row(int i) const {  // every lane of the warp asks
        return static_cast<long long>(__shfl_sync(0xffffffffu, mine, i)) - i;
    }
    __device__ __forceinline__ long long key(int i) const { return k[i]; }
    __device__ __forceinline__ long long value(int i) const { return v[i]; }
};
// Position that a lane holds: i-th of its keys, of its values.
__device__ __forceinline__ int key_pos(int lane, int i) { return (lane >> 2) + 8 * i; }
__device__ __forceinline__ int value_pos(int lane, int i) { return 2 * (lane & 3) + (i & 1) + 4 * (i & 2); }

// ---- fp16 rows ----
template <int HD_, int NB_>
struct F16Rows {
    static constexpr int HD = HD_, NB = NB_;
    static constexpr int kMinCtas = NB == 1 ? 3 : 2;
    static constexpr int kHeadCost = 1;
    static constexpr int kHeads = 4 * NB;          // query heads of a unit
    static constexpr int kSub = HD == 128 ? 1 : 2; // 16-position parts of a tile
    static constexpr int kO = HD / 16;
    uint32_t q[NB][HD / 16][2];
    float inv[NB];
    uint4 kr[kSub][2][HD / 32], vr[kSub][4][HD / 64];

    // B fragments of the unit's queries (element q0 of q): a lane splits 4
    // elements of a head at a time into buf[head][hi, lo][HD] (halves), from where
    // each lane's fragments are 16-byte words.  Columns of heads past n_heads are zero.
    template <int ACT>
    __device__ __forceinline__ void load_q(const void *src, long long q0, int n_heads, float qscale, float *buf, int lane) {
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) inv[nb] = 1.0f;
        float x[kHeads][4];  // all heads' loads in flight
#pragma unroll
        for (int j = 0; j < kHeads; ++j)
            if (j < n_heads) query_load<ACT, HD>(src, q0 + j * HD, lane, x[j]);
#pragma unroll
        for (int j = 0; j < kHeads; ++j) {
            if (j >= n_heads) continue;
            const QueryPart p = query_part(x[j]);
            if (4 * lane < HD) {
                uint2 *dst = reinterpret_cast<uint2 *>(buf + j * HD) + lane;
                dst[0] = make_uint2(half_bits2(p.hi[0], p.hi[1]), half_bits2(p.hi[2], p.hi[3]));
                dst[HD / 4] = make_uint2(half_bits2(p.lo[0], p.lo[1]), half_bits2(p.lo[2], p.lo[3]));
            }
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
                if (j == 4 * nb + t) inv[nb] = p.inv * qscale;
        }
        __syncwarp();
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const int h = 4 * nb + (g >> 1);
            const uint4 *frag = reinterpret_cast<const uint4 *>(buf + (h < n_heads ? h : 0) * HD) + (g & 1) * (HD / 8) + t;
#pragma unroll
            for (int c = 0; c < HD / 32; ++c) {
                const uint4 u = h < n_heads ? frag[4 * c] : make_uint4(0, 0, 0, 0);
                q[nb][2 * c][0] = u.x, q[nb][2 * c][1] = u.y, q[nb][2 * c + 1][0] = u.z, q[nb][2 * c + 1][1] = u.w;
            }
        }
    }
    // Rows go straight into registers: the next tile's keys are requested as
    // soon as a tile's scores are formed, its values at the start of its step.
    static constexpr int kRing = 0;
    const char *kp, *vp;  // the lane's bytes of positions g and 2t, were they in rows g and 2t
    __device__ __forceinline__ F16Rows(const PagedAttnArgs &a, char *, int lane)
        : kp(static_cast<const char *>(a.k) + 2 * HD * (lane >> 2) + 16 * (lane & 3)),
          vp(static_cast<const char *>(a.v) + 4 * HD * (lane & 3) + 16 * (lane >> 2)) {}
    template <class P>
    __device__ __forceinline__ void load_k(int s, const P &p) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int c = 0; c < HD / 32; ++c) kr[s][i][c] = ldg_stream16(kp + p.key(i) * (2 * HD) + 16 * HD * i + 64 * c);
    }
    template <class P>
    __device__ __forceinline__ void load_v(int s, const P &p) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int c = 0; c < HD / 64; ++c)
                vr[s][i][c] = ldg_stream16(vp + p.value(i) * (2 * HD) + 2 * HD * value_pos(0, i) + 128 * c);
    }
    // Values of positions that are left out (bit 0 in `there`) must not meet their weight 0 as NaN.
    __device__ __forceinline__ void clear_values(uint32_t there, int lane) {
#pragma unroll
        for (int s = 0; s < kSub; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (!(there >> (16 * s + value_pos(lane, i)) & 1))
#pragma unroll
                    for (int c = 0; c < HD / 64; ++c) vr[s][i][c] = make_uint4(0, 0, 0, 0);
    }
    // sc[nb][i]: score (log2 units) of position g + 8 i for head (nb, t)
    __device__ __forceinline__ void scores(int s, float (&sc)[NB][2]) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            float c[4], d[4];  // two shorter chains
#pragma unroll
            for (int j = 0; j < HD / 32; ++j) {
                const uint4 x = kr[s][0][j], y = kr[s][1][j];
                mma16816(c, j == 0, x.x, y.x, x.y, y.y, q[nb][2 * j][0], q[nb][2 * j][1]);
                mma16816(d, j == 0, x.z, y.z, x.w, y.w, q[nb][2 * j + 1][0], q[nb][2 * j + 1][1]);
            }
            sc[nb][0] = __fmaf_rn(c[1] + d[1], kLoInv, c[0] + d[0]) * inv[nb];
            sc[nb][1] = __fmaf_rn(c[3] + d[3], kLoInv, c[2] + d[2]) * inv[nb];
        }
    }
    __device__ __forceinline__ void reset() {}
    // Element d of a row is code(d) times scale(d / 32).
    __device__ __forceinline__ static float code(const void *rows, long long row, int d) {
        return __half2float(static_cast<const __half *>(rows)[row * HD + d]);
    }
    __device__ __forceinline__ static float scale(const __half *, long long, int) { return 1.0f; }
    // Adds the weighted values of the tile.  The tensor core's sum of a tile
    // starts from zero and is added in fp32: its own running sum is not rounded to nearest.
    __device__ __forceinline__ void values(const float (&w)[kSub][NB][2], float (&o)[NB][kO][4]) {
        uint32_t b[kSub][NB][2];
#pragma unroll
        for (int s = 0; s < kSub; ++s)
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                split_half2(w[s][nb][0], w[s][nb][1], b[s][nb][0], b[s][nb][1]);
                b[s][nb][0] = transpose8(b[s][nb][0]);
                b[s][nb][1] = transpose8(b[s][nb][1]);
            }
#pragma unroll
        for (int j = 0; j < kO; ++j) {
            float sum[NB][4];
#pragma unroll
            for (int s = 0; s < kSub; ++s) {
                const uint32_t v0 = word(vr[s][0][j / 4], j % 4), v1 = word(vr[s][1][j / 4], j % 4),
                               v2 = word(vr[s][2][j / 4], j % 4), v3 = word(vr[s][3][j / 4], j % 4);
                const uint32_t a0 = __byte_perm(v0, v1, 0x5410), a1 = __byte_perm(v0, v1, 0x7632);
                const uint32_t a2 = __byte_perm(v2, v3, 0x5410), a3 = __byte_perm(v2, v3, 0x7632);
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) mma16816(sum[nb], s == 0, a0, a1, a2, a3, b[s][nb][0], b[s][nb][1]);
            }
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[nb][j][i] += sum[nb][i];
        }
    }
    // The lane's 8 consecutive elements [64 c + 8 g, + 8) of head (nb, t).
    static constexpr int kRuns = HD / 64, kRunLen = 8;
    __device__ __forceinline__ bool owns(int) const { return true; }
    __device__ __forceinline__ static int head_of(int nb, int lane) { return 4 * nb + (lane & 3); }
    __device__ __forceinline__ static int run_start(int run, int lane) { return 64 * run + 8 * (lane >> 2); }
    __device__ __forceinline__ float element(const float (&o)[kO][4], int run, int i) const {
        const float *c = o[4 * run + i / 2];
        return i % 2 ? __fmaf_rn(c[3], kLoInv, c[2]) : __fmaf_rn(c[1], kLoInv, c[0]);
    }
};

// ---- Q4_0 rows ----
template <int HD_, int NB_>
struct Q4Rows {
    static constexpr int HD = HD_, NB = NB_;
    static constexpr int kMinCtas = HD * NB <= 128 ? 3 : 2;
    static constexpr int kHeadCost = 2;
    static constexpr int kHeads = NB;             // query heads of a unit: they share the work on the codes
    static constexpr int kSub = 2;
    static constexpr int kO = HD / 16;
    static constexpr int kBlocks = HD / 32;       // <= 4: a column pair each
    static constexpr int kKW = HD / 32;           // words of a key row a lane holds
    static constexpr int kVW = HD / 64;           // words of a value row a lane holds
    // The queries' fragments: of one head in registers; of more in shared memory,
    // where lanes that hold other blocks' codes read zeros.
    uint4 q[NB == 1 ? kKW : 1];
    uint32_t q_at, q_step;
    float inv[NB];
    float vlim, vinv;  // power of two that bounds the value scales seen so far, and its inverse
    float vs[kSub][2];
    // B fragments of the queries: a lane splits 4 elements of each and puts them
    // where the lanes that hold their codes find their fragments as 16-byte
    // words: buf[head][block][hi, lo][16] (pairs of halves).
    template <int ACT>
    __device__ __forceinline__ void load_q(const void *src, long long q0, int n_heads, float qscale, float *buf, int lane) {
        const int g = lane >> 2, t = lane & 3;
        const int i = lane & 7;  // elements 4i.. of block lane / 8
        float e[NB][4];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)  // a head past n_heads: the first again, not used
            query_load<ACT, HD>(src, q0 + (nb < n_heads ? nb : 0) * HD, lane, e[nb]);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const QueryPart x = query_part(e[nb]);
            inv[nb] = x.inv * qscale;
            if (4 * lane < HD) {
                // word 4 (i % 4): codes of bytes 4 (i % 4).. : elements 0, 2 then 1, 3; low nibbles before high ones
                uint32_t *dst = reinterpret_cast<uint32_t *>(buf + nb * HD) + (lane >> 3) * 32 + 4 * (i & 3) + (i >> 2);
                dst[0] = half_bits2(x.hi[0], x.hi[2]), dst[2] = half_bits2(x.hi[1], x.hi[3]);
                dst[16] = half_bits2(x.lo[0], x.lo[2]), dst[18] = half_bits2(x.lo[1], x.lo[3]);
            }
        }
        __syncwarp();
        // lane t holds bytes 4 w.. of block blk, w in [w0, w0 + kKW); column pair g / 2 is block g / 2
        const int blk = HD == 128 ? t : t >> 1, w0 = HD == 128 ? 0 : 2 * (t & 1);
        const bool mine = (g >> 1) == blk;
        const uint32_t at = smem_addr(buf) + 4 * (blk * 32 + (g & 1) * 16) + 16 * w0;
        if constexpr (NB == 1) {
#pragma unroll
            for (int w = 0; w < kKW; ++w) q[w] = mine ? lds16(at + 16 * w) : make_uint4(0, 0, 0, 0);
        } else {
            q_at = mine ? at : ring + 3 * kStage;
            q_step = mine ? 4 * HD : 0;
        }
    }
    __device__ __forceinline__ uint4 fragment(int nb, int w) const {
        if constexpr (NB == 1) return q[w];
        else return lds16(q_at + nb * q_step + 16 * w);
    }
    // Rows reach shared memory by asynchronous copies, two tiles ahead (the
    // arithmetic on codes leaves no registers to hold that much): a stage is
    // the tile's key codes, value codes, key scales, value scales.  16-byte
    // chunks of value rows 2, 3 (mod 4) are swapped so that a warp's reads spread over the banks.
    static constexpr int kTile = 16 * kSub, kRow = HD / 2, kScaleRow = 2 * kBlocks;
    static constexpr int kOffV = kTile * kRow, kOffKs = 2 * kOffV, kOffVs = kOffKs + kTile * kScaleRow;
    static constexpr int kStage = kOffVs + kTile * kScaleRow;
    static constexpr int kRing = 3 * kStage + (NB > 1 ? 64 : 0);  // bytes of a warp: the stages, and zeros
    const char *kp, *vp, *sp;       // the lane's bytes of rows 0..15: codes of keys and values, scales of either
    uint32_t ring, to_k, to_v, to_s;  // where they go in a stage
    uint32_t at_k, at_ks, at_v, at_vs;  // what the lane reads of a stage
    uint32_t stage;  // that of the tile whose values are added; the next one's is kStage further
    __device__ __forceinline__ Q4Rows(const PagedAttnArgs &a, char *warp_ring, int lane) : ring(smem_addr(warp_ring)) {
        constexpr int kChunks = kRow / 16;  // of a row: a lane copies chunks lane, lane + 32, .. of 16 rows
        const int g = lane >> 2, t = lane & 3, row = lane / kChunks;
        kp = static_cast<const char *>(a.k) + 16 * lane;
        vp = static_cast<const char *>(a.v) + 16 * lane;
        sp = static_cast<const char *>(lane < 16 ? static_cast<const void *>(a.k_scale) : a.v_scale) + (lane & 15) * kScaleRow;
        to_k = 16 * lane;
        to_v = kOffV + swizzle(row, lane % kChunks);
        to_s = (lane < 16 ? kOffKs : kOffVs) + (lane & 15) * kScaleRow;
        at_k = g * kRow + 4 * kKW * t;
        at_ks = kOffKs + g * kScaleRow + 2 * (t % kBlocks);
        at_v = kOffV + swizzle(2 * t, 4 * kVW * g / 16) + 4 * kVW * g % 16;
        at_vs = kOffVs + g * kScaleRow + 2 * (t % kBlocks);
        if (NB > 1 && lane < 16) reinterpret_cast<uint32_t *>(warp_ring + 3 * kStage)[lane] = 0;
    }
    // Byte of a 16-byte chunk of a value row; rows 1 and 8 on have the same swizzle.
    __device__ __forceinline__ static int swizzle(int row, int chunk) { return row * kRow + 16 * (kRow == 64 ? chunk ^ (row & 2) : chunk); }
    // Requests a tile, into the stage two after the one in use.
    template <class P>
    __device__ __forceinline__ void request(const P (&p)[kSub], int lane) {
        const uint32_t dst = stage == ring ? ring + 2 * kStage : stage - kStage;
#pragma unroll
        for (int s = 0; s < kSub; ++s) {
#pragma unroll
            for (int i = 0; i < kRow / 32; ++i) {  // 512 bytes of the 16 rows each
                const long long r = p[s].row((lane + 32 * i) / (kRow / 16)) * kRow + 512 * i;
                copy_async<16>(dst + to_k + 16 * s * kRow + 512 * i, kp + r);
                copy_async<16>(dst + to_v + 16 * s * kRow + 512 * i, vp + r);
            }
            copy_async<kScaleRow>(dst + to_s + 16 * s * kScaleRow, sp + p[s].row(lane & 15) * kScaleRow);
        }
    }
    __device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
    // All requests but the last have arrived, for all lanes.
    __device__ __forceinline__ void wait() {
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        __syncwarp();
    }
    __device__ __forceinline__ void next() { stage = stage == ring + 2 * kStage ? ring : stage + kStage; }
    // The value scales of the tile in use; those of positions that are left out
    // must not meet their weight 0 as NaN (codes are always finite).
    __device__ __forceinline__ void load_scales(uint32_t there, int lane) {
#pragma unroll
        for (int s = 0; s < kSub; ++s)
#pragma unroll
            for (int i = 0; i < 2; ++i) vs[s][i] = lds_half(stage + at_vs + (16 * s + 8 * i) * kScaleRow);
        if (there == (kTile == 32 ? 0xffffffffu : 0xffffu)) return;
#pragma unroll
        for (int s = 0; s < kSub; ++s)
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (!(there >> (16 * s + key_pos(lane, i)) & 1)) vs[s][i] = 0.0f;
    }
    __device__ __forceinline__ void scores(float (&sc)[kSub][NB][2]) {
        const uint32_t base = stage == ring + 2 * kStage ? ring : stage + kStage;  // of the next tile
        uint32_t kr[kSub][2][kKW];
        float ks[kSub][2];
#pragma unroll
        for (int s = 0; s < kSub; ++s)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t src = base + at_k + (16 * s + 8 * i) * kRow;
                if constexpr (HD == 128) {
                    const uint4 x = lds16(src);
                    kr[s][i][0] = x.x, kr[s][i][1] = x.y, kr[s][i][2] = x.z, kr[s][i][3] = x.w;
                } else {
                    const uint2 x = lds8(src);
                    kr[s][i][0] = x.x, kr[s][i][1] = x.y;
                }
                ks[s][i] = lds_half(base + at_ks + (16 * s + 8 * i) * kScaleRow);
            }
        float c[kSub][NB][4], d[kSub][NB][4];  // two shorter chains
#pragma unroll
        for (int w = 0; w < kKW; ++w) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                const uint4 u = fragment(nb, w);
#pragma unroll
                for (int s = 0; s < kSub; ++s) {
                    const uint32_t x = kr[s][0][w], y = kr[s][1][w], x8 = x >> 8, y8 = y >> 8;
                    mma16816(c[s][nb], w == 0, codes_lo(x), codes_lo(y), codes_hi(x), codes_hi(y), u.x, u.y);
                    mma16816(d[s][nb], w == 0, codes_lo(x8), codes_lo(y8), codes_hi(x8), codes_hi(y8), u.z, u.w);
                }
            }
        }
        // lanes past the row's blocks hold zero sums
#pragma unroll
        for (int s = 0; s < kSub; ++s)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    float x = __fmaf_rn(c[s][nb][2 * i + 1] + d[s][nb][2 * i + 1], kLoInv, c[s][nb][2 * i] + d[s][nb][2 * i]) * ks[s][i];
                    x += __shfl_xor_sync(0xffffffffu, x, 1);
                    x += __shfl_xor_sync(0xffffffffu, x, 2);
                    sc[s][nb][i] = x * inv[nb];
                }
            }
    }
    // Element d of a row is code(d) times scale(d / 32).
    __device__ __forceinline__ static float code(const void *rows, long long row, int d) {
        const int byte = static_cast<const uint8_t *>(rows)[row * (HD / 2) + d / 32 * 16 + d % 16];
        return static_cast<float>((d % 32 < 16 ? byte & 15 : byte >> 4) - 8);
    }
    __device__ __forceinline__ static float scale(const __half *scales, long long row, int block) {
        return __half2float(scales[row * kBlocks + block]);
    }
    __device__ __forceinline__ void reset() { stage = ring, vlim = 5.9604644775390625e-08f, vinv = 16777216.0f; }  // 2^-24, 2^24
    // Whether a value scale of part s passes the bound of what a weight may be multiplied by.
    __device__ __forceinline__ bool value_range(int s) {
        return fmaxf(fabsf(vs[s][0]), fabsf(vs[s][1])) > vlim;
    }
    __device__ __forceinline__ void raise_value_range(float (&o)[NB][kO][4]) {
        float m = vlim;
#pragma unroll
        for (int s = 0; s < kSub; ++s)
            m = fmaxf(m, fmaxf(fabsf(vs[s][0]), fabsf(vs[s][1])));
        m = warp_max(m);
        if (!(m > vlim)) return;
        const int ex = min(((__float_as_int(m) >> 23) & 255) + 2, 127 + 18);  // a power of two above 2 m
        const float lim = __int_as_float(ex << 23);
        const float f = vlim * __int_as_float((254 - ex) << 23);
        vlim = lim, vinv = __int_as_float((254 - ex) << 23);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int j = 0; j < kO; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[nb][j][i] *= f;
    }
    __device__ __forceinline__ void values(const float (&w)[kSub][NB][2], float (&o)[NB][kO][4]) {
        uint32_t vr[kSub][4][kVW];
#pragma unroll
        for (int s = 0; s < kSub; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t src = stage + at_v + (16 * s + value_pos(0, i)) * kRow;
                if constexpr (HD == 128) {
                    const uint2 x = lds8(src);
                    vr[s][i][0] = x.x, vr[s][i][1] = x.y;
                } else {
                    vr[s][i][0] = lds4(src);
                }
            }
        uint32_t b[kSub][NB][2];
#pragma unroll
        for (int s = 0; s < kSub; ++s)  // w * scale / vlim <= 2^15; columns of no block are not used
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                split_half2(w[s][nb][0] * (vs[s][0] * vinv), w[s][nb][1] * (vs[s][1] * vinv), b[s][nb][0], b[s][nb][1]);
                b[s][nb][0] = transpose8(b[s][nb][0]);
                b[s][nb][1] = transpose8(b[s][nb][1]);
            }
#pragma unroll
        for (int i = 0; i < kVW; ++i) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                float even[NB][4], odd[NB][4];
#pragma unroll
                for (int s = 0; s < kSub; ++s) {
                    const uint32_t x = __byte_perm(vr[s][0][i], vr[s][1][i], u ? 0x7632 : 0x5410);
                    const uint32_t y = __byte_perm(vr[s][2][i], vr[s][3][i], u ? 0x7632 : 0x5410);
                    const uint32_t xl = codes_lo(x), xh = codes_hi(x), yl = codes_lo(y), yh = codes_hi(y);
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) mma16816(even[nb], s == 0, xl, xh, yl, yh, b[s][nb][0], b[s][nb][1]);
                    const uint32_t xl8 = codes_lo(x >> 8), xh8 = codes_hi(x >> 8), yl8 = codes_lo(y >> 8), yh8 = codes_hi(y >> 8);
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) mma16816(odd[nb], s == 0, xl8, xh8, yl8, yh8, b[s][nb][0], b[s][nb][1]);
                }
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int c = 0; c < 4; ++c) o[nb][4 * i + 2 * u][c] += even[nb][c], o[nb][4 * i + 2 * u + 1][c] += odd[nb][c];
            }
        }
    }
    // Lane (g, t) holds bytes [4 kVW g, + 4 kVW) of the row: elements of block
    // blk(g), low nibbles then high ones; the columns of that block are lane t == blk(g)'s.
    static constexpr int kRuns = 2, kRunLen = 4 * kVW;
    __device__ __forceinline__ bool owns(int lane) const { return (lane & 3) == (lane >> 2) * kBlocks / 8; }
    __device__ __forceinline__ static int head_of(int nb, int) { return nb; }
    __device__ __forceinline__ static int run_start(int run, int lane) {
        const int g = lane >> 2;
        return HD == 128 ? 32 * (g >> 1) + 8 * (g & 1) + 16 * run : 32 * (g >> 2) + 4 * (g & 3) + 16 * run;
    }
    __device__ __forceinline__ float element(const float (&o)[kO][4], int run, int i) const {
        const float *c = o[i];
        return (run ? __fmaf_rn(c[3], kLoInv, c[2]) : __fmaf_rn(c[1], kLoInv, c[0])) * vlim;
    }
};

// A key head's share of a row on the line of tiles: up to NH query heads.
struct Head {
    int row, head0, heads;     // query heads [head0, head0 + heads) of a row
    uint32_t first, n_tiles;   // its tiles on the line
};

constexpr int kMaxCluster = 8;  // no more than the slots of a CTA's pieces

// Two pieces a warp: one that began before its part of the line, one that goes on after it.
template <int HD, int NH>
struct PaSmem {
    static constexpr int kPieces = 2 * kPaWarps;
    float buf[kPaWarps][NH * HD];            // a warp's queries, then its outputs
    float bm[kPaWarps][NH], bl[kPaWarps][NH];
    float m[kPieces][NH], l[kPieces][NH];
    float o[kPieces][NH * HD];
    float cluster_m[kMaxCluster][NH], cluster_l[kMaxCluster][NH], cluster_o[kMaxCluster][NH * HD];  // of the cluster's CTAs, in its first
    float weight[kPieces][NH], sum_m[NH], sum_l[NH];  // of the pieces that are joined
    Head head[kPieces];
    int whole[kPieces];  // -1: no piece; bit 0: begins at the head's first tile, bit 1: ends at its last
    int scan[kPaWarps], longest[kPaWarps];
    Head join_head[2];
    int join_n[2], join_c0[2];  // pieces that this CTA, last to arrive, joins; the first one's CTA
};

constexpr int kMaxGrid = 640;

__device__ __forceinline__ float lse_of(float m, float l) { return l == 0.0f ? -INFINITY : (m - kHead + log2f(l)) * kLn2; }
__device__ __forceinline__ float inverse_of(float l) { return l == 0.0f ? 0.0f : __frcp_rn(l); }

constexpr uint32_t kJoinTiles = 4;
constexpr int kClusterTiles = 3;  // most tiles of a warp
constexpr int kJoinBatch = 16;  // pieces requested at a time

// Store to the same variable of the cluster's first CTA.
__device__ __forceinline__ void remote_store(float *p, float x) {
    uint32_t to;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(to) : "r"(smem_addr(p)));
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(x) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Release of the CTA's earlier writes (ordered by a barrier before it) and acquire of the others'.
__device__ __forceinline__ int arrive(int *p) {
    int v;
    asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(v) : "l"(p) : "memory");
    return v;
}

__device__ __forceinline__ int pa_len(const PagedAttnArgs &a, int row, int &req, bool &bad) {
    req = a.row_req ? a.row_req[row] : row;
    if (req < 0 || req >= a.n_req) {
        bad = true;
        req = 0;
        return 0;
    }
    // no more than the request holds: entries of the table past that are stale, pages that others may have
    const int held = a.lens[req], cap = static_cast<int>(a.max_blocks * a.page.d), most = min(max(held, 0), cap);
    const int len = a.row_len ? a.row_len[row] : held;
    bad |= held != most || len < 0 || len > most;
    return min(max(len, 0), most);
}

template <int HD, int NH>
constexpr size_t kFixedSmem = (sizeof(PaSmem<HD, NH>) + 15) / 16 * 16;

// A piece in global memory: [heads][HD] sums, then the maxima and the weights' sums; 16-byte multiples.
template <class R>
constexpr int pa_piece_floats = (R::kHeads * (R::HD + 2) + 3) / 4 * 4;

// The heads [head0, head0 + heads) of `row` that have NaN in them once more, over
// positions [p0, p1), from the formula, by one warp: their sums (dst), maxima and
// weights' sums.  The two parts of a factor are added as two products, and with
// an infinite key or value these can be of opposite signs, or 0 times infinity.
// Whatever that spoils ends as NaN (rows that hold NaN come here, too).  Sums in
// double: speed does not matter.  Looking for NaN costs a call of small heads 0.1 to
// 0.2 us of 8, 64 sessions of 16 tiles a head 0.4 of 47, long heads nothing.
template <class R, int ACT>
__device__ __noinline__ void exact_piece(const PagedAttnArgs &a, int row, int head0, int heads, int req, int p0, int p1,
                                         float *dst, float *dst_m, float *dst_l) {
    const int lane = threadIdx.x & 31;
    constexpr int HD = R::HD;
    const int *table = a.table + static_cast<long long>(req) * a.max_blocks;
    const int kh = head0 / a.group;
    auto row_of = [&](int p) -> long long {  // -1: not there
        if (p >= p1) return -1;
        const uint32_t b = fast_div(p, a.page), page = table[b];
        return page < static_cast<uint32_t>(a.n_pages) ? (page * a.n_kv_heads + kh) * a.page.d + (p - b * a.page.d) : -1ll;
    };
#pragma unroll 1
    for (int h = 0; h < heads; ++h, dst += HD) {
        __syncwarp();
        float sum = dst_l[h];  // NaN if an element is
#pragma unroll
        for (int i = 0; i < HD; i += 32) sum += dst[i + lane];
        if (!__any_sync(0xffffffffu, sum != sum)) continue;
        const long long q = row * a.q_stride + static_cast<long long>(head0 + h) * HD;
        auto score = [&](long long r) {
            double x = 0.0, block = 0.0;
#pragma unroll 1
            for (int d = 0; d < HD; ++d) {
                block += static_cast<double>(act_load<ACT>(a.q, q + d)) * static_cast<double>(R::code(a.k, r, d));
                if (d % 32 == 31) x += block * static_cast<double>(R::scale(a.k_scale, r, d / 32)), block = 0.0;
            }
            return static_cast<float>(x * static_cast<double>(a.qscale));
        };
        float m = -INFINITY;
#pragma unroll 1
        for (int p = p0 + lane; p < p1; p += 32) {
            const long long r = row_of(p);
            if (r >= 0) m = fmaxf(m, score(r));
        }
        m = warp_max(m);
        const float ref = m == -INFINITY ? 0.0f : m - kHead;
        double l = 0.0, o[HD / 32] = {};
#pragma unroll 1
        for (int first = p0; first < p1; first += 32) {
            const long long mine = row_of(first + lane);
            const float w_mine = mine >= 0 ? ex2(score(mine) - ref) : 0.0f;
            l += w_mine;
#pragma unroll 1
            for (int j = 0; j < 32; ++j) {
                const float w = __shfl_sync(0xffffffffu, w_mine, j);
                const long long r = __shfl_sync(0xffffffffu, mine, j);
                if (r < 0) continue;
#pragma unroll
                for (int i = 0; i < HD / 32; ++i)
                    o[i] += static_cast<double>(w) * static_cast<double>(R::code(a.v, r, lane + 32 * i) * R::scale(a.v_scale, r, i));
            }
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) dst[lane + 32 * i] = static_cast<float>(o[i]);
        if (lane == 0) dst_m[h] = m, dst_l[h] = static_cast<float>(l);
    }
}

template <class R, int ACT, bool kAligned>
__global__ void __launch_bounds__(kPaThreads, R::kMinCtas) paged_attn_kernel(const __grid_constant__ PagedAttnArgs a) {
    constexpr int HD = R::HD, NB = R::NB, NH = R::kHeads, kTile = 16 * R::kSub, kO = R::kO;
    using Smem = PaSmem<HD, NH>;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    Smem &S = *reinterpret_cast<Smem *>(smem_raw);
    char *ring = reinterpret_cast<char *>(smem_raw + kFixedSmem<HD, NH>);
    uint32_t *ends = reinterpret_cast<uint32_t *>(ring + kPaWarps * R::kRing);  // of rows 0..r
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int group = a.group;        // query heads of a key head
    const uint32_t units = a.units.d;  // of a row: key heads x groups of NH query heads
    bool bad = false;

    // ---- tiles of every row, summed; a head counts kHeadCost tiles more, for what it costs besides ----
    auto row_tiles = [&](int r) -> uint32_t {
        int req;
        const int len = pa_len(a, r, req, bad);
        const int start = a.window > 0 ? max(0, len - a.window) : 0;
        return len > start ? (len + kTile - 1) / kTile - start / kTile + R::kHeadCost : 0;
    };
    // A cluster a head (a.cluster CTAs, chosen by the launcher) or a line of tiles over all warps.
    const int cluster = a.cluster;
    int rank = 0, cluster_row = 0;
    uint32_t cluster_span = 0;
    if (cluster > 1) {
        cluster_arrive_relaxed();  // waited for before another CTA's shared memory is written
        rank = blockIdx.x % cluster;
        cluster_row = fast_div(blockIdx.x / cluster, a.units);
        cluster_span = row_tiles(cluster_row);
    }
    if (lane < 2) S.whole[2 * warp + lane] = -1;
    if (tid < 2) S.join_n[tid] = 0;
    // Up to 128 rows, in every warp: of rows 0 .. 4 lane + j, so that no warp waits for another.
    uint32_t my_end[4] = {};
    uint32_t longest = 0;
    const bool few = a.n_rows <= 128;
    if (cluster > 1) {
    } else if (few) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (4 * lane + j < a.n_rows) my_end[j] = row_tiles(4 * lane + j);
            longest = max(longest, my_end[j]);
        }
        longest = __reduce_max_sync(0xffffffffu, longest);
#pragma unroll
        for (int j = 1; j < 4; ++j) my_end[j] += my_end[j - 1];
        uint32_t before = my_end[3];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t x = __shfl_up_sync(0xffffffffu, before, o);
            if (lane >= o) before += x;
        }
        before -= my_end[3];
#pragma unroll
        for (int j = 0; j < 4; ++j) my_end[j] += before;
    } else {
        const int per_thread = (a.n_rows + kPaThreads - 1) / kPaThreads;
        const int r0 = tid * per_thread, r1 = min(a.n_rows, r0 + per_thread);
        uint32_t sum = 0;
#pragma unroll 1
        for (int r = r0; r < r1; ++r) {
            const uint32_t n = row_tiles(r);
            longest = max(longest, n);
            sum += n;
            ends[r] = sum;
        }
        longest = __reduce_max_sync(0xffffffffu, longest);
        uint32_t inc = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t x = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += x;
        }
        if (lane == 31) S.scan[warp] = inc;
        if (lane == 0) S.longest[warp] = longest;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kPaWarps; ++w) longest = max(longest, S.longest[w]);
        uint32_t before = inc - sum;
#pragma unroll
        for (int w = 0; w < kPaWarps - 1; ++w) before += w < warp ? S.scan[w] : 0;
        if (before)
#pragma unroll 1
            for (int r = r0; r < r1; ++r) ends[r] += before;
        __syncthreads();
    }
    if (bad) raise_error(a.status, kErrBadIndex);
    auto end_of = [&](int r) {
        if (!few) return ends[r];
        const uint32_t lo = r & 1 ? my_end[1] : my_end[0], hi = r & 1 ? my_end[3] : my_end[2];
        return __shfl_sync(0xffffffffu, r & 2 ? hi : lo, r >> 2);
    };
    uint32_t per = 0, u, u_end;
    bool apart = cluster > 1;
    if (apart) {
        u = blockIdx.x / cluster, u_end = u + 1;
        if (cluster_span == 0 && rank == 0) {  // a row without a position
            const int unit = u - cluster_row * units, kh = fast_div(unit, a.chunks), chunk = unit - kh * a.chunks.d;
            const int h0 = kh * group + chunk * NH, n = min(NH, group - chunk * NH);
            for (int i = tid; i < n * HD; i += kPaThreads)
                act_store<ACT>(a.out, cluster_row * a.out_stride + static_cast<long long>(h0) * HD + i, 0.0f);
            if (a.lse && tid < n) a.lse[static_cast<long long>(cluster_row) * a.n_heads + h0 + tid] = -INFINITY;
        }
    } else {
        const uint32_t total = end_of(a.n_rows - 1) * units;  // below 2^31 (checked by the entry point)
        per = max(1u, (total + gridDim.x * kPaWarps - 1) / (gridDim.x * kPaWarps));
        const uint32_t me = blockIdx.x * kPaWarps + warp;
        u = static_cast<uint32_t>(min(static_cast<unsigned long long>(total), static_cast<unsigned long long>(me) * per));
        u_end = u + min(per, total - u);
        // Few, short heads: a head a CTA, so that none waits for other CTAs.  Joining
        // through global memory takes about as long as kJoinTiles tiles one after another.
        const uint32_t warp_tiles = (longest + kPaWarps - 1) / kPaWarps;
        apart = static_cast<uint32_t>(a.n_rows) * units <= gridDim.x && warp_tiles <= per + kJoinTiles;
        if (apart) u = blockIdx.x, u_end = blockIdx.x < a.n_rows * units ? u + 1 : u;

        // rows without a position
#pragma unroll 1
        for (int r = blockIdx.x; r < a.n_rows; r += gridDim.x) {
            const uint32_t e0 = end_of(max(r - 1, 0)), e1 = end_of(r);
            if (e1 != (r ? e0 : 0)) continue;
#pragma unroll 1
            for (int i = tid; i < a.n_heads * HD; i += kPaThreads) act_store<ACT>(a.out, r * a.out_stride + i, 0.0f);
            if (a.lse)
#pragma unroll 1
                for (int h = tid; h < a.n_heads; h += kPaThreads) a.lse[static_cast<long long>(r) * a.n_heads + h] = -INFINITY;
        }
    }

    R R_(a, ring + warp * R::kRing, lane);
    float *buf = S.buf[warp];
#pragma unroll 1
    while (u < u_end) {
        // ---- the head that tile u belongs to ----
        int row;
        uint32_t row0, span, unit, from, to;  // [0, kHeadCost) of a head stands for its other costs, then come its tiles
        if (apart) {
            row = fast_div(u, a.units);
            unit = u - row * units;
            row0 = 0;
            u = u_end;
            if (cluster > 1) {
                span = cluster_span;
            } else {
                const uint32_t row_end = end_of(row), row_prev = end_of(max(row - 1, 0));
                span = row_end - (row ? row_prev : 0);
            }
            if (!span) break;
            const uint32_t warps = cluster * kPaWarps, n = (span - R::kHeadCost + warps - 1) / warps;
            from = min((rank * kPaWarps + warp) * n + R::kHeadCost, span), to = min(from + n, span);
        } else {
            const uint32_t q = fast_div(u, a.units);  // row tiles before u's: u / units lies in [row0, end)
            if (few) {
                row = 4 * __popc(__ballot_sync(0xffffffffu, my_end[3] <= q));  // below 4 * 32: q lies before the last row's end
#pragma unroll
                for (int j = 0; j < 3; ++j) row += __shfl_sync(0xffffffffu, my_end[j], row >> 2) <= q ? 1 : 0;
            } else {
                int lo = 0, hi = a.n_rows - 1;
#pragma unroll 1
                while (lo < hi) {
                    const int mid = (lo + hi) >> 1;
                    if (ends[mid] > q) hi = mid;
                    else lo = mid + 1;
                }
                row = lo;
            }
            const uint32_t row_end = end_of(row), row_prev = end_of(max(row - 1, 0));
            row0 = row ? row_prev : 0;
            span = row_end - row0;
            unit = (u - row0 * units) / span;
            from = u - row0 * units - unit * span, to = min(span, from + (u_end - u));
            u += to - from;
        }
        const int tile0 = max(static_cast<int>(from) - R::kHeadCost, 0), tile1 = static_cast<int>(to) - R::kHeadCost;
        if (tile1 <= tile0) continue;
        Head hd;
        hd.row = row;
        hd.n_tiles = span - R::kHeadCost;
        hd.first = row0 * units + unit * span + R::kHeadCost;
        const int kh = fast_div(unit, a.chunks), chunk = unit - kh * a.chunks.d;
        hd.head0 = kh * group + chunk * NH;
        hd.heads = min(NH, group - chunk * NH);
        int req;
        const int len = pa_len(a, row, req, bad);
        const int start = a.window > 0 ? max(0, len - a.window) : 0;
        const int pbase = start / kTile * kTile;

        constexpr uint32_t kNoPage = 0xffffffffu;  // an entry that is not a page of the cache
        const int *table = a.table + static_cast<long long>(req) * a.max_blocks;
        auto first_row = [&](int b) {  // of block b
            const uint32_t page = static_cast<uint32_t>(b) < static_cast<uint32_t>(a.max_blocks) ? table[b] : -1;
            return page < static_cast<uint32_t>(a.n_pages) ? (page * a.n_kv_heads + kh) * a.page.d : kNoPage;
        };
        // Ring, aligned: rows of position `walk` + 16 i, in lane i; else of blocks walk + i.
        int walk;
        uint32_t entry;
        auto refill = [&](int at) {
            walk = at;
            if constexpr (kAligned) {
                const int p = at + 16 * lane, b = fast_div(p, a.page);
                const uint32_t r = first_row(b);
                entry = r == kNoPage ? r : r + (p - b * a.page.d);
            } else {
                entry = first_row(at + lane);
            }
        };
        if (R::kRing > 0 || !kAligned) refill(kAligned ? pbase + tile0 * kTile : fast_div(max(start, pbase + tile0 * kTile), a.page));
        float o[NB][kO][4], m[NB], l[NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            m[nb] = -INFINITY, l[nb] = 0.0f;
#pragma unroll
            for (int j = 0; j < kO; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[nb][j][i] = 0.0f;
        }
        R_.reset();
        __syncwarp();  // the last head's outputs have been read from buf
        R_.template load_q<ACT>(a.q, row * a.q_stride + static_cast<long long>(hd.head0) * HD, hd.heads, a.qscale, buf, lane);
        Pos16<kAligned> P[R::kSub];
        constexpr uint32_t kAll = kTile == 32 ? 0xffffffffu : (1u << kTile) - 1;
        // Rows of the next tile, and which of its positions are attended to.
        // What is left out reads some row (row 0 in the place of an invalid page) and is masked later.
        auto locate = [&](int tile) {
            const int p0 = pbase + tile * kTile;
            uint32_t mask = kAll;
            if (p0 < start || p0 + kTile > len) {
                if (p0 < start) mask &= kAll << (start - p0);
                if (p0 + kTile > len) mask &= kAll >> (p0 + kTile - len);
            }
            if constexpr (kAligned) {
                if (p0 >= walk + 16 * 32) refill(p0);
                uint32_t top = 0;
#pragma unroll
                for (int s = 0; s < R::kSub; ++s) {
                    P[s].first = __shfl_sync(0xffffffffu, entry, (p0 - walk) / 16 + s);
                    top = max(top, P[s].first);
                }
                if (top == kNoPage) {
#pragma unroll
                    for (int s = 0; s < R::kSub; ++s) {
                        if (P[s].first != kNoPage) continue;
                        P[s].first = 0;
                        bad |= (mask >> (16 * s) & 0xffff) != 0;
                        mask &= ~(0xffffu << (16 * s));
                    }
                }
            } else {
                // lane i finds the row of the tile's position i (mod 16), the others get it from there
                const int p = p0 + (lane & (kTile - 1));
                const bool in = p >= start && p < len;
                const int b = fast_div(p, a.page);
                if (static_cast<int>(fast_div(min(p0 + kTile, len) - 1, a.page)) >= walk + 32) refill(fast_div(max(p0, start), a.page));
                const uint32_t base = __shfl_sync(0xffffffffu, entry, in ? b - walk : 0);
                const bool ok = in && base != kNoPage;
                bad |= in && !ok;
                const uint32_t r = ok ? base + (p - b * a.page.d) : 0;
                mask = __ballot_sync(0xffffffffu, ok) & kAll;
#pragma unroll
                for (int s = 0; s < R::kSub; ++s) {
                    P[s].mine = __shfl_sync(0xffffffffu, r, 16 * s + (lane & 15));
#pragma unroll
                    for (int i = 0; i < 2; ++i) P[s].k[i] = P[s].row(key_pos(lane, i));
#pragma unroll
                    for (int i = 0; i < 4; ++i) P[s].v[i] = P[s].row(value_pos(lane, i));
                }
            }
            return mask;
        };
        float sc[R::kSub][NB][2] = {};  // scores, then weights
        auto mask_scores = [&](uint32_t mask) {
            if (mask == kAll) return;
#pragma unroll
            for (int s = 0; s < R::kSub; ++s)
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        if (!(mask >> (16 * s + key_pos(lane, i)) & 1)) sc[s][nb][i] = -INFINITY;
        };
        // Scores to weights; raises the maximum, and with it rescales the sums, where a score passes it by too much.
        auto weigh = [&] {
            bool rise = false;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                float top = fmaxf(sc[0][nb][0], sc[0][nb][1]);
#pragma unroll
                for (int s = 1; s < R::kSub; ++s) top = fmaxf(top, fmaxf(sc[s][nb][0], sc[s][nb][1]));
                rise |= top > m[nb] + kSlack;
            }
            if constexpr (R::kRing > 0) {
#pragma unroll
                for (int s = 0; s < R::kSub; ++s) rise |= R_.value_range(s);
            }
            if (__any_sync(0xffffffffu, rise)) {
                if constexpr (R::kRing > 0) R_.raise_value_range(o);
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    float x = m[nb];
#pragma unroll
                    for (int s = 0; s < R::kSub; ++s) x = fmaxf(x, fmaxf(sc[s][nb][0], sc[s][nb][1]));
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
                    const float f = x == -INFINITY ? 1.0f : ex2(m[nb] - x);
                    m[nb] = x;
                    l[nb] *= f;
#pragma unroll
                    for (int j = 0; j < kO; ++j)
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[nb][j][i] *= f;
                }
            }
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                const float ref = m[nb] == -INFINITY ? 0.0f : m[nb] - kHead;
#pragma unroll
                for (int s = 0; s < R::kSub; ++s) {
                    sc[s][nb][0] = ex2(sc[s][nb][0] - ref);
                    sc[s][nb][1] = ex2(sc[s][nb][1] - ref);
                    l[nb] += sc[s][nb][0] + sc[s][nb][1];
                }
            }
        };
        uint32_t there = 0;  // positions attended to of the tile requested last
        if constexpr (R::kRing == 0) {
            // Step `tile` uses the rows requested in the step before and requests the next
            // tile's.  Aligned pages are walked here, by block and place in it, from entries
            // [b0, b0 + 32) of the block table, one a lane: rows found by locate() measured 270 us against 259.
            int block = fast_div(pbase + tile0 * kTile, a.page), b0 = block;
            uint32_t offset = pbase + tile0 * kTile - block * a.page.d;
            auto pages = [&] { return b0 + lane < a.max_blocks ? table[b0 + lane] : -1; };
            int page_of = kAligned ? pages() : 0;
#pragma unroll 1
            for (int tile = tile0 - 1; tile < tile1; ++tile) {
                const uint32_t now = there;
                if (now) {
#pragma unroll
                    for (int s = 0; s < R::kSub; ++s) R_.load_v(s, P[s]);
#pragma unroll
                    for (int s = 0; s < R::kSub; ++s) R_.scores(s, sc[s]);
                    mask_scores(now);
                }
                there = 0;
                if (tile + 1 < tile1) {
                    if constexpr (kAligned) {
                        const int p0 = pbase + (tile + 1) * kTile;
                        there = kAll;
                        if (p0 < start) there &= kAll << (start - p0);
                        if (p0 + kTile > len) there &= kAll >> (p0 + kTile - len);
#pragma unroll
                        for (int s = 0; s < R::kSub; ++s) {
                            if (block >= b0 + 32) b0 = block, page_of = pages();
                            const int page = __shfl_sync(0xffffffffu, page_of, block - b0);
                            const bool ok = static_cast<uint32_t>(page) < static_cast<uint32_t>(a.n_pages);
                            P[s].first = ok ? (static_cast<uint32_t>(page) * a.n_kv_heads + kh) * a.page.d + offset : 0;
                            if (!ok) {
                                bad |= (there >> (16 * s) & 0xffff) != 0;
                                there &= ~(0xffffu << (16 * s));
                            }
                            offset += 16;
                            if (offset == a.page.d) offset = 0, ++block;
                        }
                    } else {
                        there = locate(tile + 1);
                    }
#pragma unroll
                    for (int s = 0; s < R::kSub; ++s) R_.load_k(s, P[s]);
                }
                if (!now) continue;
                if (now != kAll) R_.clear_values(now, lane);
                weigh();
                R_.values(sc, o);
            }
        } else {
            // Step `tile` requests the rows of two tiles later, forms the next
            // tile's scores and adds its own values: two independent streams of arithmetic.
#pragma unroll 1
            for (int tile = tile0 - 2; tile < tile1; ++tile) {
                const uint32_t next = there;
                __syncwarp();  // the stage that is filled now was read in the last step
                if (tile + 2 < tile1) {
                    there = locate(tile + 2);
                    R_.request(P, lane);
                }
                R_.commit();
                const bool more = tile + 1 >= tile0 && tile + 1 < tile1;
                float w[R::kSub][NB][2];
#pragma unroll
                for (int s = 0; s < R::kSub; ++s)
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) w[s][nb][0] = sc[s][nb][0], w[s][nb][1] = sc[s][nb][1];
                R_.wait();
                if (more) R_.scores(sc);
                if (tile >= tile0) R_.values(w, o);
                R_.next();
                if (more) {
                    mask_scores(next);
                    R_.load_scales(next, lane);
                    weigh();
                }
            }
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) l[nb] += __shfl_xor_sync(0xffffffffu, l[nb], d);

        // ---- a piece stays in shared memory, a whole head goes out through it ----
        const bool begins = tile0 == 0, finishes = tile1 == static_cast<int>(hd.n_tiles), whole = begins && finishes;
        const int slot = 2 * warp + (begins ? 1 : 0);
        if (!whole && lane == 0) {
            S.head[slot] = hd;
            S.whole[slot] = (begins ? 1 : 0) | (finishes ? 2 : 0);
        }
        float *dst = whole ? buf : S.o[slot], *dst_m = whole ? S.bm[warp] : S.m[slot], *dst_l = whole ? S.bl[warp] : S.l[slot];
        __syncwarp();
        float sum = 0.0f;  // NaN if an element is
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const int h = R::head_of(nb, lane);
            if (h >= hd.heads) continue;
            sum += l[nb];
            if (R_.owns(lane)) {
#pragma unroll
                for (int run = 0; run < R::kRuns; ++run)
#pragma unroll
                    for (int i = 0; i < R::kRunLen; i += 4) {
                        const float4 x = make_float4(R_.element(o[nb], run, i), R_.element(o[nb], run, i + 1),
                                                     R_.element(o[nb], run, i + 2), R_.element(o[nb], run, i + 3));
                        *reinterpret_cast<float4 *>(dst + h * HD + R::run_start(run, lane) + i) = x;
                        sum += (x.x + x.y) + (x.z + x.w);
                    }
            }
            if (g == 0 && (R::kRing == 0 || t == 0)) dst_m[h] = m[nb], dst_l[h] = l[nb];
        }
        if (__any_sync(0xffffffffu, sum != sum))
            exact_piece<R, ACT>(a, row, hd.head0, hd.heads, req, max(start, pbase + tile0 * kTile),
                                min(len, pbase + tile1 * kTile), dst, dst_m, dst_l);
        __syncwarp();
        if (whole) {
            const long long out0 = row * a.out_stride + static_cast<long long>(hd.head0) * HD + lane;
#pragma unroll 1
            for (int h = 0; h < hd.heads; ++h) {
                const float f = inverse_of(dst_l[h]);
#pragma unroll
                for (int i = 0; i < HD; i += 32) act_store<ACT>(a.out, out0 + h * HD + i, buf[h * HD + i + lane] * f);
            }
            if (a.lse && lane < hd.heads)
                a.lse[static_cast<long long>(row) * a.n_heads + hd.head0 + lane] = lse_of(dst_m[lane], dst_l[lane]);
        }
    }
    if (bad) raise_error(a.status, kErrBadIndex);
    __syncthreads();

    // ---- pieces of one head, joined ----
    // A head's pieces in the CTA follow one another and end at the one that
    // finishes the head, or at the last.  What other CTAs hold too goes to
    // global memory; the last CTA to arrive puts all its parts back into the
    // slots and comes through here once more.
    constexpr int kPieceFloats = pa_piece_floats<R>;
    int joining = -1;  // 0, 1: the slots hold that head's parts; 2: those of the cluster's CTAs
    if (cluster > 1) cluster_wait();
    for (;;) {
        const int w = lane < Smem::kPieces ? S.whole[lane] : -1;
        uint32_t left = __ballot_sync(0xffffffffu, w >= 0);
        const uint32_t begin_bits = __ballot_sync(0xffffffffu, w >= 0 && (w & 1)),
                       finish_bits = __ballot_sync(0xffffffffu, w >= 0 && (w & 2));
        const uint32_t all = left;
        int open[2] = {-1, -1};  // first slot of a head that began in an earlier CTA, of one that begins here
#pragma unroll 1
        while (left) {
            const int first = __ffs(left) - 1;
            const uint32_t ends_at = finish_bits >> first << first;
            const int last = ends_at ? __ffs(ends_at) - 1 : 31 - __clz(left);
            left = left >> last >> 1 << last << 1;
            const bool begins = begin_bits >> first & 1, complete = begins && ends_at;
            const Head h = S.head[first];
            float *dst = a.part + (2 * blockIdx.x + (begins ? 1 : 0)) * kPieceFloats;
            const bool second = joining == 2;
            const uint32_t pieces = all & (0xffffffffu >> (31 - last)) & (0xffffffffu << first);
            const bool pair = __popc(pieces) <= 2;  // weighted by each thread for itself
            if (!pair && 4 * warp < NH) {  // what each piece counts: lane % 8 a piece, lane / 8 a head of four
                static_assert(Smem::kPieces == 8, "a head's pieces are 8 lanes'");
                const int k = lane & 7, hh = min(4 * warp + (lane >> 3), NH - 1);
                const bool there = pieces >> k & 1;
                const float m = there ? (second ? S.cluster_m[k][hh] : S.m[k][hh]) : -INFINITY;
                float top = m;
#pragma unroll
                for (int d = 1; d < 8; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                const float f = m == top ? 1.0f : ex2(m - top);
                float l = there ? f * (second ? S.cluster_l[k][hh] : S.l[k][hh]) : 0.0f;
#pragma unroll
                for (int d = 1; d < 8; d <<= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
                S.weight[k][hh] = f;
                if (k == 0) S.sum_m[hh] = top, S.sum_l[hh] = l;
            }
            if (!pair) __syncthreads();
            const float *o = second ? S.cluster_o[0] : S.o[0];
#pragma unroll 1
            for (int e = tid; e < h.heads * HD; e += kPaThreads) {
                const int hh = e / HD;
                float x = 0.0f, top, l;
                if (pair) {
                    const float m0 = second ? S.cluster_m[first][hh] : S.m[first][hh], m1 = second ? S.cluster_m[last][hh] : S.m[last][hh];
                    top = fmaxf(m0, m1);
                    const float f0 = m0 == top ? 1.0f : ex2(m0 - top), f1 = last == first ? 0.0f : m1 == top ? 1.0f : ex2(m1 - top);
                    l = f0 * (second ? S.cluster_l[first][hh] : S.l[first][hh]);
                    x = f0 * o[first * NH * HD + e];
                    if (last != first) {
                        l += f1 * (second ? S.cluster_l[last][hh] : S.l[last][hh]);
                        x += f1 * o[last * NH * HD + e];
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < Smem::kPieces; ++k)
                        if (pieces >> k & 1) x += S.weight[k][hh] * o[k * NH * HD + e];
                    top = S.sum_m[hh], l = S.sum_l[hh];
                }
                if (complete) {
                    act_store<ACT>(a.out, h.row * a.out_stride + static_cast<long long>(h.head0) * HD + e, x * inverse_of(l));
                    if (a.lse && e % HD == 0)
                        a.lse[static_cast<long long>(h.row) * a.n_heads + h.head0 + hh] = lse_of(top, l);
                } else if (cluster > 1) {
                    remote_store(&S.cluster_o[rank][e], x);
                    if (e % HD == 0) {
                        remote_store(&S.cluster_m[rank][hh], top);
                        remote_store(&S.cluster_l[rank][hh], l);
                    }
                } else {
                    __stcg(dst + e, x);
                    if (e % HD == 0) {
                        __stcg(dst + NH * HD + hh, top);
                        __stcg(dst + NH * HD + NH + hh, l);
                    }
                }
            }
            if (!pair) __syncthreads();
            if (!complete) open[begins ? 1 : 0] = first;
        }
        if (joining == 2) return;
        if (cluster > 1) {
            __syncwarp();
            cluster_sync();
            // the head's CTAs that had tiles: the first cluster_parts, all of them with one piece
            const uint32_t tiles = cluster_span ? cluster_span - R::kHeadCost : 0, warps = cluster * kPaWarps;
            const uint32_t cta_tiles = (tiles + warps - 1) / warps * kPaWarps;
            const int cluster_parts = tiles > cta_tiles ? (tiles + cta_tiles - 1) / cta_tiles : 1;
            if (rank || cluster_parts == 1) return;
            if (tid < Smem::kPieces)
                S.whole[tid] = tid < cluster_parts ? (tid == 0 ? 1 : 0) | (tid == cluster_parts - 1 ? 2 : 0) : -1;
            if (tid == 0) S.head[0] = S.head[1];  // its own first piece, which begins the head
            __syncthreads();
            joining = 2;
            continue;
        }
        if (joining < 0) {
            if (open[0] < 0 && open[1] < 0) return;
            __syncthreads();
            if (tid < 2 && open[tid] >= 0) {
                const Head h = S.head[open[tid]];
                const uint32_t cta_tiles = per * kPaWarps;
                const int c0 = h.first / cta_tiles, c1 = (h.first + h.n_tiles - 1) / cta_tiles;
                if (arrive(a.cnt + c0) == c1 - c0) {
                    a.cnt[c0] = 0;
                    S.join_n[tid] = c1 - c0 + 1;
                    S.join_c0[tid] = c0;
                }
            }
            // the heads move to where a second pass finds them
            if (tid == 2 && open[0] >= 0) S.join_head[0] = S.head[open[0]];
            if (tid == 3 && open[1] >= 0) S.join_head[1] = S.head[open[1]];
        }
        __syncthreads();
        do {
            if (++joining == 2) return;
        } while (!S.join_n[joining]);

        // ---- the last CTA to arrive: every part of the slots' columns joins a share of the pieces, in line order ----
        const int n = S.join_n[joining], c0 = S.join_c0[joining];
        const Head h = S.join_head[joining];
        const int cols = h.heads * (HD / 4);                   // of 4 elements
        const int parts = min(max(1, kPaThreads / cols), n);  // <= 8
        const int part = tid / cols;
        if (tid < Smem::kPieces) S.whole[tid] = tid < parts ? (tid == 0 ? 1 : 0) | (tid == parts - 1 ? 2 : 0) : -1;
        if (tid == 0) S.head[0] = h;
        if (part < parts) {
#pragma unroll 1
            for (int c = tid - part * cols; c < cols; c += kPaThreads) {
                const int hh = c / (HD / 4);
                float top = -INFINITY, l = 0.0f;
                float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
                for (int p0 = part; p0 < n; p0 += kJoinBatch * parts) {
                    float pm[kJoinBatch], pl[kJoinBatch];
                    float4 po[kJoinBatch];
#pragma unroll
                    for (int i = 0; i < kJoinBatch; ++i) {
                        const int p = p0 + i * parts;
                        pm[i] = -INFINITY, pl[i] = 0.0f, po[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        if (p < n) {
                            const float *src = a.part + (2 * (c0 + p) + (p == 0 ? 1 : 0)) * kPieceFloats;
                            pm[i] = __ldcg(src + NH * HD + hh);
                            pl[i] = __ldcg(src + NH * HD + NH + hh);
                            po[i] = __ldcg(reinterpret_cast<const float4 *>(src + 4 * c));
                        }
                    }
                    float now = top;
#pragma unroll
                    for (int i = 0; i < kJoinBatch; ++i) now = fmaxf(now, pm[i]);
                    const float f = top == now ? 1.0f : ex2(top - now);
                    top = now;
                    l *= f, o.x *= f, o.y *= f, o.z *= f, o.w *= f;
#pragma unroll
                    for (int i = 0; i < kJoinBatch; ++i) {
                        const float w = pm[i] == top ? 1.0f : ex2(pm[i] - top);
                        l += w * pl[i];
                        o.x += w * po[i].x, o.y += w * po[i].y, o.z += w * po[i].z, o.w += w * po[i].w;
                    }
                }
                *reinterpret_cast<float4 *>(&S.o[part][4 * c]) = o;
                if (c % (HD / 4) == 0) S.m[part][hh] = top, S.l[part][hh] = l;
            }
        }
        __syncthreads();
    }
}

constexpr int kMaxDevices = 64;

// CTAs of a launch on the current device: all that are resident at once, at
// most kMaxGrid (0: the kernel cannot run here).
template <class R, int ACT, bool kAligned>
cudaError_t pa_grid(int &grid) {
    static std::atomic<int> known[kMaxDevices];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < kMaxDevices && (grid = known[dev].load(std::memory_order_acquire)) > 0) return cudaSuccess;
    constexpr int smem = static_cast<int>(kFixedSmem<R::HD, R::kHeads> + kPaWarps * R::kRing + 4 * kPagedMaxRows);
    e = cudaFuncSetAttribute(paged_attn_kernel<R, ACT, kAligned>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    int sms = 0, per_sm = 0;
    if ((e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess) return e;
    if ((e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, paged_attn_kernel<R, ACT, kAligned>, kPaThreads,
                                                           smem - 4 * kPagedMaxRows + 4 * 512)) !=
        cudaSuccess)
        return e;
    grid = sms * per_sm < kMaxGrid ? sms * per_sm : kMaxGrid;
    if (grid <= 0) return cudaErrorInvalidConfiguration;
    if (dev < kMaxDevices) known[dev].store(grid, std::memory_order_release);
    return cudaSuccess;
}

template <class R>
constexpr size_t kScratch = (4 * kMaxGrid + 255) / 256 * 256 + sizeof(float) * kMaxGrid * 2 * pa_piece_floats<R>;

template <class R, int ACT, bool kAligned>
cudaError_t pa_launch(PagedAttnArgs &a, void *scratch, size_t scratch_bytes, cudaStream_t s) {
    int grid = 0;
    const cudaError_t e = pa_grid<R, ACT, kAligned>(grid);
    if (e != cudaSuccess) return e;
    if (scratch_bytes < kScratch<R>) return cudaErrorInvalidValue;
    a.group = a.n_heads / a.n_kv_heads;
    const int chunks = (a.group + R::kHeads - 1) / R::kHeads;
    a.chunks = make_fast_div(chunks);
    a.units = make_fast_div(a.n_kv_heads * chunks);
    a.cnt = static_cast<int *>(scratch);
    a.part = reinterpret_cast<float *>(static_cast<char *>(scratch) + (4 * kMaxGrid + 255) / 256 * 256);
    const size_t smem = kFixedSmem<R::HD, R::kHeads> + kPaWarps * R::kRing + 4 * a.n_rows;
    // Few heads of bounded length: a cluster a head, whose CTAs join through
    // shared memory instead of global memory (32 heads of 512 positions: 8.3 to 8.6 us
    // against 10.7).  As many CTAs as give a warp a tile, if 3 tiles a warp are enough and the
    // clusters find room at once: with all resident CTAs in clusters, 74 heads in
    // clusters of 4 took 19.3 us, not 11.6.  Pairs of CTAs (45 to 88 heads of 150 to
    // 380 positions): Q4_0 8.0 to 10.6 us against 8.6 to 10.7 on the line, 8 query heads of
    // 128 a key head in fp16 12 to 15 against 11 to 22.
    const long long heads = static_cast<long long>(a.n_rows) * a.units.d;
    const long long table = a.max_blocks * static_cast<long long>(a.page.d);
    const long long tiles = (a.window > 0 && a.window < table ? a.window : table) / (16 * R::kSub);
    a.cluster = 1;
    while (a.cluster < kMaxCluster && tiles > kPaWarps * a.cluster && heads * 2 * a.cluster * 5 <= grid * 3) a.cluster *= 2;
    if (tiles > kPaWarps * a.cluster * kClusterTiles) a.cluster = 1;
    if (a.cluster == 1) {
        paged_attn_kernel<R, ACT, kAligned><<<grid, kPaThreads, smem, s>>>(a);
        return cudaGetLastError();
    }
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = a.cluster, attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(heads * a.cluster));
    cfg.blockDim = dim3(kPaThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, paged_attn_kernel<R, ACT, kAligned>, a);
}

template <class R>
struct PaVariant {
    using Rows = R;
};

template <class F>
auto pa_variant(int head_dim, int kv_type, int group, F f) {
    // Query heads that share a key head are taken together as far as their sums fit the
    // registers: most of the work is on the codes (4 query heads of 128 a key
    // head, 64 sessions of 1500: 99 us one by one, 77 in pairs).
    if (kv_type == kKvQ4_0 && head_dim == 128)
        return group > 1 ? f(PaVariant<Q4Rows<128, 2>>{}) : f(PaVariant<Q4Rows<128, 1>>{});
    if (kv_type == kKvQ4_0)
        return group > 2 ? f(PaVariant<Q4Rows<64, 4>>{}) : group > 1 ? f(PaVariant<Q4Rows<64, 2>>{}) : f(PaVariant<Q4Rows<64, 1>>{});
    // up to 4 query heads of a key head fill one B operand, up to 8 two of them
    if (group <= 4) return head_dim == 128 ? f(PaVariant<F16Rows<128, 1>>{}) : f(PaVariant<F16Rows<64, 1>>{});
    return head_dim == 128 ? f(PaVariant<F16Rows<128, 2>>{}) : f(PaVariant<F16Rows<64, 2>>{});
}

}  // namespace

size_t paged_attention_scratch_bytes(int head_dim, int kv_type, int n_heads, int n_kv_heads) {
    return pa_variant(head_dim, kv_type, n_heads / n_kv_heads, [](auto r) { return kScratch<typename decltype(r)::Rows>; });
}

cudaError_t launch_paged_attention(PagedAttnArgs a, int head_dim, int kv_type, int act, void *scratch,
                                   size_t scratch_bytes, cudaStream_t s) {
    return pa_variant(head_dim, kv_type, a.n_heads / a.n_kv_heads, [&](auto r) {
        using R = typename decltype(r)::Rows;
        const bool aligned = a.page.d % 16 == 0;
        auto run = [&](auto type) {
            constexpr int kAct = decltype(type)::value;
            return aligned ? pa_launch<R, kAct, true>(a, scratch, scratch_bytes, s)
                           : pa_launch<R, kAct, false>(a, scratch, scratch_bytes, s);
        };
        if (act == BMO_ACT_F32) return run(std::integral_constant<int, BMO_ACT_F32>{});
        if (act == BMO_ACT_F16) return run(std::integral_constant<int, BMO_ACT_F16>{});
        return run(std::integral_constant<int, BMO_ACT_BF16>{});
    });
}

}  // namespace bmo
