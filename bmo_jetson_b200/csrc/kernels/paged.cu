// paged.cu -- bookkeeping and row traffic of the paged key-value cache: the
// plan of a step (pages, block table, slot numbers), the append of new rows
// and the read-back of stored ones.
//
// The rows are the ring's (kernels/attention.cu): fp16, or Q4_0 blocks of 32
// along head_dim as a nibble plane and an fp16 scale plane, so a page of one
// layer is a ring of page_size slots.
#include <cuda_bf16.h>

#include <cmath>
#include <type_traits>

#include "../paged.h"
#include "common.cuh"

namespace bmo {

FastDiv make_fast_div(uint32_t d) {
    FastDiv f{d, 0, 0};
    while ((1ull << f.shift) < d) ++f.shift;
    f.mul = static_cast<uint32_t>(((1ull << 32) * ((1ull << f.shift) - d)) / d + 1);
    return f;
}

namespace {

__device__ __forceinline__ uint32_t fast_div(uint32_t n, const FastDiv &f) {
    return (__umulhi(n, f.mul) + n) >> f.shift;
}

// ---- plan ----
//
// Request r of length L with n new positions grows to L' = L + n (0 when it
// ends, n < 0).  With nb(L) = ceil(L / ps) and F(L) = floor(max(0, L - window)
// / ps) (0 without a window) it takes pages for blocks [nb(L), nb(L')) and
// gives back blocks [F(L), F(L')), or all it holds, [F(L), nb(L)), when it
// ends.  Prefix sums over the requests place each of these in the ring of free
// pages and in the list of new positions.
//
// What bounds it is latency: a few dependent loads and block barriers over a
// few KB, so one CTA does all of it and no second launch follows, unless
// there are so many new positions that one SM would take longer than the
// launch (kPlanOneCta).  Every prefix sum is searched by the thread that
// writes an entry, so entries are written side by side whatever the requests'
// lengths are.
constexpr int kPlanThreads = 1024;
constexpr int kPlanOneCta = 8192;

struct PlanItem {
    int len, add, take, give, first;  // first: first block given back
    int after;
    bool ends;
};

struct PlanSums {
    long long take, give, add;
    int bad;
};

__device__ __forceinline__ PlanItem plan_item(const PagedPlanArgs &a, int r, int &bad) {
    const bmo_page_book &b = a.book;
    const int ps = b.page_size;
    const long long cap = static_cast<long long>(b.max_blocks) * ps;  // < 2^31
    PlanItem it{};
    it.len = b.lens[r];
    if (it.len < 0 || it.len > cap) {
        bad |= 1 << kErrBadIndex;
        it.len = 0;
        return it;
    }
    const int n = a.n_new[r];
    it.ends = n < 0;
    it.add = max(n, 0);
    if (it.add > cap - it.len) {
        bad |= 1 << kErrTableFull;
        it.add = 0;
    }
    it.after = it.ends ? 0 : it.len + it.add;
    const int have = (it.len + ps - 1) / ps;
    it.take = it.ends ? 0 : (it.after + ps - 1) / ps - have;
    it.first = b.window > 0 ? max(0, it.len - b.window) / ps : 0;
    const int last = it.ends ? have : (b.window > 0 ? max(0, it.after - b.window) / ps : 0);
    it.give = last - it.first;
    return it;
}

// Inclusive prefix sum over the CTA; `total` receives the whole sum.
__device__ __forceinline__ int block_scan(int v, int *warp_sums, int &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    __syncthreads();
    if (lane == 31) warp_sums[warp] = v;
    __syncthreads();
    int w = warp_sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += u;
    }
    total = __shfl_sync(0xffffffffu, w, 31);
    const int before = __shfl_sync(0xffffffffu, w, max(warp - 1, 0));
    return v + (warp ? before : 0);
}

// First index whose inclusive prefix sum exceeds i (ends[n - 1] > i).
__device__ __forceinline__ int owner(const int *ends, int n, int i) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (ends[mid] > i) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

__global__ void __launch_bounds__(kPlanThreads) plan_kernel(PagedPlanArgs a, int list_here) {
    __shared__ int warp_sums[32];
    __shared__ int s_end[kPlanThreads], s_len[kPlanThreads], s_first[kPlanThreads];
    __shared__ unsigned long long s_tot[3];
    __shared__ int s_bad;
    const bmo_page_book &b = a.book;
    const int tid = threadIdx.x, ps = b.page_size, n_pages = b.n_pages;
    const int head = b.state[0], count = b.state[1];

    // totals, and whether the step can be served
    if (tid < 3) s_tot[tid] = 0;
    if (tid == 0) s_bad = 0;
    __syncthreads();
    {
        PlanSums t{};
        for (int r = tid; r < b.n_req; r += kPlanThreads) {
            const PlanItem it = plan_item(a, r, t.bad);
            t.take += it.take;
            t.give += it.give;
            t.add += it.add;
        }
        if (t.take) atomicAdd(&s_tot[0], static_cast<unsigned long long>(t.take));
        if (t.give) atomicAdd(&s_tot[1], static_cast<unsigned long long>(t.give));
        if (t.add) atomicAdd(&s_tot[2], static_cast<unsigned long long>(t.add));
        if (t.bad) atomicOr(&s_bad, t.bad);
    }
    __syncthreads();
    const long long all_take = static_cast<long long>(s_tot[0]), all_give = static_cast<long long>(s_tot[1]),
                    all_add = static_cast<long long>(s_tot[2]);
    int bad = s_bad;
    if (!bad) {
        if (head < 0 || head >= n_pages || count < 0 || count > n_pages) bad |= 1 << kErrBadIndex;
        else if (all_take > count) bad |= 1 << kErrNoPages;
        // more pages given back than are in use: the table is not this ring's
        else if (count - all_take + all_give > n_pages) bad |= 1 << kErrBadIndex;
        if (all_add > a.max_tokens) bad |= 1 << kErrNoRoom;
    }
    const bool ok = bad == 0;
    const int n_add = ok ? static_cast<int>(all_add) : 0;

    // new pages and the list of new positions, kPlanThreads requests at a time
    if (ok) {
        int take0 = 0, add0 = 0;
        for (int r0 = 0; r0 < b.n_req; r0 += kPlanThreads) {
            const int r = r0 + tid, nr = min(kPlanThreads, b.n_req - r0);
            int ignore = 0, takes, adds;
            PlanItem it{};
            if (r < b.n_req) it = plan_item(a, r, ignore);
            const int take_end = block_scan(it.take, warp_sums, takes);
            const int add_end = block_scan(it.add, warp_sums, adds);
            s_end[tid] = take_end;
            s_len[tid] = it.len;
            __syncthreads();
            for (int i = tid; i < takes; i += kPlanThreads) {
                const int w = owner(s_end, nr, i);
                const int block = (s_len[w] + ps - 1) / ps + i - (w ? s_end[w - 1] : 0);
                const long long at = (static_cast<long long>(head) + take0 + i) % n_pages;
                b.table[static_cast<long long>(r0 + w) * b.max_blocks + block] = b.free_pages[at];
            }
            __syncthreads();
            if (r < b.n_req) a.offsets[r] = add0 + add_end - it.add;
            if (list_here) {
                s_end[tid] = add_end;
                __syncthreads();
                for (int i = tid; i < adds; i += kPlanThreads) {
                    const int w = owner(s_end, nr, i);
                    const int p = s_len[w] + i - (w ? s_end[w - 1] : 0);
                    const int page = b.table[static_cast<long long>(r0 + w) * b.max_blocks + p / ps];
                    a.slot[add0 + i] = page * ps + p % ps;
                    a.pos[add0 + i] = p;
                    a.req[add0 + i] = r0 + w;
                }
                __syncthreads();
            }
            take0 += takes;
            add0 += adds;
        }
    } else {
        for (int r = tid; r < b.n_req; r += kPlanThreads) a.offsets[r] = 0;
    }
    if (tid == 0) a.offsets[b.n_req] = n_add;
    if (list_here)
        for (int i = n_add + tid; i < a.max_tokens; i += kPlanThreads) a.slot[i] = a.pos[i] = a.req[i] = -1;
    __syncthreads();  // every page is taken before one is given back into the ring

    int give0 = 0;
    for (int r0 = 0; r0 < b.n_req; r0 += kPlanThreads) {
        const int r = r0 + tid, nr = min(kPlanThreads, b.n_req - r0);
        int ignore = 0, gives = 0;
        PlanItem it{};
        if (r < b.n_req) it = plan_item(a, r, ignore);
        if (ok && all_give) {
            s_end[tid] = block_scan(it.give, warp_sums, gives);
            s_first[tid] = it.first;
            __syncthreads();
            for (int i = tid; i < gives; i += kPlanThreads) {
                const int w = owner(s_end, nr, i);
                const int block = s_first[w] + i - (w ? s_end[w - 1] : 0);
                const long long at = (static_cast<long long>(head) + count + give0 + i) % n_pages;
                b.free_pages[at] = b.table[static_cast<long long>(r0 + w) * b.max_blocks + block];
            }
            __syncthreads();
            give0 += gives;
        }
        if (r < b.n_req) a.lens_out[r] = ok ? it.after : b.lens[r];
    }
    if (tid == 0) {
        a.state_out[0] = ok ? static_cast<int>((head + all_take) % n_pages) : head;
        a.state_out[1] = ok ? static_cast<int>(count - all_take + all_give) : count;
        a.state_out[2] = bad;
        a.state_out[3] = n_add;
    }
}

// The list of new positions alone, over all SMs, from the plan's offsets.
__global__ void plan_list_kernel(PagedPlanArgs a) {
    const bmo_page_book &b = a.book;
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= a.max_tokens) return;
    if (i >= a.offsets[b.n_req]) {
        a.slot[i] = a.pos[i] = a.req[i] = -1;
        return;
    }
    const int r = owner(a.offsets + 1, b.n_req, i);
    const int p = a.lens_out[r] - (a.offsets[r + 1] - i);
    const int page = b.table[static_cast<long long>(r) * b.max_blocks + p / b.page_size];
    a.slot[i] = page * b.page_size + p % b.page_size;
    a.pos[i] = p;
    a.req[i] = r;
}

// ---- activations of the three types, 4 elements at a time ----
//
// Raw: the 4 elements as loaded, so that many loads can be requested before
// the first is converted.  kVec: rows start on 4 elements' alignment.

struct Act32 {
    using T = float;
    using Raw = float4;
    template <bool kVec>
    static __device__ __forceinline__ Raw load(const T *p) {
        if constexpr (kVec) return __ldcs(reinterpret_cast<const float4 *>(p));
        else return make_float4(p[0], p[1], p[2], p[3]);
    }
    static __device__ __forceinline__ float4 value(Raw r) { return r; }
    template <bool kVec>
    static __device__ __forceinline__ void store(T *p, float4 x) {
        if constexpr (kVec) *reinterpret_cast<float4 *>(p) = x;
        else p[0] = x.x, p[1] = x.y, p[2] = x.z, p[3] = x.w;
    }
};
template <class Half>
struct IsBf16 {
    static constexpr bool value = false;
};
template <>
struct IsBf16<__nv_bfloat16> {
    static constexpr bool value = true;
};
template <class Half>
struct Act16 {
    using T = Half;
    using Raw = uint2;
    template <bool kVec>
    static __device__ __forceinline__ Raw load(const T *p) {
        if constexpr (kVec) return __ldcs(reinterpret_cast<const uint2 *>(p));
        const uint16_t *h = reinterpret_cast<const uint16_t *>(p);
        return make_uint2(h[0] | static_cast<uint32_t>(h[1]) << 16, h[2] | static_cast<uint32_t>(h[3]) << 16);
    }
    static __device__ __forceinline__ float4 value(Raw r) {
        if constexpr (IsBf16<T>::value)
            return make_float4(__uint_as_float(r.x << 16), __uint_as_float(r.x & 0xffff0000u), __uint_as_float(r.y << 16),
                               __uint_as_float(r.y & 0xffff0000u));
        const float2 x = __half22float2(*reinterpret_cast<const __half2 *>(&r.x)),
                     y = __half22float2(*reinterpret_cast<const __half2 *>(&r.y));
        return make_float4(x.x, x.y, y.x, y.y);
    }
    template <bool kVec>
    static __device__ __forceinline__ void store(T *p, float4 x) {
        Raw r;
        if constexpr (IsBf16<T>::value) {
            const __nv_bfloat162 a = __floats2bfloat162_rn(x.x, x.y), b = __floats2bfloat162_rn(x.z, x.w);
            r = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
        } else {
            const __half2 a = __floats2half2_rn(x.x, x.y), b = __floats2half2_rn(x.z, x.w);
            r = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
        }
        uint16_t *h = reinterpret_cast<uint16_t *>(p);
        if constexpr (kVec) *reinterpret_cast<uint2 *>(p) = r;
        else h[0] = r.x & 0xffff, h[1] = r.x >> 16, h[2] = r.y & 0xffff, h[3] = r.y >> 16;
    }
};
template <int ACT>
struct ActOf {
    using type = Act32;
};
template <>
struct ActOf<BMO_ACT_F16> {
    using type = Act16<__half>;
};
template <>
struct ActOf<BMO_ACT_BF16> {
    using type = Act16<__nv_bfloat16>;
};
template <int ACT>
using Act = typename ActOf<ACT>::type;

// ---- append ----
//
// Bound by its bytes when there are many rows, by latency for a frame of one
// position a session.  A lane holds 4 elements of a row, two rotated pairs, and
// the same 4 of every row it meets, so a warp that takes rows of one
// token needs each of the token's angles once, two a lane, in registers: cos
// and sin in double, rounded to fp32 as the exact-order step's table.  The rows' loads are
// requested kAppendRows at a time, the first ones before the angles are computed.
// Warps take few rows each when there are few tokens (launch_paged_append), all of
// a token's when there are many.
constexpr int kAppendThreads = 128;
constexpr int kAppendRows = 8;  // row slots of a lane in flight

// One Q4_0 block per 8 lanes, 4 consecutive values each: the same codes and
// scale as warp_store_q4_0.
__device__ __forceinline__ void group_store_q4_0(float4 x, uint8_t *qs_dst, __half *d_dst, bool live) {
    const int l = threadIdx.x & 7;
    const float v[4] = {x.x, x.y, x.z, x.w};
    float am = fabsf(v[0]), mx = v[0];
    int idx = 4 * l;
#pragma unroll
    for (int j = 1; j < 4; ++j)
        if (fabsf(v[j]) > am) { am = fabsf(v[j]); mx = v[j]; idx = 4 * l + j; }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) {
        const float oam = __shfl_xor_sync(0xffffffffu, am, o);
        const float omx = __shfl_xor_sync(0xffffffffu, mx, o);
        const int oidx = __shfl_xor_sync(0xffffffffu, idx, o);
        if (oam > am || (oam == am && oidx < idx)) { am = oam; mx = omx; idx = oidx; }
    }
    const float d = __fdiv_rn(mx, -8.0f);
    const float id = (d != 0.0f) ? __frcp_rn(d) : 0.0f;
    uint32_t code = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int q = min(15, __float2int_rz(__fadd_rn(__fmul_rn(v[j], id), 8.5f)));
        code |= static_cast<uint32_t>(q & 255) << (8 * j);
    }
    const uint32_t hi = __shfl_down_sync(0xffffffffu, code, 4);
    if (live && l < 4) reinterpret_cast<uint32_t *>(qs_dst)[l] = code | (hi << 4);
    if (live && l == 0) *d_dst = __float2half_rn(d);
}

template <int HD, bool Q4, int ACT, bool kVec>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const __grid_constant__ PagedAppendArgs a) {
    using A = Act<ACT>;
    using T = typename A::T;
    constexpr int kLanes = HD / 4, kWide = 32 / kLanes;  // lanes of a row, rows of a warp's access
    const int lane = threadIdx.x & 31;
    const long long item = static_cast<long long>(blockIdx.x) * (kAppendThreads / 32) + (threadIdx.x >> 5);
    const int token = static_cast<int>(item / a.parts), part = static_cast<int>(item - static_cast<long long>(token) * a.parts);
    if (token >= a.n) return;
    const int d = lane % kLanes * 4;
    const int n_rows = a.n_heads + 2 * a.n_kv_heads;
    const int end = min(n_rows, (part + 1) * a.part_rows);
    const T *q = static_cast<const T *>(a.q) + token * a.q_stride + d;
    const T *k = static_cast<const T *>(a.k) + token * a.k_stride + d;
    const T *v = static_cast<const T *>(a.v) + token * a.v_stride + d;
    T *qo = static_cast<T *>(a.q_out) + token * a.q_out_stride + d;

    int row0 = part * a.part_rows + lane / kLanes;
    typename A::Raw raw[kAppendRows];
    auto load = [&] {
#pragma unroll
        for (int i = 0; i < kAppendRows; ++i) {
            const int row = min(row0 + i * kWide, end - 1);
            const T *src = row < a.n_heads ? q + row * HD
                                           : row < a.n_heads + a.n_kv_heads ? k + (row - a.n_heads) * HD
                                                                            : v + (row - a.n_heads - a.n_kv_heads) * HD;
            raw[i] = A::template load<kVec>(src);
        }
    };
    load();
    const int slot = a.slot[token];
    float2 c0 = make_float2(1.0f, 0.0f), c1 = c0;
    if (a.rotate) {
        const float pos = static_cast<float>(a.pos[token]);
        double sn, cn;
        sincos(static_cast<double>(__fmul_rn(pos, a.inv_freq[d / 2])), &sn, &cn);
        c0 = make_float2(__double2float_rn(cn), __double2float_rn(sn));
        sincos(static_cast<double>(__fmul_rn(pos, a.inv_freq[d / 2 + 1])), &sn, &cn);
        c1 = make_float2(__double2float_rn(cn), __double2float_rn(sn));
    }
    const bool stored = slot >= 0 && slot < a.n_slots;
    if (part == 0 && lane == 0 && !stored && slot != -1) raise_error(a.status, kErrBadIndex);
    const uint32_t page = stored ? fast_div(slot, a.page) : 0;
    const uint32_t at = stored ? slot - page * a.page.d : 0;
    const long long row_of_page = static_cast<long long>(page) * a.n_kv_heads * a.page.d + at;
    for (;;) {
#pragma unroll
        for (int i = 0; i < kAppendRows; ++i) {
            const int row = row0 + i * kWide;
            const bool is_q = row < a.n_heads, is_v = row >= a.n_heads + a.n_kv_heads;
            const float4 x = A::value(raw[i]);
            float4 y = x;
            if (a.rotate && !is_v) {
                y.x = __fsub_rn(__fmul_rn(x.x, c0.x), __fmul_rn(x.y, c0.y));
                y.y = __fadd_rn(__fmul_rn(x.x, c0.y), __fmul_rn(x.y, c0.x));
                y.z = __fsub_rn(__fmul_rn(x.z, c1.x), __fmul_rn(x.w, c1.y));
                y.w = __fadd_rn(__fmul_rn(x.z, c1.y), __fmul_rn(x.w, c1.x));
            }
            if (is_q && row < end) A::template store<kVec>(qo + row * HD, y);
            const bool live = stored && !is_q && row < end;
            if constexpr (!Q4) {
                if (!live) continue;
            }
            const int h = row - a.n_heads - (is_v ? a.n_kv_heads : 0);
            const long long e = live ? (row_of_page + static_cast<long long>(h) * a.page.d) * HD + d : 0;
            void *cache = is_v ? a.v_cache : a.k_cache;
            if constexpr (Q4) {
                __half *scale = is_v ? a.v_scale : a.k_scale;
                group_store_q4_0(y, static_cast<uint8_t *>(cache) + (e & ~31ll) / 2, scale + e / 32, live);
            } else {
                Act<BMO_ACT_F16>::store<true>(static_cast<__half *>(cache) + e, y);
            }
        }
        row0 += kAppendRows * kWide;
        if (row0 - lane / kLanes >= end) break;
        load();
    }
}

// ---- read ----
//
// Bound by its bytes.  One CTA per row number; a thread turns 16 bytes of
// fp16 or 4 bytes of nibbles into 8 elements.
constexpr int kReadThreads = 256;

template <int HD, bool Q4, int ACT>
__global__ void __launch_bounds__(kReadThreads) read_kernel(const __grid_constant__ PagedReadArgs a) {
    using A = Act<ACT>;
    using T = typename A::T;
    constexpr int kPer = HD / 8;
    const int slot = a.slot[blockIdx.x];
    const bool stored = slot >= 0 && slot < a.n_slots;
    if (threadIdx.x == 0 && !stored && slot != -1) raise_error(a.status, kErrBadIndex);
    const uint32_t page = stored ? fast_div(slot, a.page) : 0;
    const uint32_t at = stored ? slot - page * a.page.d : 0;
    const int items = a.n_kv_heads * kPer;
    const long long out0 = static_cast<long long>(blockIdx.x) * a.n_kv_heads * HD;
#pragma unroll 4
    for (int i = threadIdx.x; i < 2 * items; i += blockDim.x) {
        const bool is_v = i >= items;
        const int j = is_v ? i - items : i;
        const int h = j / kPer, c = j % kPer;
        const long long row = (static_cast<long long>(page) * a.n_kv_heads + h) * a.page.d + at;
        const void *cache = is_v ? a.v_cache : a.k_cache;
        T *out = static_cast<T *>(is_v ? a.v_out : a.k_out) + out0 + h * HD;
        float4 lo = make_float4(0.0f, 0.0f, 0.0f, 0.0f), hi = lo;
        if constexpr (Q4) {
            if (stored) {
                const uint32_t w = __ldg(reinterpret_cast<const uint32_t *>(static_cast<const uint8_t *>(cache) + row * (HD / 2)) + c);
                const float s = __half2float(__ldg((is_v ? a.v_scale : a.k_scale) + row * (HD / 32) + c / 4));
                float n[8];
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    n[b] = __fmul_rn(static_cast<float>(static_cast<int>(w >> (8 * b) & 15) - 8), s);
                    n[4 + b] = __fmul_rn(static_cast<float>(static_cast<int>(w >> (8 * b + 4) & 15) - 8), s);
                }
                lo = make_float4(n[0], n[1], n[2], n[3]);
                hi = make_float4(n[4], n[5], n[6], n[7]);
            }
            T *o = out + c / 4 * 32 + c % 4 * 4;
            A::template store<true>(o, lo);
            A::template store<true>(o + 16, hi);
        } else {
            if (stored) {
                const uint4 u = __ldg(reinterpret_cast<const uint4 *>(static_cast<const __half *>(cache) + row * HD) + c);
                const __half2 *p = reinterpret_cast<const __half2 *>(&u);
                const float2 f0 = __half22float2(p[0]), f1 = __half22float2(p[1]), f2 = __half22float2(p[2]),
                             f3 = __half22float2(p[3]);
                lo = make_float4(f0.x, f0.y, f1.x, f1.y);
                hi = make_float4(f2.x, f2.y, f3.x, f3.y);
            }
            A::template store<true>(out + 8 * c, lo);
            A::template store<true>(out + 8 * c + 4, hi);
        }
    }
}

template <int HD, bool Q4>
cudaError_t append_act(PagedAppendArgs a, int act, cudaStream_t s) {
    // Rows of a warp: one round of loads, or more rounds (fewer angles computed
    // twice) once the warps are many: 32 an SM keep its loads in flight.
    constexpr int kRound = kAppendRows * (128 / HD), kManyWarps = 148 * 32;
    const int rows = a.n_heads + 2 * a.n_kv_heads;
    const long long rounds = static_cast<long long>(a.n) * ((rows + kRound - 1) / kRound);
    const int per = static_cast<int>(rounds / kManyWarps < 1 ? 1 : rounds / kManyWarps);
    a.part_rows = per * kRound < rows ? per * kRound : rows;
    a.parts = (rows + a.part_rows - 1) / a.part_rows;
    const long long warps = static_cast<long long>(a.n) * a.parts;
    const long long grid = (warps + kAppendThreads / 32 - 1) / (kAppendThreads / 32);
    if (grid > 0x7fffffff) return cudaErrorInvalidValue;
    const unsigned g = static_cast<unsigned>(grid);
    auto run = [&](auto type) {
        constexpr int kAct = decltype(type)::value;
        using T = typename Act<kAct>::T;
        auto vec = [&](const void *p, long long stride) {
            return reinterpret_cast<uintptr_t>(p) % (4 * sizeof(T)) == 0 && (a.n == 1 || stride % 4 == 0);
        };
        if (vec(a.k, a.k_stride) && vec(a.v, a.v_stride) &&
            (!a.n_heads || (vec(a.q, a.q_stride) && vec(a.q_out, a.q_out_stride))))
            append_kernel<HD, Q4, kAct, true><<<g, kAppendThreads, 0, s>>>(a);
        else
            append_kernel<HD, Q4, kAct, false><<<g, kAppendThreads, 0, s>>>(a);
    };
    if (act == BMO_ACT_F32) run(std::integral_constant<int, BMO_ACT_F32>{});
    else if (act == BMO_ACT_F16) run(std::integral_constant<int, BMO_ACT_F16>{});
    else run(std::integral_constant<int, BMO_ACT_BF16>{});
    return cudaGetLastError();
}

template <int HD, bool Q4>
cudaError_t read_act(const PagedReadArgs &a, int act, cudaStream_t s) {
    const int items = 2 * a.n_kv_heads * (HD / 8);
    const int threads = items < kReadThreads ? (items + 31) / 32 * 32 : kReadThreads;
    if (act == BMO_ACT_F32) read_kernel<HD, Q4, BMO_ACT_F32><<<a.n, threads, 0, s>>>(a);
    else if (act == BMO_ACT_F16) read_kernel<HD, Q4, BMO_ACT_F16><<<a.n, threads, 0, s>>>(a);
    else read_kernel<HD, Q4, BMO_ACT_BF16><<<a.n, threads, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_paged_plan(const PagedPlanArgs &a, cudaStream_t s) {
    const int list_here = a.max_tokens <= kPlanOneCta;
    plan_kernel<<<1, kPlanThreads, 0, s>>>(a, list_here);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess || list_here) return e;
    plan_list_kernel<<<(a.max_tokens + 255) / 256, 256, 0, s>>>(a);
    return cudaGetLastError();
}

cudaError_t launch_paged_append(const PagedAppendArgs &a, int head_dim, int kv_type, int act, cudaStream_t s) {
    if (head_dim == 128)
        return kv_type == kKvQ4_0 ? append_act<128, true>(a, act, s) : append_act<128, false>(a, act, s);
    return kv_type == kKvQ4_0 ? append_act<64, true>(a, act, s) : append_act<64, false>(a, act, s);
}

cudaError_t launch_paged_read(const PagedReadArgs &a, int head_dim, int kv_type, int act, cudaStream_t s) {
    if (head_dim == 128) return kv_type == kKvQ4_0 ? read_act<128, true>(a, act, s) : read_act<128, false>(a, act, s);
    return kv_type == kKvQ4_0 ? read_act<64, true>(a, act, s) : read_act<64, false>(a, act, s);
}

}  // namespace bmo
