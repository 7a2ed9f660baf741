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

// Granlund and Montgomery, "Division by invariant integers using multiplication" (1994).
FastDiv make_fast_div(uint32_t d) {
    FastDiv f{d, 0, 0};
    while ((1ull << f.shift) < d) ++f.shift;
    f.mul = static_cast<uint32_t>(((1ull << 32) * ((1ull << f.shift) - d)) / d + 1);
    return f;
}

namespace {

// ---- plan ----
//
// Request r of length L with n new positions grows to L' = L + n (0 when it
// ends, n < 0).  With nb(L) = ceil(L / ps) and F(L) = floor(max(0, L - window)
// / ps) (0 without a window) it takes pages for blocks [nb(L), nb(L')) and
// gives back blocks [F(L), F(L')), or all it holds, [F(L), nb(L)), when it
// ends.  Prefix sums over the requests place each of these in the ring of free
// pages and in the list of new positions.
//
// Lengths and state can go to other buffers than they come from, so the caller
// may drop a plan and make it, or another, again from the old ones.  Table
// cells before nb(L) are not written, later ones are stale, so the table needs
// nothing for that; but pages given back past the ring's end overwrite its
// first entries, those that the step takes.  Their earlier pages are kept in
// book.undo, and a plan that begins at the same state reads them from there.
//
// What bounds it is latency: a few dependent loads and block barriers over a
// few KB, so one CTA does all of it and no second launch follows, unless
// there are so many new positions that one SM would take longer than the
// launch (kPlanOneCta).  Where no request has more than kFew of anything, the usual
// step, each thread writes what its request has.  Otherwise the thread that writes
// an entry searches the prefix sums for its request, so entries are written
// side by side whatever the requests' lengths are, kPlanBatch of a thread's in
// flight.  64 requests of one position: 3.9 us, of which about 2 are the launch; 61
// requests of up to 2999 new positions, made again over a dropped plan, both
// kernels: 12.8 to 13.4 us.
constexpr int kPlanThreads = 1024;
constexpr int kPlanOneCta = 8192;
constexpr int kFew = 2;
constexpr int kPlanBatch = 4;

struct PlanItem {
    int len, have;          // positions and pages before the step
    uint32_t add, take, give;
    int first;              // first block given back
    int after;              // positions after the step
};

__device__ __forceinline__ PlanItem plan_item(const PagedPlanArgs &a, int r, int &bad) {
    const bmo_page_book &b = a.book;
    const int ps = b.page_size;
    const long long cap = static_cast<long long>(b.max_blocks) * ps;  // < 2^31
    PlanItem it{};
    it.len = b.lens[r];
    const int n = a.n_new[r];
    if (it.len < 0 || it.len > cap) {
        bad |= 1 << kErrBadIndex;
        it.len = 0;
        return it;
    }
    it.add = max(n, 0);
    if (it.add > cap - it.len) {
        bad |= 1 << kErrTableFull;
        it.add = 0;
    }
    it.after = n < 0 ? 0 : it.len + it.add;
    it.have = (it.len + ps - 1) / ps;
    it.take = n < 0 ? 0 : (it.after + ps - 1) / ps - it.have;
    it.first = b.window > 0 ? max(0, it.len - b.window) / ps : 0;
    it.give = (n < 0 ? it.have : b.window > 0 ? max(0, it.after - b.window) / ps : 0) - it.first;
    return it;
}

// Sums below 2^31 exactly, larger ones as 2^31 - 1 (no step is that large).
__device__ __forceinline__ uint32_t add_sat(uint32_t x, uint32_t y) { return min(x + y, 0x7fffffffu); }

struct PlanSums {
    uint32_t take, give, add;
};
__device__ __forceinline__ PlanSums operator+(PlanSums x, PlanSums y) {
    return {add_sat(x.take, y.take), add_sat(x.give, y.give), add_sat(x.add, y.add)};
}
__device__ __forceinline__ PlanSums shfl_up(PlanSums x, int d) {
    return {__shfl_up_sync(0xffffffffu, x.take, d), __shfl_up_sync(0xffffffffu, x.give, d), __shfl_up_sync(0xffffffffu, x.add, d)};
}

// Inclusive prefix sums over the CTA; `total` receives the whole sums.
__device__ __forceinline__ PlanSums block_scan(PlanSums v, PlanSums *warp_sums, PlanSums &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const PlanSums u = shfl_up(v, o);
        if (lane >= o) v = v + u;
    }
    __syncthreads();
    if (lane == 31) warp_sums[warp] = v;
    __syncthreads();
    PlanSums w = warp_sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const PlanSums u = shfl_up(w, o);
        if (lane >= o) w = w + u;
    }
    auto from = [&](int l) {
        return PlanSums{__shfl_sync(0xffffffffu, w.take, l), __shfl_sync(0xffffffffu, w.give, l), __shfl_sync(0xffffffffu, w.add, l)};
    };
    total = from(31);
    const PlanSums before = from(max(warp - 1, 0));
    return warp ? v + before : v;
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

// For entries i < n of this CTA: read(i, request, number within the request)
// of up to kPlanBatch of a thread's entries, then write(i, what was read).
template <class T, class Read, class Write>
__device__ __forceinline__ void plan_fill(const int *ends, int n_req, int n, Read read, Write write) {
    for (int i0 = threadIdx.x; i0 < n; i0 += kPlanBatch * kPlanThreads) {
        T got[kPlanBatch];
#pragma unroll
        for (int k = 0; k < kPlanBatch; ++k) {
            const int i = i0 + k * kPlanThreads;
            if (i >= n) continue;
            const int w = owner(ends, n_req, i);
            got[k] = read(i, w, i - (w ? ends[w - 1] : 0));
        }
#pragma unroll
        for (int k = 0; k < kPlanBatch; ++k)
            if (i0 + k * kPlanThreads < n) write(i0 + k * kPlanThreads, got[k]);
    }
}

struct PlanCell {
    long long at;
    int page;
};
struct PlanToken {
    int slot, pos, req;
};

__global__ void __launch_bounds__(kPlanThreads) plan_kernel(PagedPlanArgs a, int list_here) {
    __shared__ PlanSums warp_sums[32];
    __shared__ int s_end[kPlanThreads], s_len[kPlanThreads], s_first[kPlanThreads];
    __shared__ unsigned long long s_tot[3];
    __shared__ int s_bad;
    const bmo_page_book &b = a.book;
    const int tid = threadIdx.x, ps = b.page_size, n_pages = b.n_pages;
    const int head = b.state[0], count = b.state[1];
    // the ring entries that the last plan has overwritten, if it began at this state
    int *const kept = b.undo ? b.undo + 4 : nullptr, *const written = b.undo ? kept + n_pages : nullptr;
    int redo = 0;
    if (b.undo) {  // loaded together: the start is a chain of loads as it is
        const int head0 = b.undo[0], count0 = b.undo[1], n = b.undo[2];
        if (head0 == head && count0 == count) redo = n;
    }
    const bool one = b.n_req <= kPlanThreads;  // each thread has one request at most

    // ---- totals, and whether the step can be served ----
    PlanItem it{};
    PlanSums end{}, total{};
    int bad = 0, old_page = -1;
    long long all_take, all_give, all_add;
    if (one) {
        if (tid < b.n_req) {
            it = plan_item(a, tid, bad);
            // the page that the request's next position lies in, unless that begins a page
            if (it.add && it.len % ps) old_page = b.table[static_cast<long long>(tid) * b.max_blocks + it.len / ps];
        }
        end = block_scan({it.take, it.give, it.add}, warp_sums, total);
        all_take = total.take, all_give = total.give, all_add = total.add;
        if (tid == 0) s_bad = 0;
        __syncthreads();
        if (bad) atomicOr(&s_bad, bad);
    } else {
        if (tid < 3) s_tot[tid] = 0;
        if (tid == 0) s_bad = 0;
        __syncthreads();
        unsigned long long t[3] = {};
        for (int r = tid; r < b.n_req; r += kPlanThreads) {
            const PlanItem x = plan_item(a, r, bad);
            t[0] += x.take, t[1] += x.give, t[2] += x.add;
        }
        for (int i = 0; i < 3; ++i)
            if (t[i]) atomicAdd(&s_tot[i], t[i]);
        if (bad) atomicOr(&s_bad, bad);
        __syncthreads();
        all_take = s_tot[0], all_give = s_tot[1], all_add = s_tot[2];
    }
    const bool few = __syncthreads_and(one && it.take <= kFew && it.give <= kFew && it.add <= kFew);
    bad = s_bad;
    if (!bad) {
        if (head < 0 || head >= n_pages || count < 0 || count > n_pages) bad |= 1 << kErrBadIndex;
        else if (all_take > count) bad |= 1 << kErrNoPages;
        // more pages given back than are in use: the table is not this ring's
        else if (count - all_take + all_give > n_pages) bad |= 1 << kErrBadIndex;
        if (all_add > a.max_tokens) bad |= 1 << kErrNoRoom;
    }
    const bool ok = bad == 0;
    const int n_add = ok ? static_cast<int>(all_add) : 0;
    auto ring_at = [&](long long i) {  // i <= count + all_give <= 2 n_pages
        long long at = head + i;
        if (at >= n_pages) at -= n_pages;
        if (at >= n_pages) at -= n_pages;
        return at;
    };
    auto cell = [&](int r, int block) { return static_cast<long long>(r) * b.max_blocks + block; };
    if (!ok || redo < 0 || redo > n_pages) redo = 0;
    if (redo) {  // the plan was dropped, unless the caller has written the ring anew
        bool same = true;
        for (int i = tid; i < redo; i += kPlanThreads) same &= b.free_pages[ring_at(i)] == written[i];
        if (!__syncthreads_and(same)) redo = 0;
    }
    auto take_page = [&](long long i) { return i < redo ? kept[i] : b.free_pages[ring_at(i)]; };
    auto give_page = [&](long long i, int page) {  // i-th given back; every page has been taken
        const long long over = count + i - n_pages;  // past the end: the entry of the ring's start
        if (over >= 0 && b.undo) {
            if (over >= redo) kept[over] = b.free_pages[ring_at(over)];
            written[over] = page;
        }
        b.free_pages[ring_at(count + i)] = page;
    };

    if (few && ok) {
        const int r = tid;
        int taken[kFew] = {-1, -1};
#pragma unroll
        for (int j = 0; j < kFew; ++j)
            if (j < it.take) {
                taken[j] = take_page(end.take - it.take + j);
                b.table[cell(r, it.have + j)] = taken[j];
            }
        int given[kFew];
#pragma unroll
        for (int j = 0; j < kFew; ++j)
            if (j < it.give) {
                const int block = it.first + j;
                given[j] = block >= it.have ? taken[block - it.have ? 1 : 0] : b.table[cell(r, block)];
            }
#pragma unroll
        for (int j = 0; j < kFew; ++j)
            if (j < it.add) {
                const int p = it.len + j, i = end.add - it.add + j, block = p / ps;
                const int page = block < it.have ? old_page : taken[block - it.have ? 1 : 0];
                if (list_here) a.slot[i] = page * ps + (p - block * ps), a.pos[i] = p, a.req[i] = r;
            }
        if (r < b.n_req) a.offsets[r] = end.add - it.add;
        __syncthreads();  // every page is taken before one is given back into the ring
#pragma unroll
        for (int j = 0; j < kFew; ++j)
            if (j < it.give) give_page(end.give - it.give + j, given[j]);
        if (r < b.n_req) a.lens_out[r] = it.after;
    } else {
        // new pages and the list of new positions, kPlanThreads requests at a time
        long long take0 = 0;
        int add0 = 0;
        for (int r0 = 0; ok && r0 < b.n_req; r0 += kPlanThreads) {
            const int r = r0 + tid, nr = min(kPlanThreads, b.n_req - r0);
            if (!one) {
                int ignore = 0;
                it = r < b.n_req ? plan_item(a, r, ignore) : PlanItem{};
                end = block_scan({it.take, it.give, it.add}, warp_sums, total);
            }
            s_end[tid] = end.take;
            s_len[tid] = it.len;
            __syncthreads();
            plan_fill<PlanCell>(
                s_end, nr, total.take,
                [&](int i, int w, int j) {
                    return PlanCell{cell(r0 + w, (s_len[w] + ps - 1) / ps + j), take_page(take0 + i)};
                },
                [&](int, PlanCell c) { b.table[c.at] = c.page; });
            __syncthreads();
            if (r < b.n_req) a.offsets[r] = add0 + static_cast<int>(end.add - it.add);
            if (list_here) {
                s_end[tid] = end.add;
                __syncthreads();
                plan_fill<PlanToken>(
                    s_end, nr, total.add,
                    [&](int, int w, int j) {
                        const int p = s_len[w] + j;
                        return PlanToken{b.table[cell(r0 + w, p / ps)] * ps + p % ps, p, r0 + w};
                    },
                    [&](int i, PlanToken t) { a.slot[add0 + i] = t.slot, a.pos[add0 + i] = t.pos, a.req[add0 + i] = t.req; });
                __syncthreads();
            }
            take0 += total.take;
            add0 += total.add;
        }
        if (!ok)
            for (int r = tid; r < b.n_req; r += kPlanThreads) a.offsets[r] = 0;
        __syncthreads();  // every page is taken before one is given back into the ring
        long long give0 = 0;
        for (int r0 = 0; r0 < b.n_req; r0 += kPlanThreads) {
            const int r = r0 + tid, nr = min(kPlanThreads, b.n_req - r0);
            if (!one && ok) {
                int ignore = 0;
                it = r < b.n_req ? plan_item(a, r, ignore) : PlanItem{};
                end = block_scan({it.take, it.give, it.add}, warp_sums, total);
            }
            if (ok && all_give) {
                s_end[tid] = end.give;
                s_first[tid] = it.first;
                __syncthreads();
                plan_fill<int>(
                    s_end, nr, total.give, [&](int, int w, int j) { return b.table[cell(r0 + w, s_first[w] + j)]; },
                    [&](int i, int page) { give_page(give0 + i, page); });
                __syncthreads();
                give0 += total.give;
            }
            if (r < b.n_req) a.lens_out[r] = ok ? it.after : b.lens[r];
        }
    }
    // entries that the dropped plan has overwritten and this one has not
    const int over = ok ? static_cast<int>(max(0ll, count + all_give - n_pages)) : 0;
    for (int i = over + tid; i < redo; i += kPlanThreads) b.free_pages[ring_at(i)] = kept[i];
    if (tid == 0) a.offsets[b.n_req] = n_add;
    if (list_here)
        for (int i = n_add + tid; i < a.max_tokens; i += kPlanThreads) a.slot[i] = a.pos[i] = a.req[i] = -1;
    if (tid == 0) {
        a.state_out[0] = ok ? static_cast<int>(ring_at(all_take)) : head;
        a.state_out[1] = ok ? static_cast<int>(count - all_take + all_give) : count;
        a.state_out[2] = bad;
        a.state_out[3] = n_add;
        if (ok && b.undo) b.undo[0] = head, b.undo[1] = count, b.undo[2] = over;
    }
}

// The list of new positions alone, over all SMs, from the plan's offsets.
constexpr int kListThreads = 256;
constexpr int kListStaged = 2048;  // offsets kept in shared memory

__global__ void __launch_bounds__(kListThreads) plan_list_kernel(PagedPlanArgs a) {
    __shared__ int s_ends[kListStaged];
    const bmo_page_book &b = a.book;
    pdl_wait();
    const bool staged = b.n_req <= kListStaged;
    if (staged) {
        for (int r = threadIdx.x; r < b.n_req; r += kListThreads) s_ends[r] = a.offsets[r + 1];
        __syncthreads();
    }
    const int *ends = staged ? s_ends : a.offsets + 1;
    const int i = blockIdx.x * kListThreads + threadIdx.x;
    if (i >= a.max_tokens) return;
    if (i >= ends[b.n_req - 1]) {
        a.slot[i] = a.pos[i] = a.req[i] = -1;
        return;
    }
    const int r = owner(ends, b.n_req, i);
    const int p = a.lens_out[r] - (ends[r] - i);
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
// Warps take few rows each when there are few tokens (share_rows), all of a
// token's when there are many.  23993 tokens of 32 + 2 x 8 rows of 128 in bf16
// (590 MB): 103 us, 5.7 TB/s; one token of 96 rows: 3.1 us; 64 tokens into Q4_0: 5.5 us.
// The 23993 tokens into Q4_0 (519 MB): 235 us, 2.2 TB/s, bound by the packing's chain.
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
// fp16 rows are bound by their bytes (23993 rows of 2 x 8 heads of 128: 33.8 us,
// 5.8 TB/s).  2999 Q4_0 rows of 2 x 32 heads to fp32 (112 MB): 23 us, 4.9 TB/s; writing
// the floats alone, 98 MB, takes 14.7 us, so that is not the writes' bound.  A lane
// makes 4 consecutive elements, so a warp writes whole lines; two lanes read the
// same 4 bytes of codes, one for the low nibbles and one for the high ones.  Rows are shared out over
// warps as for the append.
constexpr int kReadThreads = 128;
constexpr int kReadRows = 8;  // row slots of a lane in flight

template <int HD, bool Q4, int ACT>
__global__ void __launch_bounds__(kReadThreads) read_kernel(const __grid_constant__ PagedReadArgs a) {
    using A = Act<ACT>;
    using T = typename A::T;
    constexpr int kLanes = HD / 4, kWide = 32 / kLanes;  // lanes of a row, rows of a warp's access
    const int lane = threadIdx.x & 31, c = lane % kLanes;
    const long long item = static_cast<long long>(blockIdx.x) * (kReadThreads / 32) + (threadIdx.x >> 5);
    const int token = static_cast<int>(item / a.parts), part = static_cast<int>(item - static_cast<long long>(token) * a.parts);
    if (token >= a.n) return;
    const int slot = a.slot[token];
    const bool stored = slot >= 0 && slot < a.n_slots;
    if (part == 0 && lane == 0 && !stored && slot != -1) raise_error(a.status, kErrBadIndex);
    const uint32_t page = stored ? fast_div(slot, a.page) : 0;
    const uint32_t at = stored ? slot - page * a.page.d : 0;
    const long long row_of_page = static_cast<long long>(page) * a.n_kv_heads * a.page.d + at;
    const long long out0 = static_cast<long long>(token) * a.n_kv_heads * HD;
    const int end = min(2 * a.n_kv_heads, (part + 1) * a.part_rows);
#pragma unroll 1
    for (int row0 = part * a.part_rows; row0 < end; row0 += kReadRows * kWide) {
        using Raw = std::conditional_t<Q4, uint32_t, uint2>;
        Raw raw[kReadRows];
        __half scale[kReadRows];
#pragma unroll
        for (int i = 0; i < kReadRows; ++i) {  // keys of all heads, then values; past the end: the last row again
            const int row = min(row0 + i * kWide + lane / kLanes, end - 1);
            const bool is_v = row >= a.n_kv_heads;
            const long long r = row_of_page + static_cast<long long>(is_v ? row - a.n_kv_heads : row) * a.page.d;
            const void *cache = is_v ? a.v_cache : a.k_cache;
            if constexpr (Q4) {
                raw[i] = __ldcs(reinterpret_cast<const uint32_t *>(static_cast<const uint8_t *>(cache) + r * (HD / 2)) + c / 8 * 4 + c % 4);
                scale[i] = __ldg((is_v ? a.v_scale : a.k_scale) + r * (HD / 32) + c / 8);
            } else {
                raw[i] = __ldcs(reinterpret_cast<const uint2 *>(static_cast<const __half *>(cache) + r * HD) + c);
            }
        }
#pragma unroll
        for (int i = 0; i < kReadRows; ++i) {
            const int row = row0 + i * kWide + lane / kLanes;
            if (row >= end) continue;
            const bool is_v = row >= a.n_kv_heads;
            T *out = static_cast<T *>(is_v ? a.v_out : a.k_out) + out0 + (is_v ? row - a.n_kv_heads : row) * HD;
            float4 x;
            if constexpr (Q4) {
                const float d = __half2float(scale[i]);
                const uint32_t w = c & 4 ? raw[i] >> 4 : raw[i];
                auto code = [&](int b) { return __fmul_rn(static_cast<float>(static_cast<int>(w >> (8 * b) & 15) - 8), d); };
                x = make_float4(code(0), code(1), code(2), code(3));
            } else {
                x = Act<BMO_ACT_F16>::value(raw[i]);
            }
            if (!stored) x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            A::template store<true>(out + 4 * c, x);
        }
    }
}

// Rows of a warp: one round of loads, or more rounds once the warps are many (64 for each of
// B200's 148 SMs; 16, 32 and 128 measured the same for the append and 0 to 2 us of 23 more
// for the read, so the number need not follow the SMs of another part).
struct RowShare {
    int part_rows, parts;
    unsigned grid;
};
bool share_rows(int n, int rows, int round, int warps_per_cta, RowShare &out) {
    constexpr int kManyWarps = 148 * 64;
    const int rounds = (rows + round - 1) / round;
    const long long per = static_cast<long long>(n) * rounds / kManyWarps;
    out.parts = per < 1 ? rounds : per < rounds ? static_cast<int>((rounds + per - 1) / per) : 1;
    out.part_rows = (rounds + out.parts - 1) / out.parts * round;
    const long long grid = (static_cast<long long>(n) * out.parts + warps_per_cta - 1) / warps_per_cta;
    out.grid = static_cast<unsigned>(grid);
    return grid <= 0x7fffffff;
}

template <int HD, bool Q4>
cudaError_t append_act(PagedAppendArgs a, int act, cudaStream_t s) {
    RowShare r;
    if (!share_rows(a.n, a.n_heads + 2 * a.n_kv_heads, kAppendRows * (128 / HD), kAppendThreads / 32, r)) return cudaErrorInvalidValue;
    a.part_rows = r.part_rows;
    a.parts = r.parts;
    const unsigned g = r.grid;
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
cudaError_t read_act(PagedReadArgs a, int act, cudaStream_t s) {
    RowShare r;
    if (!share_rows(a.n, 2 * a.n_kv_heads, kReadRows * (128 / HD), kReadThreads / 32, r)) return cudaErrorInvalidValue;
    a.part_rows = r.part_rows;
    a.parts = r.parts;
    if (act == BMO_ACT_F32) read_kernel<HD, Q4, BMO_ACT_F32><<<r.grid, kReadThreads, 0, s>>>(a);
    else if (act == BMO_ACT_F16) read_kernel<HD, Q4, BMO_ACT_F16><<<r.grid, kReadThreads, 0, s>>>(a);
    else read_kernel<HD, Q4, BMO_ACT_BF16><<<r.grid, kReadThreads, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_paged_plan(const PagedPlanArgs &a, cudaStream_t s) {
    const int list_here = a.max_tokens <= kPlanOneCta;
    plan_kernel<<<1, kPlanThreads, 0, s>>>(a, list_here);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess || list_here) return e;
    // launched as a dependent, though the plan triggers nothing before it ends: a call of 61
    // joining histories takes 14.7 us, 16.4 without the attribute, 15.4 with a trigger at the plan's start
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((a.max_tokens + kListThreads - 1) / kListThreads);
    cfg.blockDim = dim3(kListThreads);
    cfg.stream = s;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, plan_list_kernel, a);
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
