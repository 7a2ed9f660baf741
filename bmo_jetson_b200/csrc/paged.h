// paged.h -- arguments and launchers of the paged key-value cache's kernels
// (kernels/paged.cu, kernels/paged_attention.cu; entries in kernel_api_paged.cu).
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/bmo_kernels.h"

namespace bmo {

constexpr int kPagedMaxReq = 65536;       // requests of one plan
constexpr int kPagedMaxRows = 4096;       // rows of one attention call (their tile counts sit in shared memory)
constexpr int kPagedMaxPageSize = 65536;

// n / d for 0 <= n < 2^31 by one multiply: q = (umulhi(n, mul) + n) >> shift;
struct FastDiv {
    uint32_t d, mul, shift;
};
FastDiv make_fast_div(uint32_t d);
#ifdef __CUDACC__
__device__ __forceinline__ uint32_t fast_div(uint32_t n, const FastDiv &f) { return (__umulhi(n, f.mul) + n) >> f.shift; }
#endif

struct PagedPlanArgs {
    bmo_page_book book;
    const int *n_new;
    int max_tokens;
    int *slot, *pos, *req, *offsets, *lens_out, *state_out;
};
cudaError_t launch_paged_plan(const PagedPlanArgs &a, cudaStream_t s);

constexpr int kPagedMaxPairs = 64;  // head_dim / 2
struct PagedAppendArgs {
    const void *q, *k, *v;
    void *q_out;
    long long q_stride, k_stride, v_stride, q_out_stride;  // elements
    const int *slot, *pos;
    void *k_cache, *v_cache;      // of the layer
    __half *k_scale, *v_scale;
    int n, n_heads, n_kv_heads;   // n_heads 0: no q
    int parts, part_rows;         // warps of a token and rows of each (set by the launcher)
    long long n_slots;
    FastDiv page;
    int *status;
    int rotate;
    float inv_freq[kPagedMaxPairs];
};
cudaError_t launch_paged_append(const PagedAppendArgs &a, int head_dim, int kv_type, int act, cudaStream_t s);

struct PagedReadArgs {
    const int *slot;
    const void *k_cache, *v_cache;  // of the layer
    const __half *k_scale, *v_scale;
    void *k_out, *v_out;
    int n, n_kv_heads;
    int parts, part_rows;  // as for the append
    long long n_slots;
    FastDiv page;
    int *status;
};
cudaError_t launch_paged_read(const PagedReadArgs &a, int head_dim, int kv_type, int act, cudaStream_t s);

struct PagedAttnArgs {
    const void *q;
    long long q_stride, out_stride;  // elements
    void *out;
    float *lse;
    const void *k, *v;               // of the layer
    const __half *k_scale, *v_scale;
    const int *table, *lens, *row_req, *row_len;
    int n_req, max_blocks, n_pages, window;
    FastDiv page;
    int n_rows, n_heads, n_kv_heads;
    int group;                       // query heads of a key head (this and the next set by the launcher)
    FastDiv units, chunks;           // units of a row, of a key head
    int cluster;                     // > 1: CTAs of a cluster that takes one head
    float qscale;                    // score scale * log2(e)
    int *status;
    // split rows: two partial results per CTA, one arrival counter per CTA
    float *part;
    int *cnt;
};
cudaError_t launch_paged_attention(PagedAttnArgs a, int head_dim, int kv_type, int act, void *scratch,
                                   size_t scratch_bytes, cudaStream_t s);
size_t paged_attention_scratch_bytes(int head_dim, int kv_type, int n_heads, int n_kv_heads);

}  // namespace bmo
