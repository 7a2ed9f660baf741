// kernel_api_paged.cu -- the paged key-value cache's entries of the kernel
// layer (include/bmo_kernels.h): argument checks, then the launchers of paged.h.
#include <climits>
#include <cmath>

#include "../../include/bmo_kernels.h"
#include "paged.h"
#include "layout.h"

namespace bmo {
namespace {

constexpr int kPlanRoom = 65536;  // the plan's counters step past max_tokens by no more
constexpr int kInvalid = static_cast<int>(cudaErrorInvalidValue);

bool aligned(const void *p, size_t n) { return !(reinterpret_cast<uintptr_t>(p) & (n - 1)); }

bool book_ok(const bmo_page_book &b) {
    return b.n_pages > 0 && b.page_size > 0 && b.page_size <= kPagedMaxPageSize && b.window >= 0 &&
           static_cast<long long>(b.n_pages) * b.page_size <= INT_MAX - 65535;
}

bool table_ok(const bmo_page_book &b) {
    return b.table && b.lens && b.n_req > 0 && b.max_blocks > 0 &&
           static_cast<long long>(b.max_blocks) * b.page_size <= INT_MAX - 65535;  // room to step past the end
}

bool cache_ok(const bmo_paged_kv *c) {
    if (!c || !book_ok(c->book) || !c->k || !c->v || !aligned(c->k, 16) || !aligned(c->v, 16)) return false;
    if (c->n_layers <= 0 || c->n_kv_heads <= 0 || (c->head_dim != 64 && c->head_dim != 128)) return false;
    // the kernels number a layer's rows in 32 bits
    if (static_cast<long long>(c->book.n_pages) * c->book.page_size > 0xfffffffell / c->n_kv_heads) return false;
    if (c->kv_type == kKvQ4_0) return c->k_scale && c->v_scale && aligned(c->k_scale, 16) && aligned(c->v_scale, 16);
    return c->kv_type == kKvF16;
}

size_t act_bytes(int act) { return act == BMO_ACT_F32 ? 4 : act == BMO_ACT_F16 || act == BMO_ACT_BF16 ? 2 : 0; }

// Rows of heads x head_dim elements of n rows, `stride` elements apart.
bool rows_ok(const void *p, int n, long long stride, int heads, int head_dim, size_t elem) {
    return p && aligned(p, elem) && (n <= 1 || stride >= static_cast<long long>(heads) * head_dim);
}

// Element offset of `layer` in the caches.
long long layer_rows(const bmo_paged_kv *c, int layer) {
    return static_cast<long long>(layer) * c->book.n_pages * c->n_kv_heads * c->book.page_size;
}

struct LayerPtrs {
    char *k, *v;
    __half *ks, *vs;
};
LayerPtrs layer_ptrs(const bmo_paged_kv *c, int layer) {
    const long long rows = layer_rows(c, layer);
    const long long bytes = c->kv_type == kKvQ4_0 ? rows * (c->head_dim / 2) : rows * c->head_dim * 2;
    LayerPtrs p{static_cast<char *>(c->k) + bytes, static_cast<char *>(c->v) + bytes, nullptr, nullptr};
    if (c->kv_type == kKvQ4_0) {
        p.ks = static_cast<__half *>(c->k_scale) + rows * (c->head_dim / 32);
        p.vs = static_cast<__half *>(c->v_scale) + rows * (c->head_dim / 32);
    }
    return p;
}

// theta^(-2i / head_dim) as the exact-order step's table: exponent in fp32,
// power in double, rounded once.
struct InvFreq {
    float theta = 0.0f;
    int head_dim = 0;
    float f[kPagedMaxPairs];
};
const InvFreq &inv_freq(float theta, int head_dim) {
    static thread_local InvFreq t;
    if (t.theta != theta || t.head_dim != head_dim) {
        for (int i = 0; i < head_dim / 2; ++i) {
            const float e = static_cast<float>(2 * i) / static_cast<float>(head_dim);
            t.f[i] = static_cast<float>(std::pow(static_cast<double>(theta), -static_cast<double>(e)));
        }
        t.theta = theta;
        t.head_dim = head_dim;
    }
    return t;
}

}  // namespace
}  // namespace bmo

using namespace bmo;

extern "C" {

int bmo_k_paged_plan(const bmo_page_book *book, const int32_t *n_new_dev, int max_tokens, int32_t *slot_dev,
                     int32_t *pos_dev, int32_t *req_dev, int32_t *offsets_dev, int32_t *lens_out_dev,
                     int32_t *state_out_dev, void *stream) {
    if (!book || !book_ok(*book) || !table_ok(*book) || !book->free_pages || !book->state || !n_new_dev ||
        max_tokens < 0 || max_tokens >= INT_MAX - kPlanRoom || (max_tokens && (!slot_dev || !pos_dev || !req_dev)) || !offsets_dev || !lens_out_dev ||
        !state_out_dev || book->n_req > kPagedMaxReq)
        return kInvalid;
    PagedPlanArgs a{*book,       n_new_dev,    max_tokens,   slot_dev,     pos_dev,
                    req_dev,     offsets_dev,  lens_out_dev, state_out_dev};
    return static_cast<int>(launch_paged_plan(a, static_cast<cudaStream_t>(stream)));
}

int bmo_k_paged_append(const bmo_paged_kv *cache, int layer, int n, const void *k_dev, long long k_stride,
                       const void *v_dev, long long v_stride, const int32_t *slot_dev, const int32_t *pos_dev,
                       float theta, const void *q_dev, long long q_stride, int n_heads, void *q_out_dev,
                       long long q_out_stride, int act_type, int *status_dev, void *stream) {
    const size_t elem = act_bytes(act_type);
    if (!cache_ok(cache) || layer < 0 || layer >= cache->n_layers || n < 0 || !elem) return kInvalid;
    const int kv = cache->n_kv_heads, hd = cache->head_dim;
    if (!(theta >= 0.0f) || std::isinf(theta)) return kInvalid;
    if (q_dev && (!(theta > 0.0f) || n_heads <= 0 || n_heads > 65536 || !q_out_dev)) return kInvalid;
    if (kv > 65536) return kInvalid;
    if (n == 0) return 0;
    if (!slot_dev || !rows_ok(k_dev, n, k_stride, kv, hd, elem) || !rows_ok(v_dev, n, v_stride, kv, hd, elem))
        return kInvalid;
    if (theta > 0.0f && !pos_dev) return kInvalid;
    if (q_dev && (!rows_ok(q_dev, n, q_stride, n_heads, hd, elem) || !rows_ok(q_out_dev, n, q_out_stride, n_heads, hd, elem)))
        return kInvalid;
    const LayerPtrs p = layer_ptrs(cache, layer);
    PagedAppendArgs a{};
    a.q = q_dev;
    a.k = k_dev;
    a.v = v_dev;
    a.q_out = q_out_dev;
    a.q_stride = q_stride;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.q_out_stride = q_out_stride;
    a.slot = slot_dev;
    a.pos = pos_dev;
    a.k_cache = p.k;
    a.v_cache = p.v;
    a.k_scale = p.ks;
    a.v_scale = p.vs;
    a.n = n;
    a.n_heads = q_dev ? n_heads : 0;
    a.n_kv_heads = kv;
    a.n_slots = static_cast<long long>(cache->book.n_pages) * cache->book.page_size;
    a.page = make_fast_div(cache->book.page_size);
    a.status = status_dev;
    a.rotate = theta > 0.0f;
    if (a.rotate) {
        const InvFreq &t = inv_freq(theta, hd);
        for (int i = 0; i < hd / 2; ++i) a.inv_freq[i] = t.f[i];
    }
    return static_cast<int>(launch_paged_append(a, hd, cache->kv_type, act_type, static_cast<cudaStream_t>(stream)));
}

int bmo_k_paged_read(const bmo_paged_kv *cache, int layer, int n, const int32_t *slot_dev, void *k_out_dev,
                     void *v_out_dev, int act_type, int *status_dev, void *stream) {
    const size_t elem = act_bytes(act_type);
    if (!cache_ok(cache) || layer < 0 || layer >= cache->n_layers || n < 0 || !elem || cache->n_kv_heads > 65536)
        return kInvalid;
    if (n == 0) return 0;
    if (!slot_dev || !k_out_dev || !v_out_dev || !aligned(k_out_dev, 4 * elem) || !aligned(v_out_dev, 4 * elem))
        return kInvalid;
    const LayerPtrs p = layer_ptrs(cache, layer);
    PagedReadArgs a{};
    a.slot = slot_dev;
    a.k_cache = p.k;
    a.v_cache = p.v;
    a.k_scale = p.ks;
    a.v_scale = p.vs;
    a.k_out = k_out_dev;
    a.v_out = v_out_dev;
    a.n = n;
    a.n_kv_heads = cache->n_kv_heads;
    a.n_slots = static_cast<long long>(cache->book.n_pages) * cache->book.page_size;
    a.page = make_fast_div(cache->book.page_size);
    a.status = status_dev;
    return static_cast<int>(
        launch_paged_read(a, cache->head_dim, cache->kv_type, act_type, static_cast<cudaStream_t>(stream)));
}

size_t bmo_k_paged_attention_scratch_bytes(const bmo_paged_kv *cache, int n_heads) {
    if (!cache_ok(cache) || n_heads <= 0 || n_heads % cache->n_kv_heads) return 0;
    return paged_attention_scratch_bytes(cache->head_dim, cache->kv_type, n_heads, cache->n_kv_heads);
}

int bmo_k_paged_attention(const bmo_paged_kv *cache, int layer, int n_rows, const void *q_dev, long long q_stride,
                          int n_heads, const int32_t *row_req_dev, const int32_t *row_len_dev, float scale,
                          void *out_dev, long long out_stride, float *lse_dev, int act_type, int *status_dev,
                          void *scratch_dev, size_t scratch_bytes, void *stream) {
    const size_t elem = act_bytes(act_type);
    if (!cache_ok(cache) || !table_ok(cache->book) || layer < 0 || layer >= cache->n_layers || n_rows < 0 ||
        n_rows > kPagedMaxRows || n_heads <= 0 || n_heads % cache->n_kv_heads || !elem || !std::isfinite(scale))
        return kInvalid;
    const bmo_page_book &b = cache->book;
    if (!row_req_dev && n_rows > b.n_req) return kInvalid;
    if (n_rows == 0) return 0;
    // the kernel numbers the call's tiles (16 positions or more of a head) in 31 bits
    const long long tiles = static_cast<long long>(b.max_blocks) * b.page_size / 16 + 4;
    if (n_heads > 65536 || tiles * n_rows > INT_MAX / n_heads) return kInvalid;
    const int hd = cache->head_dim;
    if (!rows_ok(q_dev, n_rows, q_stride, n_heads, hd, elem) || !rows_ok(out_dev, n_rows, out_stride, n_heads, hd, elem) ||
        !scratch_dev || !aligned(scratch_dev, 16))
        return kInvalid;
    const LayerPtrs p = layer_ptrs(cache, layer);
    PagedAttnArgs a{};
    a.q = q_dev;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.out = out_dev;
    a.lse = lse_dev;
    a.k = p.k;
    a.v = p.v;
    a.k_scale = p.ks;
    a.v_scale = p.vs;
    a.table = b.table;
    a.lens = b.lens;
    a.row_req = row_req_dev;
    a.row_len = row_len_dev;
    a.n_req = b.n_req;
    a.max_blocks = b.max_blocks;
    a.n_pages = b.n_pages;
    a.window = b.window;
    a.page = make_fast_div(b.page_size);
    a.n_rows = n_rows;
    a.n_heads = n_heads;
    a.n_kv_heads = cache->n_kv_heads;
    const double sc = scale != 0.0f ? scale : 1.0 / std::sqrt(static_cast<double>(hd));
    a.qscale = static_cast<float>(sc * 1.4426950408889634);
    a.status = status_dev;
    return static_cast<int>(launch_paged_attention(a, hd, cache->kv_type, act_type, scratch_dev, scratch_bytes,
                                                   static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
