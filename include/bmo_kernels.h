/*
 * bmo_kernels.h -- device-pointer kernel layer of libbmo.so.
 *
 * The counterpart of the reference's launch_* functions (utkarshyadav009/
 * bmo_jetson src/bmo.h:348-445): each call takes device buffers and a
 * cudaStream_t (as void*), launches the sm_100a kernels that the decode step
 * uses, and returns 0 or a CUDA error code.  Callers own every buffer,
 * including the scratch the split kernels need (size from the *_scratch_bytes
 * queries).  Calls are asynchronous on `stream`.
 */
#ifndef BMO_KERNELS_H
#define BMO_KERNELS_H

#include <stddef.h>
#include <stdint.h>

#include "bmo_api.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { BMO_PERM_IDENTITY = 0, BMO_PERM_SWIGLU = 1 };

/* Q8_1 quantisation of n floats (n % 32 == 0) into 36-byte blocks
 * (fp16 d, fp16 sum, 32 int8).  Replaces bmo_quantize_row_q8_1_kernel as
 * launched by launch_gemv_q4_0_q8_1 (bmo_cuda_kernels.cu:685-699). */
BMO_API int bmo_k_quantize_q8_1(const float *x_dev, void *out_dev, int n, void *stream);

/* Bytes of the tiled layout of a rows x cols Q4_0 matrix. */
BMO_API size_t bmo_k_q4_0_tiled_bytes(int rows, int cols, int perm, int swiglu_f);
/* ggml Q4_0 row-major blocks -> tiled layout (done once at model load). */
BMO_API int bmo_k_repack_q4_0(const void *ggml_dev, void *tiled_dev, int rows, int cols, int perm, int swiglu_f,
                              void *stream);

/* Scratch bytes bmo_k_gemv_q4_0 needs for a rows x cols matrix. */
BMO_API size_t bmo_k_gemv_scratch_bytes(int rows, int cols, int perm, int swiglu_f);
/* y = W x with the reference's Q4_0 x Q8_1 arithmetic (replaces
 * launch_gemv_q4_0_q8_1, bmo.h:405-412).  W is the tiled layout.
 * gamma_dev != NULL: x is RMS-normalised and scaled by gamma first (fused
 * launch_rmsnorm, bmo.h:358-364).  perm == SWIGLU: y receives
 * silu(gate) * up of length swiglu_f (fused launch_swiglu_split).
 * resid_dev != NULL: y = resid + W x (fused launch_residual_add).
 * q8_out_dev / xn_out_dev (optional) receive the Q8_1 blocks and the
 * normalised fp32 vector the kernel used.  scratch_dev must be zero on the
 * first call and is left zero by every call that returns 0.  x_dev and
 * xn_out_dev are 16-byte aligned; with gamma_dev, cols <= 5120.  grid 0
 * picks the launch (whole row tiles per CTA where that balances); grid > 0
 * runs that many CTAs over an even split of the (row tile, 8-block chunk)
 * units, combining straddled tiles through scratch_dev. */
BMO_API int bmo_k_gemv_q4_0(const void *tiled_dev, int rows, int cols, int perm, int swiglu_f,
                            const float *x_dev, const float *gamma_dev, float eps, const float *resid_dev,
                            float *y_dev, void *q8_out_dev, float *xn_out_dev, void *scratch_dev,
                            size_t scratch_bytes, int grid, void *stream);

/* y = W x computed in the reference kernel's own fp32 order: every row is
 * bit-identical to launch_gemv_q4_0_q8_1 (bmo.h:405-412, kernel
 * bmo_cuda_kernels.cu:560-683) on the same ggml weights and x, and with
 * gamma_dev the RMSNorm is launch_rmsnorm's (bmo.h:358-364) in its own
 * order, the SwiGLU (perm SWIGLU) launch_swiglu_split's with __expf and the
 * residual (resid_dev) launch_residual_add's.  Arguments as in
 * bmo_k_gemv_q4_0; no scratch (each CTA owns whole row tiles); with
 * gamma_dev, cols <= 4096.  status_dev (optional, device int) receives bit
 * 1 if a weight copy did not land within the wait bound. */
BMO_API int bmo_k_gemv_q4_0_ref(const void *tiled_dev, int rows, int cols, int perm, int swiglu_f,
                                const float *x_dev, const float *gamma_dev, float eps, const float *resid_dev,
                                float *y_dev, void *q8_out_dev, float *xn_out_dev, int *status_dev, void *stream);

/* Size of the fixed scratch buffer behind bmo_k_gemv_q4_0_static (4 MiB: every
 * temporal and depformer layer matrix of the 7B Moshi shapes fits; the
 * 32000-row text head does not). */
#define BMO_K_GEMV_STATIC_SCRATCH_BYTES (4u << 20)
/* Returned by bmo_k_gemv_q4_0_static when the matrix needs more scratch than
 * BMO_K_GEMV_STATIC_SCRATCH_BYTES (see bmo_k_gemv_scratch_bytes). */
#define BMO_K_ERR_SCRATCH_TOO_SMALL (-2)

/* bmo_k_gemv_q4_0 for callers that cannot allocate device memory when they
 * run it (a real-time callback that must not block in cudaMalloc, a host
 * framework that owns all allocations, a process under a device-memory cap).
 * No counterpart in the reference.  The split-K scratch is a fixed 4 MiB
 * buffer inside libbmo (held by every GPU that loads the library until
 * exit) instead of scratch_dev; nothing is allocated or freed.  Arguments
 * and results are those of bmo_k_gemv_q4_0.  The buffer is shared by every
 * call on a device and keeps the last call's contents (its counters are
 * cleared on `stream` before each launch), so calls that can overlap on the
 * GPU race: keep them on one stream or order them.  The first call on a
 * device looks up the buffer's address; make it before any stream capture.
 * That address is kept for the life of the process, so after cudaDeviceReset
 * on a device this entry point must not be used on it again.  Arguments are
 * checked before the shared buffer is touched.  Returns
 * BMO_K_ERR_SCRATCH_TOO_SMALL for matrices beyond the buffer. */
BMO_API int bmo_k_gemv_q4_0_static(const void *tiled_dev, int rows, int cols, int perm, int swiglu_f,
                                   const float *x_dev, const float *gamma_dev, float eps, const float *resid_dev,
                                   float *y_dev, void *q8_out_dev, float *xn_out_dev, int grid, void *stream);

/* Scratch bytes bmo_k_batch_gemm_q4_0 needs (on the current device). */
BMO_API size_t bmo_k_batch_gemm_scratch_bytes(int rows, int cols, int perm, int swiglu_f, int n_sess);
/* The batched decode's GEMM (no reference counterpart: the reference decodes
 * one session): for each of n_sess (1..64) sessions, y[s] = W x[s] with the
 * Q4_0 x Q8_1 arithmetic of bmo_k_gemv_q4_0.  x_dev [n_sess][cols], y_dev
 * [n_sess][rows] ([n_sess][swiglu_f] for perm SWIGLU); gamma_dev and
 * resid_dev ([n_sess][rows]) as in bmo_k_gemv_q4_0.  tensor_cores = 1: int8
 * tcgen05 MMA per 32-column block into tensor memory, the reference's
 * half-block terms summed error-free (the rounding of bmo_k_gemv_q4_0 up to
 * rare ties); 2: tensor cores with full-block terms summed in fp32
 * (fp32-accurate, not reproducible bit for bit); 0: CUDA cores with the
 * batch-1 GEMV's rounding.  scratch_dev must be zero on the first call and
 * is left reusable by every call that returns 0. */
BMO_API int bmo_k_batch_gemm_q4_0(const void *tiled_dev, int rows, int cols, int perm, int swiglu_f,
                                  const float *x_dev, const float *gamma_dev, float eps, const float *resid_dev,
                                  float *y_dev, int n_sess, int tensor_cores, void *scratch_dev,
                                  size_t scratch_bytes, void *stream);

/* Appends k, v (fp32, [n_kv_heads][head_dim]) at ring slot pos % n_ctx of
 * `layer`, then attends q over the window (replaces launch_decode_attention,
 * bmo.h:414-428).  Caches are [n_layers][n_kv_heads][n_ctx][head_dim] in
 * fp16 (kv_type 0) or Q4_0 nibble planes with fp16 scale planes (kv_type 1;
 * *_scale_dev).  pos_dev is a device int; n_ctx <= 8192.  No scratch: the
 * window splits of a head exchange partial results through distributed
 * shared memory. */
BMO_API int bmo_k_decode_attention(const float *q_dev, const float *k_dev, const float *v_dev, void *k_cache_dev,
                                   void *v_cache_dev, void *k_scale_dev, void *v_scale_dev, float *out_dev,
                                   int head_dim, int n_heads, int n_kv_heads, int n_ctx, const int *pos_dev,
                                   int layer, int kv_type, void *stream);

/* bmo_k_decode_attention over an fp16 ring, computed in the reference
 * kernel's own fp32 order: bit-identical to launch_decode_attention
 * (bmo.h:414-428, kernel bmo_cuda_kernels.cu:713-848) on the same ring,
 * q, k and v, including the appended slot.  head_dim 64 or 128; n_ctx <= 1024
 * (the reference kernel's own score buffer).  No scratch. */
BMO_API int bmo_k_decode_attention_ref(const float *q_dev, const float *k_dev, const float *v_dev, void *k_cache_dev,
                                       void *v_cache_dev, float *out_dev, int head_dim, int n_heads, int n_kv_heads,
                                       int n_ctx, const int *pos_dev, int layer, void *stream);

/* One tensor-parallel exchange over peer memory (the kernel bmo_init_tp
 * handles run after each split projection): parts[r] is rank r's buffer of n
 * double partial sums (device or peer-mapped pointers, r < size <= 8),
 * flag_out[r] this rank's 64-bit arrival word in rank r's block (ignored for
 * r == rank), flag_in this rank's words (one per source rank), seq a device
 * counter starting at 0 that the exchanges of a group share, status a device
 * int.  Publishes exchange number e into flag_out, waits (at most 2 s) for
 * flag_in[r] >= e from every peer, then y[i] = resid[i] + fl(sum over r in
 * rank order of parts[r][i]).  A wait that runs out sets bit 4 of *status and
 * leaves y untouched; while that bit is set, exchanges return at once.
 * n <= 8192. */
BMO_API int bmo_k_tp_exchange(const double *const *parts, unsigned long long *const *flag_out,
                              const unsigned long long *flag_in_dev, unsigned long long *seq_dev,
                              const float *resid_dev, float *y_dev, int *status_dev, int rank, int size, int n,
                              void *stream);

/* One draw of the daemon's token sampler (sample_token_cpp,
 * bmo_daemon.cpp:147-175) over logits_dev[0, n) on the device: first argmax
 * when top_k <= 0 or temp <= 1e-4, else the top_k logits (ties by lower
 * index), exp(l_i / temp - l_0 / temp) in float and std::discrete_distribution's
 * draw from std::mt19937.  pause_rule 1 adds the daemon's text rule
 * (:758-762): a first argmax of 3 or 0 is kept without a draw.  rng_dev holds
 * 625 words, the generator's 624 state words then its position (624 right
 * after seeding), and is advanced in place.  n <= 32768, min(top_k, n) <=
 * 2048.  One CTA. */
BMO_API int bmo_k_sample_token(const float *logits_dev, int n, float temp, int top_k, int pause_rule,
                               uint32_t *rng_dev, int32_t *out_dev, void *stream);

/* ---- paged key-value cache ----------------------------------------------
 *
 * A cache of any number of sessions ("requests") that share one pool of
 * pages instead of owning a ring each.  A page holds page_size positions of
 * every layer; a page of one layer is laid out as a ring of page_size slots
 * (bmo_k_decode_attention): [n_layers][n_pages][n_kv_heads][page_size][head_dim]
 * in fp16 (kv_type 0), or Q4_0 nibble planes (head_dim / 2 bytes a row) with
 * fp16 scale planes [..][head_dim / 32] (kv_type 1).  Position p of request r
 * is in page table[r][p / page_size] at slot p % page_size; a "slot number"
 * is page * page_size + slot.  head_dim 64 or 128; page_size 1..65536;
 * n_pages * page_size and max_blocks * page_size below 2^31 - 65535.
 * No counterpart in the reference, which decodes one session. */

/* Element types of the activations of the paged calls (q, k, v, outputs). */
enum { BMO_ACT_F32 = 0, BMO_ACT_F16 = 1, BMO_ACT_BF16 = 2 };

/* Bits of the status words of the paged calls. */
enum {
    BMO_PAGED_NO_PAGES = 1 << 5,   /* plan: the step needs more pages than are free */
    BMO_PAGED_TABLE_FULL = 1 << 6, /* plan: a request would outgrow max_blocks pages */
    BMO_PAGED_NO_ROOM = 1 << 7,    /* plan: more new positions than max_tokens */
    BMO_PAGED_BAD_INDEX = 1 << 8   /* a length, request, page or slot number out of range; the access was left out */
};

/* Which request has which pages.  All arrays are device memory. */
typedef struct bmo_page_book {
    int32_t *table;      /* [n_req][max_blocks] page of each block; entries outside a request's window are stale */
    int32_t *lens;       /* [n_req] positions each request holds */
    int32_t *free_pages; /* [n_pages] ring of page numbers */
    int32_t *state;      /* [4]: first free entry of the ring, free pages, status bits, new positions of the step */
    int32_t n_req, max_blocks, n_pages, page_size;
    int32_t window; /* > 0: a token attends to the last `window` positions, its own included; 0: to all */
    int32_t *undo;  /* [4 + 2 * n_pages], zero at first, or NULL: what lets a plan be made again (bmo_k_paged_plan) */
} bmo_page_book;

typedef struct bmo_paged_kv {
    bmo_page_book book;
    void *k, *v;             /* device, 16-byte aligned (the scales too) */
    void *k_scale, *v_scale; /* kv_type 1 only */
    int32_t n_layers, n_kv_heads, head_dim, kv_type;
} bmo_paged_kv;

/* Plans one step on the device: n_new_dev[r] > 0 appends that many positions
 * to request r, 0 leaves it, < 0 ends it (its length becomes 0).  Pages for
 * the new positions are taken from the ring of free pages in request order;
 * pages that fall out of the window of the next step's tokens, and those of ended
 * requests, are put at the ring's end.  A page given back in a step keeps its rows
 * during the step: it can be taken again from the next plan on.  The new
 * positions are listed request by request: entry i of slot_dev, pos_dev and
 * req_dev [max_tokens] is its slot number, position and request (-1 past the
 * last), offsets_dev [n_req + 1] is each request's first entry.
 * lens_out_dev [n_req] and state_out_dev [4] receive the new lengths and
 * state; they may be book->lens and book->state.  The table and the ring
 * change in place.  With book->undo, a plan into other lens_out_dev and
 * state_out_dev may be dropped: the next plan from the old lengths and state,
 * of the same step or another, is as if it had not been made.  That holds
 * for the last plan that was served, through the same undo buffer.  Without it
 * (undo NULL) a plan's outputs have to be adopted: pages given back may have
 * overwritten the ring's entries that the step took, and a second plan from
 * the old state would hand out pages that are in use.  A step that cannot be
 * served changes nothing but state_out[2], which says why
 * (BMO_PAGED_* bits), and lists no positions.  n_req <= 65536. */
BMO_API int bmo_k_paged_plan(const bmo_page_book *book, const int32_t *n_new_dev, int max_tokens, int32_t *slot_dev,
                             int32_t *pos_dev, int32_t *req_dev, int32_t *offsets_dev, int32_t *lens_out_dev,
                             int32_t *state_out_dev, void *stream);

/* Stores n rows k_dev, v_dev [n][n_kv_heads][head_dim] (rows k_stride,
 * v_stride elements apart, act_type BMO_ACT_*) at slot_dev[i] of `layer`;
 * slot -1 leaves a row out.  theta > 0: k is rotated first by pos_dev[i]
 * (interleaved pairs, angles and products as the exact-order decode step),
 * and q_dev [n][n_heads][head_dim], if not NULL, is rotated into q_out_dev
 * (which may be q_dev).  fp16 rounding and Q4_0 packing are the ring's.  Two
 * rows of one call must not have the same slot.  status_dev (optional,
 * device int) receives BMO_PAGED_BAD_INDEX for slots outside the cache. */
BMO_API int bmo_k_paged_append(const bmo_paged_kv *cache, int layer, int n, const void *k_dev, long long k_stride,
                               const void *v_dev, long long v_stride, const int32_t *slot_dev, const int32_t *pos_dev,
                               float theta, const void *q_dev, long long q_stride, int n_heads, void *q_out_dev,
                               long long q_out_stride, int act_type, int *status_dev, void *stream);

/* Reads the rows at slot_dev[0, n) of `layer` back: k_out_dev, v_out_dev
 * [n][n_kv_heads][head_dim], dense and aligned to 4 elements, in act_type; slot -1 and slots outside
 * the cache read as zeros (the latter set BMO_PAGED_BAD_INDEX). */
BMO_API int bmo_k_paged_read(const bmo_paged_kv *cache, int layer, int n, const int32_t *slot_dev, void *k_out_dev,
                             void *v_out_dev, int act_type, int *status_dev, void *stream);

/* Scratch bytes of bmo_k_paged_attention (0: the cache is not one it accepts). */
BMO_API size_t bmo_k_paged_attention_scratch_bytes(const bmo_paged_kv *cache, int n_heads);
/* Attention of single tokens over the pages of `layer`: row i of q_dev
 * [n_rows][n_heads][head_dim] attends to the last `window` (book.window; 0:
 * all) of the first row_len_dev[i] positions of request row_req_dev[i].
 * row_req_dev NULL: row i is request i; row_len_dev NULL: the request's
 * length.  So several rows may be tokens of one request.  row_len_dev[i] is
 * at most the request's length in book.lens, where lengths planned into a
 * separate lens_out_dev have to be first; a larger one sets BMO_PAGED_BAD_INDEX
 * and means that length.  With a window the caller sees to it that row_len_dev[i]
 * is above the length that the request had before the last plan, or that
 * its window begins in pages that were not given back before: those may be
 * another request's.  Query head h reads
 * key head h / (n_heads / n_kv_heads); scale 0 means 1 / sqrt(head_dim).
 * out_dev [n_rows][n_heads][head_dim] in act_type; lse_dev (optional, fp32
 * [n_rows][n_heads]) receives log(sum(exp(score))).  A row of length 0 gives
 * zeros and -inf.  Rows are q_stride, out_stride elements apart.  What
 * lies in slots past a row's length, or before its window, has no part in its result.  Sums, maxima and products are fp32
 * (each fp32 factor as two fp16 parts; heads that meet an infinite or NaN
 * element are computed from the formula instead, in which a block of a Q4_0 key
 * is its scale times the sum of its codes' products); the result is the same from call to
 * call.  A row of one position gives the stored value, rounded or packed, where
 * a ring's attention (bmo_k_decode_attention) gives v as it came.  scratch_dev must be zero on the first call, is left reusable, and
 * serves one call at a time.  n_rows <= 4096, and n_rows * n_heads *
 * (max_blocks * page_size / 16 + 4) below 2^31.  status_dev as above. */
BMO_API int bmo_k_paged_attention(const bmo_paged_kv *cache, int layer, int n_rows, const void *q_dev,
                                  long long q_stride, int n_heads, const int32_t *row_req_dev,
                                  const int32_t *row_len_dev, float scale, void *out_dev, long long out_stride,
                                  float *lse_dev, int act_type, int *status_dev, void *scratch_dev,
                                  size_t scratch_bytes, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* BMO_KERNELS_H */
