/*
 * bnn_b200_paged.h - attention of many requests over a paged key-value cache.
 *
 * The engine of bnn_b200_engine.h decodes a fixed set of rows in lockstep,
 * each over a contiguous FP32 cache of its own. A program that serves many
 * requests of unlike lengths keeps one pool of pages instead and hands pages
 * out as requests grow. These operators are the attention part of such a
 * program's layer, between the W1A8 q|k|v linear (whose FP32 rows they read
 * as they are) and the o linear:
 *
 *   bnn_b200_paged_append     q and k normalised per head and rotated by their
 *                             positions; q returned, k and v written to their
 *                             slots of the cache, in one pass
 *   bnn_b200_paged_attention  attention of each request's new tokens (one, a
 *                             few, or a prompt chunk) over its pages, causal,
 *                             with an optional sliding window and first tokens
 *                             that stay visible
 *
 * No counterpart in the reference: its attention is one host loop over one
 * sequence (bnn-sw-v2/qwen3/qwen3.c:440-480).
 *
 * Calls validate on the host, enqueue on the given stream and return without
 * waiting; they can be captured into a CUDA graph. All pointers are device
 * pointers on the handle's GPU. Strides and sizes count elements. What only
 * the device sees (a position outside the rotation table, a slot outside the
 * cache, a request with more new tokens than max_q, with tokens outside the
 * call's or with a length that its page table does not hold) is recorded and
 * read by bnn_b200_paged_sync.
 */
#ifndef BNN_B200_PAGED_H
#define BNN_B200_PAGED_H

#include "bnn_b200_accel.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types. The cache holds BF16 or F16; projections come in any. */
typedef enum { BNN_PAGED_F32 = 1, BNN_PAGED_BF16 = 2, BNN_PAGED_F16 = 3 } BNN_PagedType;

#define BNN_PAGED_MAX_BATCH 4096
#define BNN_PAGED_MAX_GROUP 16   /* query heads per KV head */

/* The pool of pages of one layer. Position p of a request lies in page
 * table[p / page_size], row p % page_size; slot = page * page_size + row.
 * Strides go from page to page, head to head, row to row; a row's head_dim
 * values are adjacent. Pointers are 16-byte aligned and strides multiples of
 * 8 elements. page_size: 16, 32, 64, 128 or 256; head_dim: 64 or 128. */
typedef struct {
    void* k;
    void* v;
    int64_t k_page_stride, k_head_stride, k_row_stride;
    int64_t v_page_stride, v_head_stride, v_row_stride;
    int64_t pages, kv_heads, page_size, head_dim;
    int64_t type; /* BNN_PAGED_BF16 or BNN_PAGED_F16 */
} BNN_PagedCache;

/* Token t's q, k, v rows: y = x / sqrt(mean(x^2) + eps) * gain per head (no
 * norm where the gain is NULL), then dimensions below rotary_dim rotated by
 * row positions[t] of the cos/sin tables [table_rows][rotary_dim / 2]:
 * (a, b) -> (a cos - b sin, b cos + a sin) over pairs (i, i + rotary_dim / 2),
 * or (2i, 2i + 1) with interleaved != 0 (gains and tables on 16-byte boundaries). All in FP32, rounded once to the
 * cache's type. q goes to q_out (same type as the cache), k and v to slot
 * slots[t]; a negative slot stores neither. rotary_dim: 0, or a multiple of 8
 * up to head_dim. A position outside the table leaves the token's q_out rows
 * zero and stores nothing, a slot outside the cache stores nothing; both make
 * the next bnn_b200_paged_sync return BNN_ERANGE. Two tokens of one call
 * must not share a slot. Outputs overlap no input. q_out's rows lie on 8-byte boundaries; q, k and v may
 * lie anywhere (16-byte rows load faster). */
typedef struct {
    BNN_PagedCache cache;
    const void* q;
    const void* k;
    const void* v;
    const float* q_norm; /* [head_dim] or NULL */
    const float* k_norm;
    const float* cos;
    const float* sin;
    const int32_t* positions; /* [tokens] */
    const int32_t* slots;     /* [tokens] */
    void* q_out;
    int64_t tokens, heads;
    int64_t type; /* of q, k, v: any BNN_PagedType */
    int64_t q_token_stride, q_head_stride, k_token_stride, k_head_stride, v_token_stride, v_head_stride;
    int64_t out_token_stride, out_head_stride;
    int64_t rotary_dim, table_rows, interleaved;
    double eps;
} BNN_PagedAppend;
BNN_Status bnn_b200_paged_append(BNN_Device device, const BNN_PagedAppend* desc, void* stream);

/* o_i = sum_j softmax_j(scale * q_i . k_j) v_j over the visible keys j.
 * Request b owns tokens q_starts[b] .. q_starts[b + 1] - 1, the last of its
 * kv_lens[b] positions (its own keys are in the cache already); token i of n
 * stands at position p = kv_lens[b] - n + i. Key j is visible when
 * 0 <= j <= p, its page_table entry is a page of the pool (entries outside
 * [0, pages), say of released pages, hide their keys), and window == 0 or
 * j > p - window or j < sinks. A token with no visible key, or with a softmax
 * sum of zero, gets o = 0 and lse = -inf. Cache rows that no token of the
 * call sees are never used, whatever they hold.
 * Scores, maxima and sums are FP32; the weights enter the value product in the
 * cache's type (as any 16-bit tensor-core product), the result is rounded once
 * to out_type. lse (natural log of the softmax sum) may be NULL.
 * q has the cache's type; heads is a multiple of kv_heads, at most
 * BNN_PAGED_MAX_GROUP times. max_q bounds the new tokens of any request. The
 * tokens of a request that has more of them, or some outside [0, tokens), or a
 * kv_len below zero or above table_width * page_size, stay unwritten and the
 * next bnn_b200_paged_sync returns BNN_ERANGE. workspace: bnn_b200_paged_workspace
 * bytes, zeroed once before its first use and used by one call at a time
 * (calls on one stream may share it). Outputs overlap no input. Results do not
 * depend on what else is in flight: sums are joined in a fixed order. Which
 * kernels serve a call goes by the sizes given here, the longest cache by
 * table_width: a table no wider than its requests need is the faster one. */
typedef struct {
    BNN_PagedCache cache;
    const void* q;
    void* out;
    float* lse;
    const int32_t* page_table; /* [batch][table_width], rows table_stride >= 0 apart (0: one row for all) */
    const int32_t* kv_lens;    /* [batch] */
    const int32_t* q_starts;   /* [batch + 1] */
    void* workspace;
    int64_t workspace_bytes;
    int64_t batch, tokens, heads, max_q;
    int64_t q_token_stride, q_head_stride, out_token_stride, out_head_stride, lse_token_stride;
    int64_t table_stride, table_width;
    int64_t window, sinks;
    int64_t out_type; /* the cache's type or BNN_PAGED_F32 */
    double scale;     /* positive; scale * log2(e) is a finite float */
} BNN_PagedAttention;
BNN_Status bnn_b200_paged_attention(BNN_Device device, const BNN_PagedAttention* desc, void* stream);

/* Bytes of the workspace (the device's size alone decides: about 20 MB). */
BNN_Status bnn_b200_paged_workspace(BNN_Device device, size_t* bytes);

/* Waits for `stream` and returns what the paged calls of this handle recorded
 * since the last one: BNN_ERANGE (see above), BNN_ETIMEOUT (a bounded device
 * wait expired; outputs are partial), BNN_EIO on a CUDA failure, else BNN_OK. */
BNN_Status bnn_b200_paged_sync(BNN_Device device, void* stream);

#ifdef __cplusplus
}
#endif

#endif
