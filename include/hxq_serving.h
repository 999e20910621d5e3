/*
 * hxq_serving.h -- the operators a serving step needs beside the compressed
 * projections (B200, sm_100a): maps from request lengths to cache blocks, an
 * 8-bit KV cache and attention over it, and low-rank adapters of many
 * requests beside a shared projection.
 *
 * No counterpart in the reference library.  Device pointers throughout
 * unless a parameter says host; every call is stream-ordered on `stream` (a
 * cudaStream_t; NULL = the legacy default stream) of the current device,
 * allocates nothing, keeps no state between calls and can be captured in a
 * CUDA graph.  Lengths, tables and slots stay on the device, so a captured
 * step may be replayed with others.  Arguments the host can see are checked
 * and refused before anything is enqueued; what only the device sees (a
 * block number, a length) is checked there, never used to form an address
 * when it is out of range, and recorded in *d_status (device word, may be
 * NULL): bits are ORed in and never cleared by the library.
 */
#ifndef HXQ_SERVING_H
#define HXQ_SERVING_H

#include <stddef.h>
#include <stdint.h>

#include "hxq.h"

#ifdef __cplusplus
extern "C" {
#endif

#define HXQ_SERVING_NO_BLOCKS   1u   /* more blocks needed than the free list holds */
#define HXQ_SERVING_BAD_BLOCK   2u   /* a block number or slot outside the cache, or a table too narrow */
#define HXQ_SERVING_BAD_LENGTH  4u   /* negative length, or starts outside the rows given */
#define HXQ_SERVING_FULL        8u   /* more tokens than the slot map has room for */
#define HXQ_SERVING_ORDER      16u   /* slots of one block repeated or descending in one append */
#define HXQ_SERVING_BAD_ADAPTER 32u  /* an adapter number >= n_adapters (treated as none) */
#define HXQ_SERVING_TIMEOUT    64u   /* a pipeline wait ran out; the results are not valid */

/* Element types of unquantised operands. */
#define HXQ_ELEM_F32  0
#define HXQ_ELEM_BF16 1
#define HXQ_ELEM_F16  2

/* -- Step plan --------------------------------------------------------------
 * Request b brings d_new[b] tokens to the d_cached[b] it already holds.
 * Writes, for B requests:
 *   d_starts[B + 1]  exclusive sums of d_new (row of each request's first token),
 *   d_lens[B]        d_cached + d_new,
 *   d_slots[n_slots], d_positions[n_slots]  per token row: where its key and
 *                    value go (block * block_tokens + offset) and its position
 *                    in its request; rows behind the last token get -1,
 *   d_table[B, table_width]  entries of the blocks this step begins, taken in
 *                    request order from d_free[n_free]; other entries are
 *                    read (a request's last, partly filled block) or left,
 *   d_taken[1]       how many of d_free were taken.
 * When the free list ends, the entries behind it become -1 and so do their
 * tokens' slots (HXQ_SERVING_NO_BLOCKS).  No array that is written overlaps
 * another one (d_lens is not d_cached).  1 <= block_tokens <= 65536,
 * B <= HXQ_PLAN_MAX_REQUESTS.  B = 0 writes d_starts[0] = 0 and the map. */
#define HXQ_PLAN_MAX_REQUESTS 8192
hxq_error_t hxq_cuda_kv_plan(const int32_t *d_new, const int32_t *d_cached, uint32_t B, int32_t *d_table,
                             uint32_t table_width, uint32_t block_tokens, const int32_t *d_free, uint32_t n_free,
                             int32_t *d_starts, int32_t *d_lens, int32_t *d_slots, int32_t *d_positions,
                             uint32_t n_slots, int32_t *d_taken, uint32_t *d_status, void *stream);

/* -- KV cache in 8 bits ------------------------------------------------------
 * Codes [n_blocks][n_heads][block_tokens][head_dim], 16-byte aligned, with
 * one fp32 scale >= 0 per (block, head); a value is code * scale.  Filled by
 * hxq_cuda_kv_append; the caller owns the memory. */
#define HXQ_KV_INT8 0   /* -127..127, scale = max |x| / 127 */
#define HXQ_KV_E4M3 1   /* fp8 e4m3 (finite), scale = max |x| / 448 */
typedef struct {
    void    *k, *v;
    float   *k_scales, *v_scales;
    uint32_t n_blocks, n_heads, block_tokens, head_dim;
    uint32_t format;
} hxq_kv_cache_t;

/* Quantise the keys and values of n_tokens rows into the cache: row t, head h
 * at d_k[t * k_stride_t + h * k_stride_h ...] (strides in elements, head_dim
 * consecutive elements), type elem.  Slot -1 (any negative) skips a row; a
 * slot outside the cache is skipped and recorded.
 * A block's scale only grows: s' = max(s, max |x| / qmax) over the rows the
 * call writes to it; where it grew, codes the block already holds become
 * round(code * (s / s')) (round to nearest even).  Writing a block's first
 * slot begins it anew: its old scale does not count and its old codes, at
 * slots the call does not write, keep no meaning.  A scale below 2^-126
 * becomes 0 (all codes 0).  An infinity or NaN among a block's new values
 * makes its scale infinite or NaN, and what is read from the block NaN.
 * Rows of one block must be consecutive with ascending slots, each slot once
 * (as hxq_cuda_kv_plan makes them), and a block written by one request only;
 * otherwise that block's content is unspecified (adjacent violations are
 * recorded as HXQ_SERVING_ORDER).
 * head_dim 64, 128 or 256; block_tokens a multiple of 16, at most 256;
 * n_blocks * block_tokens < 2^31. */
hxq_error_t hxq_cuda_kv_append(const hxq_kv_cache_t *cache, const void *d_k, const void *d_v, int elem,
                               int64_t k_stride_t, int64_t k_stride_h, int64_t v_stride_t, int64_t v_stride_h,
                               const int32_t *d_slots, uint32_t n_tokens, uint32_t *d_status, void *stream);
/* code * scale (in fp32, then rounded to elem) at the given slots: contiguous
 * [n_tokens, n_heads, head_dim] into d_k and d_v (either may be NULL).
 * Negative slots give rows of zeros, slots outside the cache also (recorded). */
hxq_error_t hxq_cuda_kv_read(const hxq_kv_cache_t *cache, const int32_t *d_slots, uint32_t n_tokens, void *d_k,
                             void *d_v, int elem, uint32_t *d_status, void *stream);

/* -- Attention over the cache -----------------------------------------------
 * Rows d_starts[b] .. d_starts[b + 1] of q are the last tokens of request b,
 * whose d_lens[b] keys and values (its own among them) are in the blocks
 * d_table[b, 0 ..]; heads h * G .. h * G + G - 1 of q read head h of the
 * cache (G = n_heads / cache->n_heads):
 *     out[t, j] = sum_i softmax_i(scale * q[t, j] . k_i) v_i
 * over i <= position of t (causal; every i < d_lens[b] otherwise) and, with a
 * window, i > position - window; table entries of blocks that no row of the
 * request sees are not looked at, and what their slots hold does not matter.  A row that sees nothing (d_lens[b] = 0, or
 * more rows than d_lens[b]) becomes 0 and its lse -infinity.  Rows outside
 * every request are left as they were; where starts descend, rows that two
 * requests claim get either one's result, or all rows are left (recorded).
 * q and out are bf16 or f16 (elem), head_dim consecutive elements, strides in
 * elements, q rows 16-byte aligned.  Elements of out have a place each, and it
 * shares none with q unless it is q, strides and all.  Codes enter the products exactly, sums
 * and the softmax are fp32; for the second product a softmax weight times its
 * block's value scale is rounded to f16: by up to 2^-11 of it, and below 2^-21
 * of the row's largest by up to 2^-32 of that.  out is rounded once.  Value
 * blocks with a scale below 2^-80 count as 0.  A key is not counted in the
 * softmax's sum where its weight times its value scale (2^-80 at least) is less
 * than 2^-130 of the row's largest such product; while the value scales that a
 * row sees are below 2^26 that is what fp32 sums do not hold either.  Codes of e4m3 caches are finite (hxq_cuda_kv_append
 * writes no others; slots that no request reads may hold anything).
 * d_lse (optional): [n_rows, n_heads] fp32, natural log of the softmax sums.
 * max_new: the most rows of any request; it only chooses the kernel, results
 * hold for any value.  workspace: hxq_cuda_kv_attention_workspace bytes,
 * 16-byte aligned, contents don't matter before or after; calls that may
 * overlap in time need one each.  At most HXQ_ATTENTION_MAX_REQUESTS requests;
 * n_blocks * n_heads * block_tokens < 2^31. */
#define HXQ_ATTENTION_MAX_REQUESTS 8192
typedef struct {
    const void    *d_q;
    void          *d_out;
    float         *d_lse;
    int64_t        q_stride_t, q_stride_h, out_stride_t, out_stride_h;
    const int32_t *d_starts, *d_lens, *d_table;
    uint32_t       n_requests, n_rows, n_heads, table_width;
    uint32_t       max_new, window;   /* window 0: no limit */
    float          scale;
    int            elem, causal;
} hxq_kv_attention_t;
size_t hxq_cuda_kv_attention_workspace(const hxq_kv_cache_t *cache, const hxq_kv_attention_t *args);
hxq_error_t hxq_cuda_kv_attention(const hxq_kv_cache_t *cache, const hxq_kv_attention_t *args, void *d_workspace,
                                  size_t workspace_bytes, uint32_t *d_status, void *stream);

/* -- Low-rank adapters beside a shared projection ----------------------------
 * For every token t with adapter a:
 *     out[t] = y[t] + scales[a] * (x[t] A_a^T) B_a^T,
 * and out[t] = y[t] for tokens without one.  A [n_adapters, rank,
 * in_features] and B [n_adapters, out_features, rank] bf16, contiguous,
 * 16-byte aligned; adapters of a smaller rank are padded with zeros.  rank a
 * multiple of 8, at most 128; in_features a multiple of 8.
 *
 * The plan sorts the tokens of a step by adapter, once for all projections of
 * the step: request b (rows d_starts[b] .. d_starts[b + 1]) uses d_adapters[b],
 * negative: none.  d_order [n_tokens] receives the sorted token rows, d_tiles
 * [hxq_lora_tiles(B, n_adapters, n_tokens)] groups of up to HXQ_LORA_TILE
 * tokens of one adapter.  Tokens behind d_starts[B] belong to no group and
 * their rows of out are left as they were. */
#define HXQ_LORA_TILE 64
#define HXQ_LORA_MAX_ADAPTERS 4096
#define HXQ_LORA_MAX_REQUESTS 8192
typedef struct { int32_t adapter, first, count, zero; } hxq_lora_tile_t;
uint32_t hxq_lora_tiles(uint32_t B, uint32_t n_adapters, uint32_t n_tokens);
hxq_error_t hxq_cuda_lora_plan(const int32_t *d_starts, const int32_t *d_adapters, uint32_t B, uint32_t n_adapters,
                               uint32_t n_tokens, int32_t *d_order, hxq_lora_tile_t *d_tiles, uint32_t *d_status,
                               void *stream);
typedef struct {
    const uint16_t *d_a, *d_b;   /* bf16 */
    const float    *d_scales;    /* [n_adapters] */
    uint32_t        n_adapters, rank, in_features, out_features;
} hxq_lora_t;
/* x: bf16 [n_tokens] rows of in_features, ldx elements apart (a multiple of
 * 8, 16-byte aligned); y, out: fp32 rows of out_features, ldy and ldo apart;
 * out may be y, ldo then being ldy, and shares no element with it otherwise;
 * rows of out do not overlap.  n_requests is the B of the plan.  x A^T is summed in fp32 and
 * enters the second product as three bf16 parts (together its 24 bits).
 * workspace: hxq_cuda_lora_workspace bytes, 16-byte aligned, contents don't
 * matter; calls that may overlap in time need one each. */
size_t hxq_cuda_lora_workspace(const hxq_lora_t *adapters, uint32_t n_requests, uint32_t n_tokens);
hxq_error_t hxq_cuda_lora(const hxq_lora_t *adapters, const uint16_t *d_x, int64_t ldx, const float *d_y, int64_t ldy,
                          float *d_out, int64_t ldo, uint32_t n_requests, uint32_t n_tokens, const int32_t *d_order,
                          const hxq_lora_tile_t *d_tiles, void *d_workspace, size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* HXQ_SERVING_H */
