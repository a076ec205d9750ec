/*
 * pulsar_paged.h -- C ABI of the paged key-value cache operators and of the
 * log probabilities of given tokens, in libpulsar_w4a16.so (gfx950).
 *
 * The conventions of pulsar_w4a16.h: every tensor argument is a device pointer,
 * every size and stride an element count unless it says bytes, every call is
 * asynchronous on `stream`, returns 0 or a negative PW4_ERR_* status, allocates
 * nothing and may be captured into a graph.  Scratch comes in through
 * (workspace, workspace_bytes), sized by the matching *_workspace_size query,
 * 16-byte aligned; it needs no clearing, and calls that share it must be ordered.
 *
 * The cache.  A pool of pages holds, per layer, keys and values of page_size
 * tokens a page.  Sequence b's token j lies in page block_tables[b][j /
 * page_size] at row j % page_size.  The book-keeping is on the device, in int32:
 *   ref_counts   [pages]         how many sequences hold the page, 0: free
 *   block_tables [rows, width]   each row's pages in order, -1 after its last
 *   seq_lens     [rows]          tokens of each row
 * so a serving step needs no host wait.  What a kernel reads from them is
 * checked against the pool before it is used as an address: a page id outside
 * the pool reads the last page (attention), or is passed over (everything else).
 */
#ifndef PULSAR_PAGED_H
#define PULSAR_PAGED_H

#include "pulsar_w4a16.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---------------------------------------------------------------------------
 * paged_attention: attention of the newest tokens of each sequence over its
 * pages.  Query i of sequence b, of its n_b = cu_q[b+1] - cu_q[b] new tokens,
 * stands at position p = seq_lens[b] - n_b + i (the new tokens' keys and values
 * are in the cache already) and sees key j where j <= p and, with window > 0,
 * j > p - window:
 *   s_j = scale * q . k_j       with softcap c > 0:  c * tanh(s_j / c)
 *   lse = ln sum_j e^{s_j},  out = sum_j e^{s_j - lse} v_j
 * A query that sees no key gets out = 0 and lse = -inf, and so do the rows of q
 * past cu_q[batch] and those of queries past max_q_len.  Keys that no query of their sequence sees may hold
 * anything, NaN included.
 *
 * Heads are grouped: query head h reads key-value head h / (q_heads / kv_heads).
 * Sums and softmax statistics are fp32; the probabilities are rounded to the
 * cache's type for the product with the values.
 *   q        [num_tokens, q_heads, head_dim], strides q_token_stride and
 *            q_head_stride, head_dim contiguous
 *   k_cache, v_cache  [num_pages, page_size, kv_heads, head_dim] by the strides
 *            page_stride, row_stride, kv_head_stride, head_dim contiguous
 *   out      [num_tokens, q_heads, head_dim] contiguous, lse [num_tokens,
 *            q_heads] fp32 or NULL
 *   max_q_len, max_seq_len  upper bounds of n_b and seq_lens[b]: the grid is
 *            sized by them, longer sequences are cut to them (keys past
 *            max_seq_len are not seen, queries past max_q_len come out empty)
 * scale and softcap are finite.  A sequence has fewer than 2^31 - 1024 rows (new
 * tokens times the query heads of a key-value head).  head_dim: a multiple of 8 up to 256.  Pointers
 * 16-byte aligned, strides multiples of 8, row_stride below 2^24. */
typedef struct pw4_paged_attention_args {
    const void* q;
    const void* k_cache;
    const void* v_cache;
    const int32_t* block_tables; /* [batch, table_width], rows table_stride apart */
    const int32_t* seq_lens;     /* [batch] */
    const int32_t* cu_q;         /* [batch + 1], ascending from 0 */
    void* out;
    float* lse;
    int64_t num_tokens, batch, q_heads, kv_heads, head_dim;
    int64_t num_pages, page_size, table_width, table_stride;
    int64_t q_token_stride, q_head_stride, page_stride, row_stride, kv_head_stride;
    int64_t max_q_len, max_seq_len;
    int64_t window;
    float scale, softcap;
    int dtype; /* of q, both caches and out: PW4_DTYPE_F16 or PW4_DTYPE_BF16 */
} pw4_paged_attention_args;
size_t pw4_paged_attention_workspace_size(const pw4_paged_attention_args* args);
int pw4_paged_attention(const pw4_paged_attention_args* args, void* workspace, size_t workspace_bytes,
                        pw4_stream_t stream);

/* ---------------------------------------------------------------------------
 * paged_cache_extend: room for new tokens.  Row b gets n_b = cu_q[b+1] - cu_q[b]
 * of them: the pages that its last page does not hold are the pool's
 * lowest-numbered free ones, dealt to the rows in order; seq_lens grows, and
 * slots[t] (int64 [num_tokens]) is token t's place page * page_size + row, -1 for
 * t past cu_q[rows].  All or nothing: where the pool has too few free pages or a
 * table too few columns nothing changes, every slot is -1 and *missing (int32) is
 * the number of pages that the pool lacks plus the columns that the tables lack
 * (2^18 of a row at most); else it is 0.  rows up to 4096. */
int pw4_paged_cache_extend(int32_t* ref_counts, int64_t num_pages, int32_t* block_tables, int64_t table_width,
                           int64_t table_stride, int32_t* seq_lens, const int32_t* cu_q, int64_t rows,
                           int64_t num_tokens, int64_t page_size, int64_t* slots, int32_t* missing,
                           pw4_stream_t stream);

/* paged_cache_write: key and value of token t into slot slots[t] of one layer's
 * caches; a slot outside the pool is passed over.  k and v are [num_tokens,
 * kv_heads, head_dim] by k_token_stride, k_head_stride (and v's).  Any 16-bit
 * type; no two tokens may name one slot. */
int pw4_paged_cache_write(const void* k, const void* v, void* k_cache, void* v_cache, const int64_t* slots,
                          int64_t num_tokens, int64_t kv_heads, int64_t head_dim, int64_t k_token_stride,
                          int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride, int64_t num_pages,
                          int64_t page_size, int64_t page_stride, int64_t row_stride, int64_t kv_head_stride,
                          pw4_stream_t stream);

/* A pool that the page operators move whole pages of: `planes` of them (keys and
 * values of every layer), each of num_pages pages of page_bytes contiguous bytes,
 * plane_stride_bytes and page_stride_bytes apart. */
typedef struct pw4_page_pool {
    void* base;
    int64_t planes, num_pages, page_bytes, plane_stride_bytes, page_stride_bytes;
} pw4_page_pool;

/* paged_cache_copy: page dst[i] = page src[i] in every plane, i < n.  Pairs with a
 * page outside the pool are passed over.  No page may be a dst twice, or a dst and
 * a src. */
int pw4_paged_cache_copy(const pw4_page_pool* pool, const int32_t* src, const int32_t* dst, int64_t n,
                         pw4_stream_t stream);

/* paged_cache_fork: row dst_rows[i] becomes a copy of row src_rows[i], i < n.  Full
 * pages are shared (their count grows); a last page in part filled is copied into
 * the lowest-numbered free page, in the order of i, so that both rows can go on
 * writing.  A source may appear many times; each destination appears once, is no
 * source, and is empty (what it held is not given back).  All or nothing, as
 * paged_cache_extend: *missing is the number of free pages that the pool lacks.
 * A pair with a row outside the table is passed over.  n up to 4096. */
size_t pw4_paged_cache_fork_workspace_size(int64_t n);
int pw4_paged_cache_fork(const pw4_page_pool* pool, int32_t* ref_counts, int32_t* block_tables, int64_t rows,
                         int64_t table_width, int64_t table_stride, int32_t* seq_lens, const int32_t* src_rows,
                         const int32_t* dst_rows, int64_t n, int64_t page_size, int32_t* missing, void* workspace,
                         size_t workspace_bytes, pw4_stream_t stream);

/* paged_cache_free: rows give their pages back (a page is free once no row holds
 * it), their tables become -1 and their lengths 0.  A row named twice is freed once. */
int pw4_paged_cache_free(int32_t* ref_counts, int64_t num_pages, int32_t* block_tables, int64_t rows,
                         int64_t table_width, int64_t table_stride, int32_t* seq_lens, const int32_t* which, int64_t n,
                         pw4_stream_t stream);

/* paged_cache_compact: moves pages so that the *used pages in use are the pages
 * [0, *used): the i-th free page below that takes the i-th used page at or above
 * it, in every plane, and tables and counts are renamed.  No page moves that need
 * not. */
size_t pw4_paged_cache_compact_workspace_size(int64_t num_pages);
int pw4_paged_cache_compact(const pw4_page_pool* pool, int32_t* ref_counts, int32_t* block_tables, int64_t rows,
                            int64_t table_width, int64_t table_stride, int32_t* used, void* workspace,
                            size_t workspace_bytes, pw4_stream_t stream);

/* ---------------------------------------------------------------------------
 * token_logprobs: over each row x of logits [num_tokens, vocab] (fp16, bf16 or
 * fp32, rows row_stride apart), with lse = ln sum e^x:
 *   logprobs  [num_tokens] fp32  x[targets[t]] - lse, 0 where the target is
 *             outside [0, vocab) (no token given)
 *   ranks     [num_tokens] int64 tokens ahead of the given one: a greater logit,
 *             or an equal one and a lower index (0: the likeliest), -1 for none
 *   entropy   [num_tokens] fp32  -sum p ln p
 *   top_logprobs, top_ids  [num_tokens, top_k] fp32 and int64: the likeliest
 *             tokens, equal logits by lower index first
 * Logits of -inf have probability 0 and add nothing to the entropy.  A row whose
 * logits are all -inf has log probabilities -inf and entropy 0.  A row with a NaN
 * or +inf has NaN log probabilities and entropy; among its top tokens a NaN
 * counts as -inf, and its ranks count the logits that compare greater.
 * top_k from 0 to 32, at most vocab. */
size_t pw4_token_logprobs_workspace_size(int64_t num_tokens, int64_t vocab, int64_t top_k);
int pw4_token_logprobs(const void* logits, int dtype, int64_t num_tokens, int64_t vocab, int64_t row_stride,
                       const int64_t* targets, int64_t top_k, float* logprobs, int64_t* ranks, float* entropy,
                       float* top_logprobs, int64_t* top_ids, void* workspace, size_t workspace_bytes,
                       pw4_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* PULSAR_PAGED_H */
