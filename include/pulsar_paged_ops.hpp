// pulsar_paged_ops.hpp -- the at::Tensor operator API of the paged key-value
// cache and of the log probabilities of given tokens, beside the W4A16 operators
// of pulsar_w4a16_ops.hpp and in the same library.  Each function checks its
// arguments (TORCH_CHECK -> c10::Error), allocates its outputs and scratch with
// the caching allocator, and launches on the current HIP stream through the C ABI
// of pulsar_paged.h, which says what each computes.
#pragma once

#include <ATen/ATen.h>

#include <optional>
#include <tuple>

namespace pulsar {

// Attention of the newest tokens q [T, Hq, D] of each sequence over k_cache and
// v_cache [P, page, Hkv, D].  Returns (out [T, Hq, D], lse fp32 [T, Hq], empty
// unless return_lse).  scale defaults to 1 / sqrt(D); window and softcap 0: none.
std::tuple<at::Tensor, at::Tensor> paged_attention_cuda(const at::Tensor& q, const at::Tensor& k_cache,
                                                        const at::Tensor& v_cache, const at::Tensor& block_tables,
                                                        const at::Tensor& seq_lens, const at::Tensor& cu_q,
                                                        int64_t max_q_len, int64_t max_seq_len,
                                                        std::optional<double> scale, int64_t window, double softcap,
                                                        bool return_lse);

// Pages for cu_q's new tokens: (slots int64 [num_tokens], missing int32 [1]).
std::tuple<at::Tensor, at::Tensor> paged_cache_extend_cuda(at::Tensor& ref_counts, at::Tensor& block_tables,
                                                           at::Tensor& seq_lens, const at::Tensor& cu_q,
                                                           int64_t num_tokens, int64_t page_size);

// k and v [T, Hkv, D] into the slots of one layer's caches.
void paged_cache_write_cuda(const at::Tensor& k, const at::Tensor& v, at::Tensor& k_cache, at::Tensor& v_cache,
                            const at::Tensor& slots);

// Whole pages of a pool [planes, P, page, ...]: dst[i] = src[i] in every plane.
void paged_cache_copy_cuda(at::Tensor& pool, const at::Tensor& src_pages, const at::Tensor& dst_pages);

// Rows dst become copies of rows src; returns missing int32 [1].
at::Tensor paged_cache_fork_cuda(at::Tensor& pool, at::Tensor& ref_counts, at::Tensor& block_tables,
                                 at::Tensor& seq_lens, const at::Tensor& src_rows, const at::Tensor& dst_rows);

void paged_cache_free_cuda(at::Tensor& ref_counts, at::Tensor& block_tables, at::Tensor& seq_lens,
                           const at::Tensor& rows);

// Moves the pages in use to the pool's start; returns how many are, int32 [1].
at::Tensor paged_cache_compact_cuda(at::Tensor& pool, at::Tensor& ref_counts, at::Tensor& block_tables);

// (logprobs [T], ranks int64 [T], entropy [T], top_logprobs [T, k], top_ids int64 [T, k]).
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> token_logprobs_cuda(const at::Tensor& logits,
                                                                                           const at::Tensor& targets,
                                                                                           int64_t top_k);

}  // namespace pulsar
