"""Python wrappers and fake (meta) kernels for the W4A16, paged-cache and log-probability ops.

Same wrapper names, argument meaning and fake-kernel output shapes as the
reference pulsar/src/pulsar/core/ops.py:117-165,369-445, so code written
against `pulsar.core.ops` switches by importing `pulsar_amd.ops`.  The ops
themselves are registered by _pulsar_w4a16_torch.so (torch.ops.pulsar.*).

The paged cache.  A pool holds pages of page_size tokens; row b's token j lies in page
block_tables[b, j // page_size] at place j % page_size.  The book-keeping is int32 tensors on the
device, changed in place: ref_counts [pages] (0: free), block_tables [rows, width] (-1 past a
row's last page) and seq_lens [rows].  No call waits for the device, and each can be captured
into a graph.
"""

from __future__ import annotations

import torch

# MARLIN tiling constants; must match the C ABI's size rule (pw4_marlin_words).
_MARLIN_BN = 64
_MARLIN_BK = 64


def _gemm_w4a16_fake(x, weight_packed, weight_scale, group_size):
    return x.new_empty((x.shape[0], weight_packed.shape[0]))


def _gemm_w4a16_split_fake(x, weight_packed, weight_scale, group_size, num_splits):
    return x.new_empty((x.shape[0], weight_packed.shape[0]))


def _repack_w4a16_fake(weight_packed, weight_scale, group_size):
    n = weight_packed.shape[0]
    k = weight_packed.shape[1] * 8
    npad = -(-n // _MARLIN_BN) * _MARLIN_BN
    kpad = -(-k // _MARLIN_BK) * _MARLIN_BK
    weight_marlin = weight_packed.new_empty((npad * kpad // 8,))
    scale_marlin = weight_scale.new_empty((k // group_size, n), dtype=torch.float32)
    return weight_marlin, scale_marlin


def _gemm_w4a16_marlin_fake(x, weight_marlin, scale_marlin, group_size):
    return x.new_empty((x.shape[0], scale_marlin.shape[1]))


def _gemm_w4a16_marlin_split_fake(x, weight_marlin, scale_marlin, group_size, num_splits):
    return x.new_empty((x.shape[0], scale_marlin.shape[1]))


def _repack_w4a16_gptq_fake(qweight, g_idx, group_size):
    k = qweight.shape[0] * 8
    n = qweight.shape[1]
    npad = -(-n // _MARLIN_BN) * _MARLIN_BN
    kpad = -(-k // _MARLIN_BK) * _MARLIN_BK
    weight_marlin = qweight.new_empty((npad * kpad // 8,))
    perm = qweight.new_empty((k if g_idx is not None else 0,))
    return weight_marlin, perm


def _gemm_w4a16_gptq_fake(x, weight_marlin, scales, qzeros, perm, group_size):
    return x.new_empty((x.shape[0], scales.shape[1]))


def _gemm_w4a16_silu_mul_fake(x, weight_marlin, scales, qzeros, perm, group_size):
    return x.new_empty((x.shape[0], scales.shape[1] // 2))


def _paged_attention_fake(q, k_cache, v_cache, block_tables, seq_lens, cu_q, max_q_len, max_seq_len, scale=None,
                          window=0, softcap=0.0, return_lse=False):
    lse = q.new_empty((q.shape[0] if return_lse else 0, q.shape[1]), dtype=torch.float32)
    return q.new_empty(q.shape), lse


def _paged_cache_extend_fake(ref_counts, block_tables, seq_lens, cu_q, num_tokens, page_size):
    return block_tables.new_empty((num_tokens,), dtype=torch.int64), block_tables.new_empty((1,))


def _paged_cache_write_fake(k, v, k_cache, v_cache, slots):
    return None


def _paged_cache_copy_fake(pool, src_pages, dst_pages):
    return None


def _paged_cache_fork_fake(pool, ref_counts, block_tables, seq_lens, src_rows, dst_rows):
    return block_tables.new_empty((1,))


def _paged_cache_free_fake(ref_counts, block_tables, seq_lens, rows):
    return None


def _paged_cache_compact_fake(pool, ref_counts, block_tables):
    return block_tables.new_empty((1,))


def _token_logprobs_fake(logits, targets, top_k):
    t = logits.shape[0]
    f32 = [logits.new_empty(shape, dtype=torch.float32) for shape in ((t,), (t,), (t, top_k))]
    return f32[0], targets.new_empty((t,)), f32[1], f32[2], targets.new_empty((t, top_k))


def _register_fakes() -> None:
    fakes = {
        "pulsar::gemm_w4a16": _gemm_w4a16_fake,
        "pulsar::gemm_w4a16_split": _gemm_w4a16_split_fake,
        "pulsar::repack_w4a16": _repack_w4a16_fake,
        "pulsar::gemm_w4a16_marlin": _gemm_w4a16_marlin_fake,
        "pulsar::gemm_w4a16_marlin_split": _gemm_w4a16_marlin_split_fake,
        "pulsar::repack_w4a16_gptq": _repack_w4a16_gptq_fake,
        "pulsar::gemm_w4a16_gptq": _gemm_w4a16_gptq_fake,
        "pulsar::gemm_w4a16_silu_mul": _gemm_w4a16_silu_mul_fake,
        "pulsar::paged_attention": _paged_attention_fake,
        "pulsar::paged_cache_extend": _paged_cache_extend_fake,
        "pulsar::paged_cache_write": _paged_cache_write_fake,
        "pulsar::paged_cache_copy": _paged_cache_copy_fake,
        "pulsar::paged_cache_fork": _paged_cache_fork_fake,
        "pulsar::paged_cache_free": _paged_cache_free_fake,
        "pulsar::paged_cache_compact": _paged_cache_compact_fake,
        "pulsar::token_logprobs": _token_logprobs_fake,
    }
    for name, func in fakes.items():
        torch.library.register_fake(name, func)


_register_fakes()


def gemm_w4a16(x: torch.Tensor, weight_packed: torch.Tensor, weight_scale: torch.Tensor,
               group_size: int) -> torch.Tensor:
    """Fused w4a16 dequant-GEMM computing y = x @ dequant(W)^T.

    y[m, n] = sum_k x[m, k] * int4(weight_packed[n, k]) * weight_scale[n, k // group_size].

    Args:
        x: [M, K] fp16 or bf16, contiguous.
        weight_packed: int32 [N, K/8]; column k in nibble k % 8 of word [n, k // 8],
            LSB-first, two's complement in [-8, 7].
        weight_scale: [N, K/group_size], any float dtype (upcast to fp32).
        group_size: quantization group along K (multiple of 16; K a multiple of it).

    Returns:
        y [M, N] in x's dtype.
    """
    return torch.ops.pulsar.gemm_w4a16(x, weight_packed, weight_scale, group_size)


def gemm_w4a16_split(x, weight_packed, weight_scale, group_size: int, num_splits: int) -> torch.Tensor:
    """gemm_w4a16 with the K-split count forced to num_splits (split + combine path)."""
    return torch.ops.pulsar.gemm_w4a16_split(x, weight_packed, weight_scale, group_size, num_splits)


def repack_w4a16(weight_packed: torch.Tensor, weight_scale: torch.Tensor,
                 group_size: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Repack the compressed-tensors packing into the MARLIN fragment layout.

    Returns (weight_marlin int32 [Npad*Kpad/8], scale_marlin fp32 [K/group_size, N]);
    Npad / Kpad are N / K rounded up to 64.  Bit-identical to the reference packer.
    """
    return torch.ops.pulsar.repack_w4a16(weight_packed, weight_scale, group_size)


def gemm_w4a16_marlin(x: torch.Tensor, weight_marlin: torch.Tensor, scale_marlin: torch.Tensor,
                      group_size: int) -> torch.Tensor:
    """y = x @ dequant(W)^T from (weight_marlin, scale_marlin) produced by repack_w4a16."""
    return torch.ops.pulsar.gemm_w4a16_marlin(x, weight_marlin, scale_marlin, group_size)


def gemm_w4a16_marlin_split(x, weight_marlin, scale_marlin, group_size: int, num_splits: int) -> torch.Tensor:
    """gemm_w4a16_marlin with the K-split count forced (test seam)."""
    return torch.ops.pulsar.gemm_w4a16_marlin_split(x, weight_marlin, scale_marlin, group_size, num_splits)


def repack_w4a16_gptq(qweight: torch.Tensor, g_idx: torch.Tensor | None,
                      group_size: int) -> tuple[torch.Tensor, torch.Tensor]:
    """GPTQ qweight int32 [K/8, N] (+ optional act-order g_idx [K]) -> (weight_marlin, perm).

    perm is int32 [K] (empty without g_idx): repacked row j is original row perm[j].
    """
    return torch.ops.pulsar.repack_w4a16_gptq(qweight, g_idx, group_size)


def gemm_w4a16_gptq(x: torch.Tensor, weight_marlin: torch.Tensor, scales: torch.Tensor,
                    qzeros: torch.Tensor | None, perm: torch.Tensor | None, group_size: int) -> torch.Tensor:
    """y = x[:, perm] @ ((u - z) * s)^T with scales [K/G, N] (fp16/fp32) and optional GPTQ qzeros."""
    if perm is not None and perm.numel() == 0:
        perm = None
    return torch.ops.pulsar.gemm_w4a16_gptq(x, weight_marlin, scales, qzeros, perm, group_size)


def gemm_w4a16_silu_mul(x: torch.Tensor, weight_marlin: torch.Tensor, scales: torch.Tensor,
                        qzeros: torch.Tensor | None, perm: torch.Tensor | None, group_size: int) -> torch.Tensor:
    """silu(x @ Wg^T) * (x @ Wu^T), [M, N/2], from a gate|up weight interleaved by 8 columns
    (fused columns 16j..16j+7 gate 8j..8j+7, 16j+8..16j+15 up 8j..8j+7): the reference MLP's
    at::silu(gate) * up after two at::linear calls (qwen3.cpp:116-118) as one op."""
    if perm is not None and perm.numel() == 0:
        perm = None
    return torch.ops.pulsar.gemm_w4a16_silu_mul(x, weight_marlin, scales, qzeros, perm, group_size)


# The overloads themselves: looking one up costs as much as a small operator's checks.
_paged_attention = torch.ops.pulsar.paged_attention.default
_paged_cache_compact = torch.ops.pulsar.paged_cache_compact.default
_paged_cache_copy = torch.ops.pulsar.paged_cache_copy.default
_paged_cache_extend = torch.ops.pulsar.paged_cache_extend.default
_paged_cache_fork = torch.ops.pulsar.paged_cache_fork.default
_paged_cache_free = torch.ops.pulsar.paged_cache_free.default
_paged_cache_write = torch.ops.pulsar.paged_cache_write.default
_token_logprobs = torch.ops.pulsar.token_logprobs.default


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                    seq_lens: torch.Tensor, cu_q: torch.Tensor, max_q_len: int, max_seq_len: int,
                    scale: float | None = None, window: int = 0, softcap: float = 0.0, return_lse: bool = False):
    """Attention of each sequence's newest tokens over its pages.

    The n = cu_q[b+1] - cu_q[b] new tokens of sequence b are its last ones, their keys and values
    in the cache already: query i stands at p = seq_lens[b] - n + i and sees the keys j <= p, with
    window > 0 only those j > p - window.  softcap c > 0 caps scores as c * tanh(s / c).

    Args:
        q: [T, q_heads, head_dim] fp16 or bf16, any token and head strides; head h reads key-value
            head h // (q_heads // kv_heads).
        k_cache, v_cache: [pages, page_size, kv_heads, head_dim] in q's dtype, head_dim (a multiple
            of 8 up to 256) contiguous; any other strides that keep rows 16-byte aligned.
        block_tables, seq_lens, cu_q: int32 [batch, width], [batch] and [batch + 1].
        max_q_len, max_seq_len: bounds of n and seq_lens that the host knows; keys past the latter
            are not seen, queries past the former come out empty.
        scale: defaults to 1 / sqrt(head_dim).

    Returns:
        out like q (contiguous), and with return_lse also lse = ln sum e^s, fp32 [T, q_heads].  A
        query that sees no key or is past max_q_len, and a row of q past cu_q[-1], has out 0 and
        lse -inf.
    """
    out, lse = _paged_attention(q, k_cache, v_cache, block_tables, seq_lens, cu_q, max_q_len,
                                                max_seq_len, scale, window, softcap, return_lse)
    return (out, lse) if return_lse else out


def paged_cache_extend(ref_counts: torch.Tensor, block_tables: torch.Tensor, seq_lens: torch.Tensor,
                       cu_q: torch.Tensor, num_tokens: int, page_size: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Room for cu_q[b+1] - cu_q[b] new tokens of each row: the lowest-numbered free pages, dealt to
    the rows in order.  Returns (slots int64 [num_tokens], missing int32 [1]): token t's place
    page * page_size + row.  Where pages or table columns lack nothing changes, the slots are -1 and
    missing says how many."""
    return _paged_cache_extend(ref_counts, block_tables, seq_lens, cu_q, num_tokens, page_size)


def paged_cache_write(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                      slots: torch.Tensor) -> None:
    """Stores k and v [T, kv_heads, head_dim] in the slots of one layer's caches (fp16 or bf16); a
    slot outside the caches (-1) is passed over."""
    _paged_cache_write(k, v, k_cache, v_cache, slots)


def paged_cache_copy(pool: torch.Tensor, src_pages: torch.Tensor, dst_pages: torch.Tensor) -> None:
    """pool[:, dst_pages[i]] = pool[:, src_pages[i]] over a pool [planes, pages, page_size, ...] of any
    dtype with contiguous pages.  No page may be a destination twice, or a destination and a source."""
    _paged_cache_copy(pool, src_pages, dst_pages)


def paged_cache_fork(pool: torch.Tensor, ref_counts: torch.Tensor, block_tables: torch.Tensor, seq_lens: torch.Tensor,
                     src_rows: torch.Tensor, dst_rows: torch.Tensor) -> torch.Tensor:
    """Row dst_rows[i] becomes a copy of row src_rows[i]: full pages are shared, a last page in part
    filled is copied into a free one in every plane of the pool.  A source may come many times; the
    destinations are empty rows, each named once.  Returns missing int32 [1]: the free pages that
    lacked, in which case nothing changed."""
    return _paged_cache_fork(pool, ref_counts, block_tables, seq_lens, src_rows, dst_rows)


def paged_cache_free(ref_counts: torch.Tensor, block_tables: torch.Tensor, seq_lens: torch.Tensor,
                     rows: torch.Tensor) -> None:
    """The rows give their pages back: a page is free once no row holds it."""
    _paged_cache_free(ref_counts, block_tables, seq_lens, rows)


def paged_cache_compact(pool: torch.Tensor, ref_counts: torch.Tensor, block_tables: torch.Tensor) -> torch.Tensor:
    """Moves pages so that those in use are the pool's first, and renames them in the tables: the i-th
    free page among them takes the i-th used page behind them.  Returns how many are in use, int32 [1]."""
    return _paged_cache_compact(pool, ref_counts, block_tables)


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, top_k: int):
    """Log probabilities of given tokens under logits [T, vocab] (fp16, bf16 or fp32).

    Returns (logprobs [T], ranks int64 [T], entropy [T], top_logprobs [T, top_k], top_ids int64
    [T, top_k]), computed numbers in fp32.  A rank counts the tokens ahead of the given one; equal
    logits stand by index.  targets int64 [T]; one outside the vocabulary has logprob 0 and rank -1.
    top_k is 0 to 32.
    """
    return _token_logprobs(logits, targets, top_k)
