"""Attention calls of more workgroups than a launch has threads for are refused: the device would run what is
left of the count, and leave the other sequences' outputs unwritten."""

import ctypes

import pytest

import pulsar_amd
from test_paged_attention_fp4 import _Args


@pytest.mark.parametrize("entry,page_stride", [("pw4_paged_attention", 16 * 2 * 64), ("pw4_paged_attention_fp4", 16 * 2 * 34)])
def test_more_tiles_than_a_launch_holds_are_refused(entry, page_stride):
    lib = pulsar_amd.capi()
    f = getattr(lib, entry)
    f.argtypes = [ctypes.POINTER(_Args), ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p]

    def call(batch, new, kv_heads=2, dim=64, keys=16):
        scale = dim // 64 * kv_heads // 2
        return f(ctypes.byref(_Args(
            q=4096, k_cache=4096, v_cache=4096, block_tables=4096, seq_lens=4096, cu_q=4096, out=4096, num_tokens=batch * new,
            batch=batch, q_heads=2 * kv_heads, kv_heads=kv_heads, head_dim=dim, num_pages=4, page_size=16, table_width=keys // 16,
            table_stride=keys // 16, q_token_stride=2 * kv_heads * dim, q_head_stride=dim, page_stride=page_stride * scale,
            row_stride=kv_heads * dim, kv_head_stride=dim, max_q_len=new, max_seq_len=keys, scale=1.0, dtype=1)), None, 0, None)

    # one token of each sequence: four waves a workgroup, in heads of 256 two
    assert call(2 ** 23, 1) == call(2 ** 21, 1, 8) == call(2 ** 24, 1, 2, 256) == call(2 ** 30, 1) == -2
    assert call(2 ** 30, 1, 4096) == -2
    # chunks: tiles of 128 rows
    assert call(2 ** 22, 100) == call(2 ** 22, 300) == -2  # (2^20 of 300 tokens: 5 * 2 * 2^20 of 256 threads, below 2^32)
