"""PagedKVCache.append with tables of rotations that end before a row does."""

import pytest
import torch

from paged_case import DEV, gen
from pulsar_amd import ops
from pulsar_amd.paged import PagedKVCache

B = torch.bfloat16


def _cache(bits, **kw):
    args = dict(layers=2, pages=40, page_size=8, kv_heads=2, head_dim=64, rows=4, max_seq_len=128, dtype=B, bits=bits)
    cache = PagedKVCache(**{**args, **kw})
    cache.pool.fill_(1)
    return cache


def _qkv(t, seed=1):
    return [torch.randn(t, h, 64, generator=gen(seed)).to(B).to(DEV) for h in (4, 2, 2)]


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 4])
def test_a_table_shorter_than_a_row_is_refused(bits):
    """Its last tokens would not be stored, and their places would be read as they were."""
    cache = _cache(bits)
    step = cache.extend([9, 0, 3, 0])
    qkv = _qkv(12)
    before = cache.pool.clone()
    for rows in (8, 1, 0):
        with pytest.raises(ValueError, match="rope.*9"):
            cache.append(0, *qkv, step, ops.rope_table(rows, 64))
        assert torch.equal(cache.pool, before)
    # the step stands: with a table that is long enough it goes on, layer by layer
    want = _cache(bits)
    other = want.extend([9, 0, 3, 0])
    for layer in range(2):
        a = cache.append(layer, *qkv, step, ops.rope_table(9, 64))
        assert torch.equal(a, want.append(layer, *qkv, other, ops.rope_table(100, 64)))
        assert torch.equal(cache.pool, want.pool)
        with pytest.raises(ValueError, match="rope"):
            cache.append(layer, *qkv, step, ops.rope_table(8, 64))
    # rows without new tokens do not count
    step = cache.extend([0, 2, 0, 0])
    cache.append(0, *_qkv(2), step, ops.rope_table(2, 64))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 4])
def test_bounds_that_are_too_high_refuse_nothing(bits):
    """The host's bounds of rows also count what a full pool refused and rows that a reordering gave back."""
    cache = _cache(bits, pages=3)
    cache.extend([10, 0, 0, 0])
    for _ in range(3):
        assert int(cache.extend([30, 0, 0, 0]).missing) > 0
    step = cache.extend([1, 0, 0, 0])
    assert step.max_seq_len > 11
    cache.append(0, *_qkv(1), step, ops.rope_table(11, 64))
    with pytest.raises(ValueError, match="rope.*11"):
        cache.append(0, *_qkv(1), step, ops.rope_table(10, 64))
    # a step that was refused stores nothing, whatever its tokens' positions would be
    step = cache.extend([30, 0, 0, 0])
    assert int(step.missing) > 0
    before = cache.pool.clone()
    cache.append(0, *_qkv(30), step, ops.rope_table(20, 64))
    assert torch.equal(cache.pool, before)

    cache = _cache(bits)
    cache.extend([20, 0, 0, 0])
    cache.reorder(torch.zeros(1, dtype=torch.int32, device=DEV), [0], [1])
    step = cache.extend([5, 0, 0, 0])  # row 0 begins again
    assert step.max_seq_len > 5
    cache.append(0, *_qkv(5), step, ops.rope_table(5, 64))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 4])
def test_a_table_that_the_bounds_fit_does_not_wait(bits):
    cache = _cache(bits)
    rope, (q, k, v) = ops.rope_table(9, 64), _qkv(4)

    def use():
        for layers in range(2):
            step = cache.extend([4, 0, 0, 0])
            for layer in range(2):
                cache.append(layer, q, k, v, step, rope)
        cache.free([0])

    for _ in range(3):  # the allocators' first memory
        use()
    torch.cuda.synchronize()
    busy = torch.cuda.Event()
    torch.cuda._sleep(1 << 28)  # a tenth of a second or more
    busy.record()
    use()
    assert not busy.query()
    torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 4])
def test_an_append_in_a_graph(bits):
    """While a graph is captured nothing is read from the device, so a table is taken as it is."""
    cache = _cache(bits)
    cache.extend([6, 0, 0, 0])
    cache.reorder(torch.zeros(1, dtype=torch.int32, device=DEV), [0], [1])
    step = cache.extend([5, 0, 0, 0])
    rope, qkv = ops.rope_table(5, 64), _qkv(5)
    assert step.max_seq_len > 5
    expect = cache.append(0, *qkv, step, ops.rope_table(100, 64))
    want = cache.pool.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = cache.append(0, *qkv, step, rope)
    for _ in range(3):
        cache.pool[:, step.slots // 8] = 1
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, expect) and torch.equal(cache.pool, want)
