"""The paged cache, its attention and the token log probabilities together, as
examples/branching_decode.py runs them: against the same decoder without a cache, whose attention is
computed in 64 bits over the whole sequence at every step."""

import os
import sys

import pytest
import torch

from pulsar_amd import ops
from pulsar_amd.paged import PagedKVCache

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
import branching_decode as example  # noqa: E402


def _dense(layer, q, k, v):
    """Causal attention of a whole sequence, on the host in 64 bits."""
    g = q.shape[1] // k.shape[1]
    q, k, v = (t.cpu().double().transpose(0, 1) for t in (q, k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)))
    s = q @ k.transpose(1, 2) * q.shape[-1] ** -0.5
    s = s.masked_fill(torch.ones(s.shape[-2:], dtype=torch.bool).triu(1), float("-inf"))
    return (torch.softmax(s, -1) @ v).transpose(0, 1).half().cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("page,prompt,beams,steps", [(16, 100, 4, 8), (8, 17, 2, 5), (64, 130, 3, 4)])
def test_beams_score_as_without_a_cache(page, prompt, beams, steps):
    model = example.Decoder(seed=page)
    cache = PagedKVCache(layers=2, pages=200, page_size=page, kv_heads=2, head_dim=64, rows=2 * beams, max_seq_len=256,
                         dtype=torch.float16)
    tokens = torch.randint(0, 1003, (prompt,), device="cuda:0", generator=torch.Generator("cuda:0").manual_seed(3))
    found, scored = example.beam_search(model, cache, tokens, beams, steps)
    assert len(found) == beams and all(len(t) == steps for _, t in found)
    assert [s for s, _ in found] == sorted((s for s, _ in found), reverse=True)
    for score, new in found:
        whole = torch.cat([tokens, torch.tensor(new, device="cuda:0")])
        logits = model.forward(whole, torch.arange(len(whole), device="cuda:0"), _dense)
        lp = torch.log_softmax(logits.double(), -1)
        want = lp[torch.arange(len(whole) - 1), whole[1:]]
        # fp16 activations through two layers either way: each logit is a sum of 512 products of
        # rounded factors near 1 with weights of 3 / sqrt(512); some units of 2^-11 of 3 sigma
        assert abs(score - float(want[prompt - 1:].sum())) < 0.03 * steps
        assert float((scored[:-1].double() - want[:prompt - 1]).abs().max()) < 0.1
    # only the beams' rows hold pages; compacting packs them and changes no result
    lens = cache.seq_lens.tolist()
    assert sorted(lens) == [0] * beams + [prompt + steps - 1] * beams
    held = {p for r in cache.block_tables.tolist() for p in r if p >= 0}
    assert int((cache.ref_counts > 0).sum()) == len(held)
    q = torch.randn(beams, 8, 64, device="cuda:0").half()
    live = [r for r, n in enumerate(lens) if n]
    args = (torch.arange(beams + 1, dtype=torch.int32, device="cuda:0"), 1, max(lens))

    def look():
        return ops.paged_attention(q, *cache.layer(1), cache.block_tables[live], cache.seq_lens[live], *args)

    before = look()
    assert int(cache.compact()) == len(held)
    assert {p for r in cache.block_tables.tolist() for p in r if p >= 0} == set(range(len(held)))
    assert torch.equal(before, look())
    cache.free(list(range(cache.rows)))
    assert int(cache.ref_counts.abs().sum()) == 0


@pytest.mark.gpu
def test_a_full_pool_takes_nothing():
    cache = PagedKVCache(layers=1, pages=3, page_size=8, kv_heads=1, head_dim=64, rows=2, max_seq_len=64)
    first = cache.extend([20, 0])
    assert int(first.missing) == 0
    second = cache.extend([1, 9])
    assert int(second.missing) == 2 and cache.seq_lens.tolist() == [20, 0] and set(second.slots.tolist()) == {-1}
    assert int(cache.fork([0], [1])) == 1


def test_refusals():
    with pytest.raises(ValueError, match="positive"):
        PagedKVCache(1, 0, 8, 1, 64, 1, 64, device="cpu")
    with pytest.raises(ValueError, match="dtype"):
        PagedKVCache(1, 4, 8, 1, 64, 1, 64, dtype=torch.float32, device="cpu")
    cache = PagedKVCache(1, 4, 8, 1, 64, 2, 64, device="cpu")
    with pytest.raises(ValueError, match="counts"):
        cache.extend([1])
    with pytest.raises(ValueError, match="counts"):
        cache.extend([1, -1])
    with pytest.raises(ValueError, match="rows"):
        cache.free([2])
    with pytest.raises(ValueError, match="destination"):
        cache.fork([0, 1], [1, 0])


@pytest.mark.gpu
def test_forking_onto_rows_in_use_gives_their_pages_back():
    cache = PagedKVCache(layers=1, pages=12, page_size=8, kv_heads=1, head_dim=64, rows=4, max_seq_len=64)
    cache.extend([20, 17, 9, 0])
    assert int((cache.ref_counts > 0).sum()) == 8
    assert int(cache.fork([0, 0], [1, 3])) == 0
    assert cache.seq_lens.tolist() == [20, 20, 9, 20]
    tables = [[p for p in r if p >= 0] for r in cache.block_tables.tolist()]
    assert tables[1][:2] == tables[3][:2] == tables[0][:2] and [len(t) for t in tables] == [3, 3, 2, 3]
    held = torch.bincount(torch.tensor([p for r in tables for p in r]), minlength=12)
    assert torch.equal(held.int(), cache.ref_counts.cpu())  # every count is of a row that is there
    cache.free([0, 1, 2, 3])
    assert int(cache.ref_counts.abs().sum()) == 0


@pytest.mark.gpu
def test_a_beam_search_that_runs_out_of_pages_says_so():
    model = example.Decoder(seed=1)
    tokens = torch.randint(0, 1003, (33,), device="cuda:0", generator=torch.Generator("cuda:0").manual_seed(3))

    def search(pages, most=64):
        cache = PagedKVCache(layers=2, pages=pages, page_size=16, kv_heads=2, head_dim=64, rows=8, max_seq_len=most,
                             dtype=torch.float16)
        return example.beam_search(model, cache, tokens, beams=4, steps=3)

    search(pages=10)  # 2 full pages shared by all, and a last one for each of 4 beams and each of their children
    for pages in (9, 6, 2):  # in a later fork, in the first one, in the prompt
        with pytest.raises(RuntimeError, match="pages"):
            search(pages)
    with pytest.raises(RuntimeError, match="pages"):
        search(pages=40, most=32)  # no column for the prompt's last token


@pytest.mark.gpu
def test_the_bound_of_a_row_is_held_to_its_table_and_its_length():
    cache = PagedKVCache(layers=1, pages=3, page_size=8, kv_heads=1, head_dim=64, rows=2, max_seq_len=32)
    cache.extend([20, 0])
    for _ in range(5):
        step = cache.extend([10, 0])  # refused
        assert int(step.missing) == 1
    assert step.max_seq_len == 32  # what the row's table holds
    assert cache.lengths() == [20, 0]  # and after this the bounds are the lengths
    step = cache.extend([1, 0])
    assert int(step.missing) == 0 and step.max_seq_len == 21


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [4, 4000])
def test_no_method_waits_for_the_device(rows):
    """While the device is busy with something else each returns."""
    cache = PagedKVCache(layers=1, pages=8 * rows, page_size=8, kv_heads=1, head_dim=64, rows=rows, max_seq_len=64)
    k = torch.zeros(rows, 1, 64, dtype=torch.bfloat16, device="cuda:0")
    half = list(range(rows // 2))

    def use():
        step = cache.extend([1] * rows)
        cache.write(0, k, k, step)
        cache.attend(0, k, step)
        cache.fork(half, [r + rows // 2 for r in half])
        cache.free(list(range(rows)))
        cache.compact()

    for _ in range(3):  # the allocators' first memory
        use()
    torch.cuda.synchronize()
    busy = torch.cuda.Event()
    torch.cuda._sleep(1 << 28)  # a tenth of a second or more
    busy.record()
    use()
    assert not busy.query()
    torch.cuda.synchronize()
    assert cache.lengths() == [0] * rows and int(cache.ref_counts.abs().sum()) == 0
