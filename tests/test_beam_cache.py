"""PagedKVCache in 16 and in 4 bits with the rotating append, its attention, beam selection and reordering, as
a beam search runs them: each step against the definitions in 64 bits over what each beam's history holds."""

import os
import sys

import pytest
import torch

from fp4_case import fp4_round
from paged_case import DEV, attention_ref, check_attention, gen
from pulsar_amd import ops
from pulsar_amd.paged import PagedKVCache
from test_beam_search import _check
from test_paged_append import check16, rotate_ref

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
import branching_decode as example  # noqa: E402

H, B = torch.float16, torch.bfloat16


def _cache(bits, **kw):
    args = dict(layers=2, pages=120, page_size=16, kv_heads=2, head_dim=64, rows=8, max_seq_len=256, dtype=H, bits=bits)
    return PagedKVCache(**{**args, **kw})


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dtype", [H, B])
@pytest.mark.parametrize("page,dim,heads,group,prompt,beams,steps", [
    (16, 64, 2, 4, 50, 4, 6), (7, 96, 1, 3, 20, 3, 9), (24, 128, 3, 2, 24, 5, 4), (1, 32, 1, 1, 1, 2, 5)])
def test_a_search_step_by_step(page, dim, heads, group, prompt, beams, steps, dtype, bits):
    """The rows' keys and values are kept on the host too, as the cache has to hold them: rotated and rounded
    by the append's definition."""
    layers, vocab, most = 2, 300, prompt + steps
    cache = _cache(bits, layers=layers, page_size=page, kv_heads=heads, head_dim=dim, rows=2 * beams, dtype=dtype,
                   pages=2 * beams * -(-most // page), max_seq_len=most)
    rope = ops.rope_table(most, dim)
    g = gen(page + dim)
    head = (torch.randn(heads * group * dim, vocab, generator=g) * 0.3).to(dtype).to(DEV)
    # what live[j]'s row holds: by layer, keys and values [length, heads, dim]
    held = {0: [[torch.zeros(0, heads, dim, dtype=dtype)] * 2 for _ in range(layers)]}

    def forward(rows, n):
        """n new tokens of each of rows, through the cache's layers; the last layer's output."""
        counts = [n if r in rows else 0 for r in range(cache.rows)]
        step = cache.extend(counts)
        pos = torch.arange(len(held[rows[0]][0][0]), len(held[rows[0]][0][0]) + n).repeat(len(rows))
        assert int(step.missing) == 0 and torch.equal(cache.positions(step).cpu(), pos)
        for i in range(layers):
            q, k, v = (torch.randn(n * len(rows), h, dim, generator=g).to(dtype) for h in (heads * group, heads, heads))
            if i == 0:  # views of one tensor, as a fused projection leaves them
                whole = torch.cat([q, k, v], 1).to(DEV)
                args = whole.split([heads * group, heads, heads], 1)
            else:
                args = [t.to(DEV) for t in (q, k, v)]
            qr = cache.append(i, *args, step, rope)
            check16(qr, *rotate_ref(q, rope.cpu(), pos, False), dtype)
            kr, size = rotate_ref(k, rope.cpu(), pos, False)
            kc, vc = cache.layer(i)
            if bits == 4:
                kr, vr = (fp4_round(x.float(), dtype == H)[2].to(dtype) for x in (kr, v.double()))
                got = ops.paged_cache_read_fp4(kc, vc, step.slots, dtype)
                assert torch.equal(got[0].cpu(), kr) and torch.equal(got[1].cpu(), vr)
            else:
                flat = kc.view(-1, heads, dim)[step.slots]
                check16(flat, kr, size, dtype)
                kr, vr = flat.cpu(), v
            for j, r in enumerate(rows):
                at = slice(j * n, (j + 1) * n)
                held[r][i] = [torch.cat([held[r][i][0], kr[at]]), torch.cat([held[r][i][1], vr[at]])]
            out, lse = cache.attend(i, qr, step, return_lse=True)
            for j, r in enumerate(rows):
                at, length = slice(j * n, (j + 1) * n), len(held[r][i][0])
                ref = attention_ref(qr[at].cpu(), *held[r][i], length, n, dim ** -0.5, 0, 0.0)
                check_attention(out[at], lse[at], ref, dim, length, dtype)
        return out

    logits = (forward([0], prompt).flatten(1) @ head)[-1:]
    live, scores, width = [0], torch.zeros(1, 1), beams
    tokens = torch.full((1, steps), -1, device=DEV)
    for i in range(steps):
        scores, rows, new = _check(logits.cpu(), scores, width)
        spare = [r for r in range(2 * beams) if r not in live][:beams] if i else list(range(beams, 2 * beams))
        was = tokens.cpu()
        tokens, = ops.beam_reorder([tokens], rows.to(DEV))
        assert torch.equal(tokens.cpu(), was[rows[0].long()])
        tokens[:, i] = new[0].to(DEV)
        assert int(cache.reorder(rows.to(DEV), live, spare)) == 0
        held = {s: [list(layer) for layer in held[live[int(rows[0, j])]]] for j, s in enumerate(spare)}
        live = spare
        length = prompt + i
        assert cache.seq_lens.tolist() == [length if r in live else 0 for r in range(cache.rows)]
        tables = cache.block_tables.cpu()
        count = torch.bincount(tables[tables >= 0].long(), minlength=cache.ref_counts.numel())
        assert torch.equal(count.int(), cache.ref_counts.cpu())
        if i % 2:
            cache.compact()
        logits = forward(live, 1).flatten(1) @ head
    cache.free(live)
    assert int(cache.ref_counts.abs().sum()) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 4])
def test_the_example_in_both_kinds_of_cache(bits):
    """The search ends with its rows alone in the pool, its beams in order and all different; with one beam it
    is the greedy continuation."""
    model = example.Decoder(seed=5)
    tokens = torch.randint(0, 1003, (70,), device=DEV, generator=torch.Generator(DEV).manual_seed(3))
    cache = _cache(bits)
    found, scored = example.beam_search(model, cache, tokens, 4, 6)
    assert scored.shape == (70,) and len({tuple(t) for _, t in found}) == 4
    assert [s for s, _ in found] == sorted((s for s, _ in found), reverse=True)
    assert sorted(cache.lengths()) == [0] * 4 + [75] * 4
    cache.free(list(range(8)))
    (score, best), = example.beam_search(model, cache, tokens, 1, 6, chunk=128)[0]
    cache.free(list(range(8)))
    step = cache.extend([70] + [0] * 7)
    rope = ops.rope_table(80, 64)
    logits, total = model.forward(tokens, None, example.paged(cache, step, rope)), 0.0
    for t in best:
        top = torch.log_softmax(logits[-1].double(), 0)
        # logits of fp16 activations, whatever tiles they went through: some units of 2^-11 of 9
        assert float(top[t]) >= float(top.max()) - 0.1
        total += float(top[t])
        step = cache.extend([1] + [0] * 7)
        logits = model.forward(torch.tensor([t], device=DEV), None, example.paged(cache, step, rope))
    assert abs(total - score) < 0.2


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("page,dim,heads", [(16, 64, 2), (5, 96, 3), (1, 32, 1)])
def test_writing_and_forking(page, dim, heads, bits):
    """Without a rotation; a fork's copy of a page in part filled goes on by itself."""
    cache = _cache(bits, page_size=page, head_dim=dim, kv_heads=heads, rows=2, max_seq_len=40, pages=80)
    assert cache.pool.stride(1) * cache.pool.element_size() % 16 == 0 or bits == 16

    def read(layer, row):
        n = int(cache.seq_lens[row])
        j = torch.arange(n, device=DEV)
        slots = cache.block_tables[row, j // page].long() * page + j % page
        if bits == 4:
            return ops.paged_cache_read_fp4(*cache.layer(layer), slots, H)
        return [c.reshape(-1, heads, dim)[slots] for c in cache.layer(layer)]

    def write(counts, seed):
        step = cache.extend(counts)
        kv = [torch.randn(2, sum(counts), heads, dim, generator=gen(seed + i)).half() for i in range(2)]
        for i in range(2):
            cache.write(i, kv[i][0].to(DEV), kv[i][1].to(DEV), step)
        return [x if bits == 16 else fp4_round(x, True)[2].half() for x in kv]

    first = write([18, 0], 1)
    cache.fork([0], [1])
    second = write([3, 5], 5)
    for i in range(2):
        for plane in range(2):
            got = [read(i, r)[plane].cpu() for r in range(2)]
            assert torch.equal(got[0], torch.cat([first[i][plane], second[i][plane][:3]]))
            assert torch.equal(got[1], torch.cat([first[i][plane], second[i][plane][3:]]))


@pytest.mark.gpu
def test_reorder():
    """Rows that go on twice, once and not at all; one that names none; a full pool; and back again."""
    cache = _cache(16, layers=1, page_size=8, pages=9, rows=6, kv_heads=1, max_seq_len=64)
    cache.extend([10, 16, 3, 0, 0, 0])
    assert int((cache.ref_counts > 0).sum()) == 5

    def rows(*r):
        return torch.tensor(r, dtype=torch.int32, device=DEV)

    assert int(cache.reorder(rows(1, 0, 0), [0, 1, 2], [5, 4, 3])) == 0
    assert cache.seq_lens.tolist() == [0, 0, 0, 10, 10, 16] and int((cache.ref_counts > 0).sum()) == 5
    before = (cache.ref_counts.tolist(), cache.block_tables.tolist())
    # a row that is not there leaves its place empty; both of the others are of one parent
    assert int(cache.reorder(rows(7, 2, 2), [5, 4, 3], [0, 1, 2])) == 0
    assert cache.seq_lens.tolist() == [0, 10, 10, 0, 0, 0] and int((cache.ref_counts > 0).sum()) == 3
    assert int(cache.reorder(rows(-1, 0, 1), [1, 2], [3, 4, 5])) == 0
    assert cache.seq_lens.tolist() == [0, 0, 0, 0, 10, 10]
    cache.extend([30, 0, 0, 0, 0, 0])  # 7 of 9 pages
    before = (cache.ref_counts.tolist(), cache.block_tables.tolist(), cache.seq_lens.tolist())
    assert int(cache.reorder(rows(0, 1, 1), [4, 5], [1, 2, 3])) == 1
    assert (cache.ref_counts.tolist(), cache.block_tables.tolist(), cache.seq_lens.tolist()) == before
    step = cache.extend([0, 0, 0, 0, 1, 1])  # the rows that stayed go on, by their bounds too
    assert int(step.missing) == 0 and step.max_seq_len >= 11
    assert cache.positions(step).tolist() == [10, 10]
    cache.free([0])
    assert int(cache.reorder(rows(0, 1, 1), [4, 5], [1, 2, 3])) == 0  # rows whose bounds a refusal left
    assert cache.lengths() == [0, 11, 11, 11, 0, 0]
    cache.extend([0, 0, 0, 0, 0, 20])
    with pytest.raises(RuntimeError, match="int32"):  # refused with nothing changed
        cache.reorder(rows(2).long(), [1, 2, 3], [5])
    assert cache.lengths() == [0, 11, 11, 11, 0, 20]
    assert int(cache.reorder(rows(2), [1, 2, 3], [5])) == 0  # a spare row in use gives its pages back
    assert cache.lengths() == [0, 0, 0, 0, 0, 11] and int(cache.ref_counts.sum()) == 2


@pytest.mark.gpu
def test_positions_are_of_a_step_that_stands():
    cache = _cache(16, layers=1)
    first = cache.extend([3, 0, 2, 0, 0, 0, 0, 0])
    assert cache.positions(first).tolist() == [0, 1, 2, 0, 1] and cache.positions(first).dtype == torch.int64
    second = cache.extend([1, 1, 2, 0, 0, 0, 0, 0])
    third = cache.extend([1, 0, 0, 0, 0, 0, 0, 0])
    assert cache.positions(first).tolist() == [0, 1, 2, 0, 1]  # made before
    assert cache.positions(third).tolist() == [4]
    with pytest.raises(ValueError, match="changed"):
        cache.positions(second)
    for change in (lambda: cache.fork([0], [7]), lambda: cache.free([0]),
                   lambda: cache.reorder(torch.zeros(1, dtype=torch.int32, device=DEV), [2], [3])):
        step = cache.extend([1] + [0] * 7)
        change()
        with pytest.raises(ValueError, match="changed"):
            cache.positions(step)
    full = _cache(16, layers=1, pages=1)
    full.extend([10] + [0] * 7)
    refused = full.extend([3, 20] + [0] * 6)
    assert int(refused.missing) > 0
    assert full.positions(refused).tolist() == [10, 11, 12, *range(20)]  # as they would have been
    empty = full.extend([0] * 8)
    assert full.positions(empty).tolist() == []


def test_refusals():
    for bits, dim in ((8, 64), (4, 48), (4, 288)):
        with pytest.raises(ValueError, match="bits"):
            PagedKVCache(1, 4, 8, 1, dim, 1, 64, device="cpu", bits=bits)
    cache = PagedKVCache(1, 4, 7, 3, 96, 4, 64, device="cpu", bits=4)
    assert cache.pool.dtype == torch.uint8 and cache.pool.shape == (2, 4, 7, 3, 51)
    assert cache.pool.stride(1) == 1072 and cache.pool.stride(0) == 4 * 1072
    k = torch.zeros(0, 3, 96, dtype=H)  # a cache of bf16
    for call in (lambda: cache.write(0, k, k, None), lambda: cache.append(0, k, k, k, None, None),
                 lambda: cache.attend(0, k, None)):
        with pytest.raises(ValueError, match="cache is of torch.bfloat16, got torch.float16"):
            call()
    rows = torch.zeros(2, dtype=torch.int32)
    for live, spare in (([0, 1], [2, 2]), ([0, 1], [1, 2]), ([0, 1], [2]), ([0, 1], [1, 2, 3])):
        with pytest.raises(ValueError, match="spare row"):
            cache.reorder(rows, live, spare)
    for live, spare in (([0, 4], [2, 3]), ([0, 1], [2, -1])):
        with pytest.raises(ValueError, match="rows are 0 to 3"):
            cache.reorder(rows, live, spare)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 4])
def test_no_method_waits_for_the_device(bits):
    cache = _cache(bits)
    q, k = torch.zeros(4, 8, 64, dtype=H, device=DEV), torch.zeros(4, 2, 64, dtype=H, device=DEV)
    rope = ops.rope_table(256, 64)
    logits = torch.zeros(4, 5000, device=DEV)

    def use():
        cache.extend([9] * 4 + [0] * 4)
        scores = torch.zeros(1, 4, device=DEV)
        for live, spare in (([0, 1, 2, 3], [4, 5, 6, 7]), ([4, 5, 6, 7], [0, 1, 2, 3])):
            step = cache.extend([int(r in live) for r in range(8)])
            cache.attend(0, cache.append(0, q, k, k, step, rope), step)
            scores, rows, _ = ops.beam_select(logits, scores)
            cache.reorder(rows, live, spare)
        cache.free(list(range(8)))

    for _ in range(3):  # the allocators' first memory
        use()
    torch.cuda.synchronize()
    busy = torch.cuda.Event()
    torch.cuda._sleep(1 << 28)  # a tenth of a second or more
    busy.record()
    use()
    assert not busy.query()
    torch.cuda.synchronize()
    assert cache.lengths() == [0] * 8 and int(cache.ref_counts.abs().sum()) == 0
