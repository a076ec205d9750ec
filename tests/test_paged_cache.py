"""The paged cache's book-keeping and moves against their definitions (paged_case.Pages): every whole
number and every moved byte is equal."""

import ctypes
import random

import pytest
import torch

import pulsar_amd
from paged_case import DEV, Pages, gen, offsets
from pulsar_amd import ops


def _state(rows, pages, page, width, lens, seed, planes=3, heads=2, dim=8, dtype=torch.bfloat16):
    """A pool of random bytes and its book-keeping, on the host."""
    g = gen(seed)
    tables = torch.full((rows, width), -1, dtype=torch.int32)
    refs = torch.zeros(pages, dtype=torch.int32)
    order = torch.randperm(pages, generator=g).tolist()
    for b, n in enumerate(lens):
        for c in range(-(-n // page)):
            p = order.pop()
            tables[b, c] = p
            refs[p] = 1
    pool = torch.randn(planes, pages, page, heads, dim, generator=g).to(dtype)
    lens = torch.tensor(list(lens) + [0] * (rows - len(lens)), dtype=torch.int32)
    return pool, refs, tables, lens


def _dev(*tensors):
    return [t.to(DEV) for t in tensors]


def _same(host: Pages, refs, tables, lens=None):
    assert torch.equal(host.refs, refs.cpu())
    assert torch.equal(host.tables, tables.cpu())
    if lens is not None:
        assert torch.equal(host.lens, lens.cpu())


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


# ---- extend ------------------------------------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("page", [1, 8, 16, 24])
@pytest.mark.parametrize("lens,counts", [
    ([0], [1]), ([0], [0]), ([5, 16, 17], [1, 1, 1]), ([15, 0, 31, 3], [1, 40, 0, 200]), ([7] * 40, [1] * 40),
    ([0, 0], [3000, 1])])
def test_extend(page, lens, counts):
    width = max(-(-(l + c) // page) for l, c in zip(lens, counts)) + 2
    pages = sum(-(-(l + c) // page) for l, c in zip(lens, counts)) + 5
    _, refs, tables, n = _state(len(lens), pages, page, width, lens, sum(lens) + page)
    host = Pages(refs, tables, n, page)
    r, t, l = _dev(refs, tables, n)
    slots, missing = ops.paged_cache_extend(r, t, l, offsets(counts).to(DEV), sum(counts) + 2, page)
    want, lack = host.extend(counts)
    assert lack == 0 and missing.tolist() == [0]
    assert slots.tolist() == want + [-1, -1]  # tokens past the last row have no slot
    _same(host, r, t, l)


@pytest.mark.gpu
def test_extend_over_many_rows_and_pages():
    """More rows than a step of the prefix sum, more pages than a step of the scan, most of them taken."""
    rng = random.Random(1)
    rows, pages, page = 2500, 40000, 16
    refs = torch.ones(pages, dtype=torch.int32)
    free = rng.sample(range(pages), 3000)
    refs[free] = 0
    lens = torch.tensor([rng.randint(0, 40) for _ in range(rows)], dtype=torch.int32)
    tables = torch.full((rows, 8), -1, dtype=torch.int32)
    for b in range(rows):
        tables[b, :-(-int(lens[b]) // page)] = 7
    counts = [rng.choice((0, 1, 1, 1, 20)) for _ in range(rows)]
    host = Pages(refs, tables, lens, page)
    r, t, l = _dev(refs, tables, lens)
    slots, missing = ops.paged_cache_extend(r, t, l, offsets(counts).to(DEV), sum(counts), page)
    want, lack = host.extend(counts)
    assert missing.tolist() == [lack] == [0] and slots.tolist() == want
    _same(host, r, t, l)


@pytest.mark.gpu
def test_extend_is_all_or_nothing():
    page = 16
    _, refs, tables, lens = _state(3, 10, page, 6, [30, 16, 0], 2)
    host = Pages(refs, tables, lens, page)
    r, t, l = _dev(refs, tables, lens)
    for counts in ([2, 16 * 4, 16 * 3 + 1], [200, 1, 0], [3, 16 * 9, 16 * 9]):  # pages, columns, both
        slots, missing = ops.paged_cache_extend(r, t, l, offsets(counts).to(DEV), sum(counts), page)
        want, lack = host.extend(counts)
        assert lack > 0 and missing.tolist() == [lack] and slots.tolist() == want
        _same(host, r, t, l)
    slots, missing = ops.paged_cache_extend(r, t, l, offsets([2, 16 * 4, 16 * 2]).to(DEV), 98, page)  # the last free page
    assert missing.tolist() == [0]
    assert slots.tolist() == host.extend([2, 16 * 4, 16 * 2])[0]
    _same(host, r, t, l)


@pytest.mark.gpu
def test_extend_on_views():
    """ref_counts at an address that 16-byte loads cannot use, tables whose rows are apart."""
    page = 8
    _, refs, tables, lens = _state(4, 70, page, 9, [3, 60, 0, 8], 2)
    host = Pages(refs, tables, lens, page)
    flat = torch.zeros(71, dtype=torch.int32, device=DEV)
    flat[1:] = refs.to(DEV)
    wide = torch.full((4, 12), 99, dtype=torch.int32, device=DEV)
    wide[:, :9] = tables.to(DEV)
    l = lens.to(DEV)
    counts = [1, 12, 33, 8]
    slots, missing = ops.paged_cache_extend(flat[1:], wide[:, :9], l, offsets(counts).to(DEV), sum(counts), page)
    assert slots.tolist() == host.extend(counts)[0]
    _same(host, flat[1:], wide[:, :9], l)
    assert bool((wide[:, 9:] == 99).all()) and int(flat[0]) == 0


# ---- write --------------------------------------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,dim,page", [(8, 128, 16), (1, 8, 1), (3, 80, 24), (2, 5, 7), (5, 256, 64)])
@pytest.mark.parametrize("t", [0, 1, 67])
def test_write(heads, dim, page, t, dtype):
    g = gen(t + dim)
    pages = 100 // page + 4
    pool = torch.randn(2, pages, page, heads, dim, generator=g).to(dtype)
    slots = torch.randperm(pages * page, generator=g)[:t]
    if t > 3:
        slots[1], slots[2] = -1, pages * page  # no place of this cache
    fused = torch.randn(t, 2 * heads * dim + 8, generator=g).to(dtype)
    dev, f, s = _dev(pool, fused, slots)
    k, v = (x.view(t, heads, dim) for x in (f[:, :heads * dim], f[:, heads * dim:2 * heads * dim]))
    ops.paged_cache_write(k, v, dev[0], dev[1], s)
    for i in range(t):
        at = int(slots[i])
        if 0 <= at < pages * page:
            pool[0, at // page, at % page] = k[i].cpu()
            pool[1, at // page, at % page] = v[i].cpu()
    assert torch.equal(dev.cpu(), pool)


@pytest.mark.gpu
def test_write_into_other_layouts():
    """Pages that keep a head's tokens together, and keys that lie head by head."""
    g = gen(3)
    pool = torch.randn(2, 6, 4, 16, 64, generator=g).half().to(DEV)
    hnd = pool.transpose(2, 3)  # [2, pages, page 16, heads 4, dim]
    want = hnd.clone()
    k, v = (torch.randn(4, 9, 64, generator=g).half().to(DEV).transpose(0, 1) for _ in range(2))
    slots = torch.randperm(96, generator=g)[:9].to(DEV)
    ops.paged_cache_write(k, v, hnd[0], hnd[1], slots)
    for c, x in zip(want, (k, v)):
        c[slots // 16, slots % 16] = x
    assert torch.equal(hnd, want)


# ---- copy ----------------------------------------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("planes,page,heads,dim,dtype", [
    (1, 16, 8, 128, torch.bfloat16), (6, 64, 8, 128, torch.float16), (4, 3, 1, 5, torch.float16),
    (2, 2, 3, 7, torch.uint8), (3, 16, 2, 66, torch.bfloat16), (2, 1, 1, 1, torch.float32)])
def test_copy(planes, page, heads, dim, dtype):
    g = gen(page)
    pool = torch.randint(0, 100, (planes, 40, page, heads, dim), generator=g).to(dtype)
    perm = torch.randperm(40, generator=g).int()
    src, dst = perm[:12].clone(), perm[12:24].clone()
    src[5] = src[4]
    src[6], dst[7] = -1, 40  # no pages of this pool
    dev, s, d = _dev(pool, src, dst)
    ops.paged_cache_copy(dev, s, d)
    for a, b in zip(src.tolist(), dst.tolist()):
        if a >= 0 and b < 40:
            pool[:, b] = pool[:, a]
    assert torch.equal(dev.cpu(), pool)
    ops.paged_cache_copy(dev, s[:0], d[:0])
    assert torch.equal(dev.cpu(), pool)


@pytest.mark.gpu
def test_copy_in_a_slice_of_a_pool():
    """Planes and pages that are apart."""
    whole = torch.randn(4, 10, 16, 2, 64, generator=gen(1)).half().to(DEV)
    want = whole.clone()
    ops.paged_cache_copy(whole[1:3, 2:9], _i32([0, 3]), _i32([6, 1]))
    want[1:3, 8], want[1:3, 3] = want[1:3, 2].clone(), want[1:3, 5].clone()
    assert torch.equal(whole, want)


@pytest.mark.gpu
def test_copy_past_32_bits():
    page_bytes = 1 << 20
    pages = (1 << 32) // page_bytes + 3
    pool = torch.zeros(1, pages, 16, page_bytes // 16, dtype=torch.uint8, device=DEV)
    pool[0, pages - 1] = 5
    pool[0, 0] = 9
    ops.paged_cache_copy(pool, _i32([pages - 1, 0]), _i32([1, pages - 2]))
    assert bool((pool[0, 1] == 5).all()) and bool((pool[0, pages - 2] == 9).all())


# ---- fork and free -----------------------------------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("page", [8, 16, 24])
@pytest.mark.parametrize("lens,src,dst", [
    ([5], [0], [1]), ([16], [0], [1]), ([0], [0], [1]), ([100, 33, 7], [2, 2, 0], [3, 4, 5]),
    ([250, 1, 24, 48], [0, 1, 2, 3, 0], [8, 7, 6, 5, 4])])
def test_fork_then_free(page, lens, src, dst):
    rows = max(dst) + 1
    pool, refs, tables, n = _state(rows, 90, page, 40, lens, page + len(lens))
    host = Pages(refs, tables, n, page)
    dev, r, t, l = _dev(pool, refs, tables, n)
    missing = ops.paged_cache_fork(dev, r, t, l, _i32(src), _i32(dst))
    assert host.fork(src, dst, pool) == 0 and missing.tolist() == [0]
    _same(host, r, t, l)
    assert torch.equal(dev.cpu(), pool)
    ops.paged_cache_free(r, t, l, _i32(src + [src[0], -1, rows]))  # named again, and no rows at all
    host.free(src)
    _same(host, r, t, l)
    ops.paged_cache_free(r, t, l, _i32(list(range(rows))))
    host.free(list(range(rows)))
    _same(host, r, t, l)
    assert int(r.abs().sum()) == 0


@pytest.mark.gpu
def test_fork_is_all_or_nothing():
    page = 16
    pool, refs, tables, n = _state(6, 6, page, 4, [20, 30], 3)  # four pages used, two free
    host = Pages(refs, tables, n, page)
    dev, r, t, l = _dev(pool, refs, tables, n)
    missing = ops.paged_cache_fork(dev, r, t, l, _i32([0, 1, 0]), _i32([2, 3, 4]))
    assert missing.tolist() == [host.fork([0, 1, 0], [2, 3, 4], pool)] == [1]
    _same(host, r, t, l)
    assert torch.equal(dev.cpu(), pool)


@pytest.mark.gpu
def test_fork_passes_over_rows_that_are_none():
    page = 16
    pool, refs, tables, n = _state(5, 12, page, 4, [20, 30], 3)
    host = Pages(refs, tables, n, page)
    dev, r, t, l = _dev(pool, refs, tables, n)
    ops.paged_cache_fork(dev, r, t, l, _i32([-1, 1, 9, 0]), _i32([2, 3, 4, -7]))
    host.fork([1], [3], pool)
    _same(host, r, t, l)
    assert torch.equal(dev.cpu(), pool)


@pytest.mark.gpu
def test_many_forks():
    rng = random.Random(4)
    page, rows = 8, 1400
    lens = [rng.randint(0, 30) for _ in range(200)]
    pool, refs, tables, n = _state(rows, 2500, page, 5, lens, 1, planes=1, heads=1)
    host = Pages(refs, tables, n, page)
    dev, r, t, l = _dev(pool, refs, tables, n)
    src, dst = [rng.randrange(200) for _ in range(1200)], list(range(200, 1400))
    assert ops.paged_cache_fork(dev, r, t, l, _i32(src), _i32(dst)).tolist() == [host.fork(src, dst, pool)] == [0]
    _same(host, r, t, l)
    assert torch.equal(dev.cpu(), pool)


@pytest.mark.gpu
def test_free_of_wide_tables():
    _, refs, tables, n = _state(3, 1500, 1, 700, [600, 3, 520], 5)
    host = Pages(refs, tables, n, 1)
    r, t, l = _dev(refs, tables, n)
    ops.paged_cache_free(r, t, l, _i32([2, 0]))
    host.free([2, 0])
    _same(host, r, t, l)


# ---- compact -------------------------------------------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("pages", [1, 2, 15, 16, 17, 333, 20000])
@pytest.mark.parametrize("share", [0.0, 0.3, 0.9, 1.0])
def test_compact(pages, share):
    rng = random.Random(pages + int(10 * share))
    page, rows = 4, 5
    used = rng.sample(range(pages), int(round(pages * share)))
    width = max(1, -(-len(used) // rows)) + 1
    refs, tables = torch.zeros(pages, dtype=torch.int32), torch.full((rows, width), -1, dtype=torch.int32)
    for i, p in enumerate(used):
        tables[i % rows, i // rows] = p
        refs[p] += 1
        if rng.random() < 0.1:  # held twice
            tables[(i + 1) % rows, width - 1] = p
            refs[p] += 1
    for b in range(rows):  # a count for each entry that was written over
        pass
    refs = torch.zeros(pages, dtype=torch.int32).index_add_(0, tables[tables >= 0].long(), torch.ones(
        int((tables >= 0).sum()), dtype=torch.int32))
    pool = torch.randn(2, pages, page, 1, 8, generator=gen(pages)).half()
    host = Pages(refs, tables, torch.zeros(rows, dtype=torch.int32), page)
    dev, r, t = _dev(pool, refs, tables)
    n = ops.paged_cache_compact(dev, r, t)
    assert n.tolist() == [host.compact(pool)]
    _same(host, r, t)
    assert torch.equal(dev.cpu(), pool)
    assert bool((r[:int(n)] > 0).all()) and int(r[int(n):].sum()) == 0
    again = ops.paged_cache_compact(dev, r, t)  # nothing left to move
    assert torch.equal(again, n) and torch.equal(dev.cpu(), pool)
    _same(host, r, t)


@pytest.mark.gpu
def test_a_table_entry_that_no_count_covers_keeps_its_name():
    refs = torch.tensor([0, 1, 0, 1, 0], dtype=torch.int32)
    tables = torch.tensor([[1, 3, 4, 99, -5]], dtype=torch.int32)
    pool = torch.arange(5.0).view(1, 5, 1, 1).to(DEV)
    r, t = _dev(refs, tables)
    assert ops.paged_cache_compact(pool, r, t).tolist() == [2]
    assert t.tolist() == [[1, 0, 4, 99, -5]] and r.tolist() == [1, 1, 0, 0, 0]
    assert pool.flatten().tolist() == [3.0, 1.0, 2.0, 3.0, 4.0]


# ---- together ------------------------------------------------------------------------------------------


@pytest.mark.gpu
def test_a_long_life():
    """Random steps of every operation against the host's book-keeping."""
    rng = random.Random(9)
    page, rows, pages = 8, 12, 60
    pool, refs, tables, n = _state(rows, pages, page, 20, [], 1)
    host = Pages(refs, tables, n, page)
    dev, r, t, l = _dev(pool, refs, tables, n)
    for step in range(60):
        what = rng.choice(("extend", "extend", "extend", "fork", "free", "compact"))
        if what == "extend":
            counts = [rng.choice((0, 0, 1, 3, 17)) for _ in range(rows)]
            slots, missing = ops.paged_cache_extend(r, t, l, offsets(counts).to(DEV), sum(counts), page)
            want, lack = host.extend(counts)
            assert slots.tolist() == want and missing.tolist() == [lack]
        elif what == "fork":
            empty = [i for i in range(rows) if host.lens[i] == 0]
            full = [i for i in range(rows) if host.lens[i] > 0]
            if not empty or not full:
                continue
            dst = rng.sample(empty, rng.randint(1, len(empty)))
            src = [rng.choice(full) for _ in dst]
            assert ops.paged_cache_fork(dev, r, t, l, _i32(src), _i32(dst)).tolist() == [host.fork(src, dst, pool)]
        elif what == "free":
            gone = rng.sample(range(rows), 4)
            ops.paged_cache_free(r, t, l, _i32(gone))
            host.free(gone)
        else:
            assert ops.paged_cache_compact(dev, r, t).tolist() == [host.compact(pool)]
        _same(host, r, t, l)
    assert torch.equal(dev.cpu(), pool)


@pytest.mark.gpu
def test_graph_replays():
    """A decode step's extend and write as a graph, replayed between eager work."""
    page, rows = 8, 3
    pool, refs, tables, n = _state(rows, 40, page, 10, [7, 8, 0], 1, planes=2)
    host = Pages(refs, tables, n, page)
    dev, r, t, l = _dev(pool, refs, tables, n)
    cu = offsets([1] * rows).to(DEV)
    k, v = (torch.zeros(rows, 2, 8, dtype=torch.bfloat16, device=DEV) for _ in range(2))

    def step():
        slots, missing = ops.paged_cache_extend(r, t, l, cu, rows, page)
        ops.paged_cache_write(k, v, dev[0], dev[1], slots)
        return slots, missing

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        slots, missing = step()
    for i in range(12):
        k.fill_(i + 1)
        v.fill_(-i - 1)
        if i % 3 == 2:
            s, m = step()
        else:
            graph.replay()
            s, m = slots, missing
        want, lack = host.extend([1] * rows)
        torch.cuda.synchronize()
        assert s.tolist() == want and m.tolist() == [lack] == [0]
        for at in want:
            pool[0, at // page, at % page] = i + 1
            pool[1, at // page, at % page] = -i - 1
        _same(host, r, t, l)
        assert torch.equal(dev.cpu(), pool)


# ---- refusals -------------------------------------------------------------------------------------------


@pytest.mark.gpu
def test_refusals():
    pool, refs, tables, lens = _state(2, 8, 16, 3, [5, 20], 1, planes=2)
    p, r, t, l = _dev(pool, refs, tables, lens)
    cu = offsets([1, 1]).to(DEV)
    k = torch.zeros(2, 2, 8, dtype=torch.bfloat16, device=DEV)
    s = torch.zeros(2, dtype=torch.int64, device=DEV)
    bad = [
        (lambda: ops.paged_cache_extend(r.long(), t, l, cu, 2, 16), "int32"),
        (lambda: ops.paged_cache_extend(r, t, l[:1], cu, 2, 16), "seq_lens"),
        (lambda: ops.paged_cache_extend(r, t, l, cu[:2], 2, 16), "cu_q"),
        (lambda: ops.paged_cache_extend(r, t, l, cu, 2, 0), "page_size"),
        (lambda: ops.paged_cache_extend(r, t, l, cu, -1, 16), "num_tokens"),
        (lambda: ops.paged_cache_extend(r, t.t(), l, cu, 2, 16), "contiguous|rows"),
        (lambda: ops.paged_cache_extend(r, t[:1].expand(2, 3), l, cu, 2, 16), "overlap"),
        (lambda: ops.paged_cache_write(k, k, p[0], p[1], s.int()), "int64"),
        (lambda: ops.paged_cache_write(k, k, p[0], p[1], s[:1]), "slots"),
        (lambda: ops.paged_cache_write(k.half(), k.half(), p[0], p[1], s), "one dtype"),
        (lambda: ops.paged_cache_write(k[..., :4], k[..., :4], p[0], p[1], s), "head_dim"),
        (lambda: ops.paged_cache_write(k, k[:1], p[0], p[1], s), "3-D"),
        (lambda: ops.paged_cache_write(k, k, p[0], p[1][:4], s), "one shape"),
        (lambda: ops.paged_cache_copy(p.transpose(2, 3), _i32([0]), _i32([1])), "contiguous"),
        (lambda: ops.paged_cache_copy(p, _i32([0, 1]), _i32([1])), "length"),
        (lambda: ops.paged_cache_copy(p, _i32([0]).long(), _i32([1])), "int32"),
        (lambda: ops.paged_cache_fork(p, r[:4], t, l, _i32([0]), _i32([1])), "ref_counts"),
        (lambda: ops.paged_cache_fork(p, r, t, l, _i32([0]), _i32([1, 0])), "length"),
        (lambda: ops.paged_cache_free(r, t, l, torch.tensor([0], dtype=torch.int32)), "one CUDA device"),
        (lambda: ops.paged_cache_compact(p, r[:3], t), "ref_counts"),
    ]
    for call, message in bad:
        with pytest.raises(RuntimeError, match=message):
            call()
    many = torch.full((4097, 1), -1, dtype=torch.int32, device=DEV)
    with pytest.raises(RuntimeError, match="size"):
        ops.paged_cache_extend(r, many, torch.zeros(4097, dtype=torch.int32, device=DEV),
                               torch.zeros(4098, dtype=torch.int32, device=DEV), 0, 16)
    assert torch.equal(r.cpu(), refs) and torch.equal(t.cpu(), tables) and torch.equal(l.cpu(), lens)


def test_c_entries_refuse_before_any_launch():
    lib = pulsar_amd.capi()
    P, I, SZ = ctypes.c_void_p, ctypes.c_int64, ctypes.c_size_t

    class Pool(ctypes.Structure):
        _fields_ = [("base", P)] + [(n, I) for n in ("planes", "num_pages", "page_bytes", "plane_stride_bytes",
                                                     "page_stride_bytes")]

    x = P(4096)  # never dereferenced
    lib.pw4_paged_cache_extend.argtypes = [P, I, P, I, I, P, P, I, I, I, P, P, P]
    ext = lib.pw4_paged_cache_extend
    assert ext(x, 4, x, 2, 2, x, x, 1, 1, 16, x, None, None) == -1
    assert ext(x, 4, x, 2, 1, x, x, 1, 1, 16, x, x, None) == -2
    assert ext(x, 4, x, 2, 2, x, x, 4097, 1, 16, x, x, None) == -2
    assert ext(x, 4, x, 2, 2, x, x, 1, 1, 0, x, x, None) == -2
    assert ext(None, 4, x, 2, 2, x, x, 1, 1, 16, x, x, None) == -1
    lib.pw4_paged_cache_write.argtypes = [P] * 5 + [I] * 12 + [P]
    w = lib.pw4_paged_cache_write
    assert w(x, x, x, x, None, 1, 2, 8, 16, 8, 16, 8, 4, 16, 256, 16, 8, None) == -1
    assert w(x, x, x, x, x, 1, 2, 8, 16, 8, 16, 8, 4, 0, 256, 16, 8, None) == -1
    assert w(x, x, x, x, x, 1, 2, 8, 16, 8, 16, 8, 2 ** 28, 16, 256, 16, 8, None) == -2
    assert w(P(4097), x, x, x, x, 1, 2, 8, 16, 8, 16, 8, 4, 16, 256, 16, 8, None) == -1
    assert w(None, None, None, None, None, 0, 2, 8, 16, 8, 16, 8, 4, 16, 256, 16, 8, None) == 0
    lib.pw4_paged_cache_copy.argtypes = [ctypes.POINTER(Pool), P, P, I, P]
    good = Pool(4096, 2, 4, 512, 2048, 512)
    assert lib.pw4_paged_cache_copy(None, x, x, 1, None) == -1
    assert lib.pw4_paged_cache_copy(ctypes.byref(good), None, x, 1, None) == -1
    assert lib.pw4_paged_cache_copy(ctypes.byref(Pool(None, 2, 4, 512, 2048, 512)), x, x, 1, None) == -1
    assert lib.pw4_paged_cache_copy(ctypes.byref(good), x, x, 0, None) == 0
    lib.pw4_paged_cache_fork.argtypes = [ctypes.POINTER(Pool), P, P, I, I, I, P, P, P, I, I, P, P, SZ, P]
    lib.pw4_paged_cache_fork_workspace_size.argtypes, lib.pw4_paged_cache_fork_workspace_size.restype = [I], SZ
    need = lib.pw4_paged_cache_fork_workspace_size(3)
    assert need >= 24
    fork = lib.pw4_paged_cache_fork
    assert fork(ctypes.byref(good), x, x, 2, 2, 2, x, x, x, 3, 16, x, x, need - 1, None) == -3
    assert fork(ctypes.byref(good), x, x, 2, 2, 2, x, x, x, 4097, 16, x, x, 1 << 20, None) == -2
    assert fork(ctypes.byref(good), x, x, 2, 2, 2, x, None, x, 3, 16, x, x, need, None) == -1
    lib.pw4_paged_cache_free.argtypes = [P, I, P, I, I, I, P, P, I, P]
    assert lib.pw4_paged_cache_free(x, 4, x, 2, 2, 2, None, x, 1, None) == -1
    assert lib.pw4_paged_cache_free(x, 4, x, 2, 2, 2, x, None, 0, None) == 0
    lib.pw4_paged_cache_compact.argtypes = [ctypes.POINTER(Pool), P, P, I, I, I, P, P, SZ, P]
    lib.pw4_paged_cache_compact_workspace_size.argtypes, lib.pw4_paged_cache_compact_workspace_size.restype = [I], SZ
    assert lib.pw4_paged_cache_compact(ctypes.byref(good), x, x, 2, 2, 2, x, x, 4, None) == -3
    assert lib.pw4_paged_cache_compact(ctypes.byref(good), x, x, 2, 2, 2, None, x, 4096, None) == -1


def test_fake_kernels():
    def meta(shape, dtype=torch.int32):
        return torch.empty(shape, dtype=dtype, device="meta")

    pool, r, t, l = meta((2, 8, 16, 2, 8), torch.half), meta((8,)), meta((3, 4)), meta((3,))
    slots, missing = ops.paged_cache_extend(r, t, l, meta((4,)), 9, 16)
    assert slots.shape == (9,) and slots.dtype == torch.int64 and missing.shape == (1,)
    assert ops.paged_cache_write(meta((9, 2, 8), torch.half), meta((9, 2, 8), torch.half), pool[0], pool[1], slots) is None
    assert ops.paged_cache_copy(pool, l, l) is None
    assert ops.paged_cache_fork(pool, r, t, l, l, l).shape == (1,)
    assert ops.paged_cache_free(r, t, l, l) is None
    assert ops.paged_cache_compact(pool, r, t).shape == (1,)


@pytest.mark.gpu
def test_opcheck():
    pool, refs, tables, lens = _state(4, 8, 16, 3, [5, 20], 1, planes=2)
    p, r, t, l = _dev(pool, refs, tables, lens)
    k = torch.zeros(2, 2, 8, dtype=torch.bfloat16, device=DEV)
    s = torch.arange(2, device=DEV)
    lib = torch.ops.pulsar
    for op, args in ((lib.paged_cache_extend, (r, t, l, offsets([1, 1, 0, 0]).to(DEV), 2, 16)),
                     (lib.paged_cache_write, (k, k, p[0], p[1], s)),
                     (lib.paged_cache_copy, (p, _i32([0]), _i32([1]))),
                     (lib.paged_cache_fork, (p, r, t, l, _i32([0]), _i32([2]))),
                     (lib.paged_cache_free, (r, t, l, _i32([0]))),
                     (lib.paged_cache_compact, (p, r, t))):
        torch.library.opcheck(op.default, args, test_utils=("test_schema", "test_faketensor"))


def _compact_size(pages):
    lib = pulsar_amd.capi()
    lib.pw4_paged_cache_compact_workspace_size.argtypes = [ctypes.c_int64]
    lib.pw4_paged_cache_compact_workspace_size.restype = ctypes.c_size_t
    return lib.pw4_paged_cache_compact_workspace_size(pages)


def test_compact_workspace_holds_what_is_written():
    """A count (and a place to align), both ends of each of up to pages / 2 moves, a name for each page."""
    for pages in (1, 2, 3, 63, 64, 575, 4095, 4096):
        assert _compact_size(pages) >= 4 * (2 + 2 * ((pages + 1) // 2) + pages)


@pytest.mark.gpu
@pytest.mark.parametrize("pages", [1, 2, 63, 64, 127, 575])
def test_compact_writes_nothing_past_its_workspace(pages):
    page, used = 8, max(1, pages // 3)
    rng = random.Random(pages)
    held = rng.sample(range(pages), used)
    tables = torch.tensor([held], dtype=torch.int32)
    refs = torch.zeros(pages, dtype=torch.int32)
    refs[held] = 1
    pool = torch.randn(2, pages, page, 1, 8, generator=gen(pages)).bfloat16()
    host, want = Pages(refs, tables, torch.tensor([used * page], dtype=torch.int32), page), pool.clone()
    p, r, t = _dev(pool, refs, tables)
    size = _compact_size(pages)
    ws = torch.full((size + 64,), 0x5a, dtype=torch.uint8, device=DEV)

    class Pool(ctypes.Structure):
        _fields_ = [("base", ctypes.c_void_p)] + [(n, ctypes.c_int64) for n in (
            "planes", "num_pages", "page_bytes", "plane_stride_bytes", "page_stride_bytes")]

    lib = pulsar_amd.capi()
    P, I = ctypes.c_void_p, ctypes.c_int64
    lib.pw4_paged_cache_compact.argtypes = [ctypes.POINTER(Pool), P, P, I, I, I, P, P, ctypes.c_size_t, P]
    count = torch.zeros(1, dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    args = Pool(p.data_ptr(), 2, pages, page * 16, pages * page * 16, page * 16)
    assert lib.pw4_paged_cache_compact(ctypes.byref(args), r.data_ptr(), t.data_ptr(), 1, used, used, count.data_ptr(),
                                       ws.data_ptr(), size, None) == 0
    torch.cuda.synchronize()
    assert count.tolist() == [host.compact(want)]
    _same(host, r, t)
    assert torch.equal(p.cpu(), want) and bool((ws[size:] == 0x5a).all())


@pytest.mark.gpu
@pytest.mark.parametrize("page", [1, 16])
@pytest.mark.parametrize("lens,counts", [([5, 40], [2 ** 31 - 50, 0]), ([2 ** 31 - 20, 0], [30, 0]),
                                         ([2 ** 31 - 1, 3], [2 ** 31 - 1, 0]), ([7, 9], [0, 2 ** 31 - 1])])
def test_extend_by_more_than_any_table_holds(lens, counts, page):
    """Tokens whose sum passes 31 or 32 bits: refused as any others that no table has room for, and
    neither the tables nor what lies around them changes."""
    wide = torch.full((4, 12), 99, dtype=torch.int32, device=DEV)
    tables = wide[1:3, :8]
    tables.fill_(-1)
    refs = torch.zeros(64, dtype=torch.int32, device=DEV)
    l = torch.tensor(lens, dtype=torch.int32, device=DEV)
    slots, missing = ops.paged_cache_extend(refs, tables, l, offsets(counts).to(DEV), 40, page)
    assert int(missing) > 0 and set(slots.tolist()) == {-1}
    assert l.tolist() == lens and int(refs.abs().sum()) == 0 and bool((tables == -1).all())
    wide[1:3, :8] = 99
    assert bool((wide == 99).all())


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 3, 37])
def test_fork_writes_nothing_past_its_workspace(n):
    page, width = 8, 4
    pool, refs, tables, lens = _state(2 * n, 6 * n, page, width, [3 + 5 * (b % 4) for b in range(n)], n)
    host, want = Pages(refs, tables, lens, page), pool.clone()
    p, r, t, l = _dev(pool, refs, tables, lens)

    class Pool(ctypes.Structure):
        _fields_ = [("base", ctypes.c_void_p)] + [(k, ctypes.c_int64) for k in (
            "planes", "num_pages", "page_bytes", "plane_stride_bytes", "page_stride_bytes")]

    lib = pulsar_amd.capi()
    P, I, SZ = ctypes.c_void_p, ctypes.c_int64, ctypes.c_size_t
    lib.pw4_paged_cache_fork_workspace_size.argtypes, lib.pw4_paged_cache_fork_workspace_size.restype = [I], SZ
    lib.pw4_paged_cache_fork.argtypes = [ctypes.POINTER(Pool), P, P, I, I, I, P, P, P, I, I, P, P, SZ, P]
    size = lib.pw4_paged_cache_fork_workspace_size(n)
    ws = torch.full((size + 64,), 0x5a, dtype=torch.uint8, device=DEV)
    src, dst = _i32(list(range(n))), _i32(list(range(n, 2 * n)))
    missing = torch.full((16,), 77, dtype=torch.int32, device=DEV)
    page_bytes = pool[0, 0].numel() * 2
    args = Pool(p.data_ptr(), pool.shape[0], pool.shape[1], page_bytes, pool.shape[1] * page_bytes, page_bytes)
    torch.cuda.synchronize()
    assert lib.pw4_paged_cache_fork(ctypes.byref(args), r.data_ptr(), t.data_ptr(), 2 * n, width, width, l.data_ptr(),
                                    src.data_ptr(), dst.data_ptr(), n, page, missing.data_ptr(), ws.data_ptr(), size,
                                    None) == 0
    torch.cuda.synchronize()
    assert host.fork(list(range(n)), list(range(n, 2 * n)), want) == 0
    _same(host, r, t, l)
    assert torch.equal(p.cpu(), want) and bool((ws[size:] == 0x5a).all()) and missing.tolist() == [0] + [77] * 15
