"""paged_attention_fp4 against attention in 64 bits over the values that its cache holds: the bounds are
paged_case.check_attention's, since a 4-bit value is exact in 16 bits."""

import ctypes
import math

import pytest
import torch

import pulsar_amd
from fp4_case import fp4_kv, fp4_round, row_bytes
from paged_case import DEV, attention_ref, check_attention, gen, offsets
from pulsar_amd import ops

H, B = torch.float16, torch.bfloat16


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _run(lens, new, *, heads=2, group=4, dim=128, page=16, dtype=B, window=0, cap=0.0, scale=None, seed=0, q=None,
         extra=0, lse=True, pad=0):
    """Runs one call and checks every sequence; returns (out, lse)."""
    kc, vc, tables, ks, vs = fp4_kv(lens, page, heads, dim, dtype, seed, pad=pad)
    t = sum(new) + extra
    if q is None:
        q = torch.randn(t, heads * group, dim, generator=gen(seed + 1)).to(dtype).to(DEV)
    cu = offsets(new)
    got = ops.paged_attention_fp4(q, kc, vc, tables, _i32(lens), cu.to(DEV), max(new + [0]), max(lens + [0]), scale=scale,
                                  window=window, softcap=cap, return_lse=lse)
    out, l = got if lse else (got, None)
    assert out.shape == q.shape and out.dtype == dtype and out.is_contiguous()
    s = 1 / math.sqrt(dim) if scale is None else scale
    for b, n in enumerate(new):
        if n == 0:
            continue
        at = slice(int(cu[b]), int(cu[b]) + n)
        ref = attention_ref(q[at].cpu(), ks[b], vs[b], lens[b], n, s, window, cap)
        check_attention(out[at], None if l is None else l[at], ref, dim, lens[b], dtype)
    if extra:  # rows past the last sequence
        assert bool((out[sum(new):] == 0).all()) and bool((l[sum(new):] == -math.inf).all())
    return out, l


@pytest.fixture
def plan(monkeypatch):
    """Pins the split, the units of a piece and the tile rows (the library reads these in tests)."""
    def pin(split=None, units=None, tile=None):
        for name, value in (("SPLIT", split), ("UNITS", units), ("TILE", tile)):
            if value is None:
                monkeypatch.delenv(f"PW4_ATTN_{name}", raising=False)
            else:
                monkeypatch.setenv(f"PW4_ATTN_{name}", str(value))
    return pin


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [H, B])
@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 500, 1025])
def test_one_token(length, dtype):
    _run([length], [1], dtype=dtype, seed=length)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [H, B])
@pytest.mark.parametrize("heads,group", [(1, 1), (8, 1), (2, 2), (3, 5), (2, 7), (4, 8), (1, 16), (1, 17), (2, 32),
                                         (1, 40), (1, 71)])
def test_head_groups(heads, group, dtype):
    """One token, a few and a chunk in one batch, for each layout of query over key-value heads."""
    _run([300, 77, 130], [1, 5, 70], heads=heads, group=group, dim=64, dtype=dtype, seed=group)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [H, B])
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("new", [1, 10, 130])
def test_head_dims(dim, new, dtype):
    _run([333, 140], [new, new], heads=2, group=2, dim=dim, dtype=dtype, seed=dim)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [1, 7, 8, 16, 24, 32, 60, 64, 128, 256, 1000])
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("dim", [64, 96])
def test_page_sizes(page, new, dim):
    """Pages that end inside a block of keys, pages of many blocks, and pages further apart than they are long."""
    _run([421, 64, 40], [new, new, new], page=page, dim=dim, seed=page, pad=page % 3)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [H, B])
@pytest.mark.parametrize("lens,new", [
    ([0], [0]), ([5], [0]), ([0, 9, 0, 200], [0, 9, 0, 3]),       # nothing cached, nothing asked
    ([64], [64]), ([65], [65]), ([128], [128]), ([257], [257]), ([1000], [1000]),  # whole prompts
    ([700, 33, 1, 512, 129], [129, 33, 1, 1, 128]),               # prompts, chunks and tokens in one batch
    ([2000, 2000], [31, 33]), ([1500], [16]), ([1500], [17]),     # rows around a tile's
])
def test_lengths(lens, new, dtype):
    _run(lens, new, dtype=dtype, seed=sum(lens))


@pytest.mark.gpu
@pytest.mark.parametrize("window", [1, 2, 16, 63, 64, 65, 100, 5000])
@pytest.mark.parametrize("new", [1, 90])
def test_windows(window, new):
    _run([700, 90, 311], [new, new, new], window=window, seed=window)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [H, B])
@pytest.mark.parametrize("new", [1, 100])
def test_softcap_and_scale(new, dtype):
    _run([400, 123], [new, new], cap=2.0, dtype=dtype, seed=1)       # saturates
    _run([400, 123], [new, new], cap=50.0, scale=1.0, dtype=dtype, seed=2)
    _run([400, 123], [new, new], scale=0.0, dtype=dtype, seed=3)     # the mean
    _run([400, 123], [new, new], scale=-0.1, dtype=dtype, seed=4)
    _run([200, 123], [new, new], scale=3.0, dtype=dtype, seed=5)     # one key takes all
    _run([400, 123], [new, new], cap=5.0, window=70, dtype=dtype, seed=6)


@pytest.mark.gpu
def test_long_context_is_split():
    _run([9000, 300, 4097], [1, 1, 1], heads=2, group=4, seed=1)
    _run([6000, 5], [3, 3], heads=1, group=4, dtype=H, seed=2)
    _run([5000, 70], [60, 60], heads=1, group=2, seed=3)


@pytest.mark.gpu
@pytest.mark.parametrize("dim,length", [(64, 30000), (128, 26000), (256, 14000)])
@pytest.mark.parametrize("new,dtype", [(1, B), (5, H)])
def test_sequences_in_many_pieces(dim, length, new, dtype):
    """Pieces by the hundred to join, and a short sequence beside them."""
    out, lse = _run([length, 7], [new, new], heads=1, group=4, dim=dim, dtype=dtype, seed=dim)
    again = _run([length, 7], [new, new], heads=1, group=4, dim=dim, dtype=dtype, seed=dim)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])


@pytest.mark.gpu
@pytest.mark.parametrize("split,units", [(0, None), (1, 1), (1, 3)])
@pytest.mark.parametrize("new", [1, 6])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_few_rows_whole_and_split(plan, dim, new, split, units):
    plan(split, units)
    _run([1500, 40, 0, 777, 3], [new, new, 0, new, min(new, 3)], heads=2, group=4, dim=dim, seed=dim + new)
    _run([900, 1300], [new, new], heads=1, group=3, dim=dim, window=200, cap=3.0, dtype=H, seed=dim)
    _run([700] * 70, [new] * 70, heads=1, group=2, dim=dim, page=24, seed=dim)  # more sequences than lanes


@pytest.mark.gpu
@pytest.mark.parametrize("split,units", [(0, None), (1, 1), (1, 3)])
@pytest.mark.parametrize("tile", [32, 128, 256])
@pytest.mark.parametrize("dim,dtype", [(64, H), (128, B), (96, B), (256, H)])
def test_many_rows_whole_and_split(plan, dim, dtype, tile, split, units):
    plan(split, units, tile)
    _run([600, 257, 64, 400], [600, 129, 1, 90], heads=2, group=2, dim=dim, dtype=dtype, seed=dim)
    _run([900, 333], [200, 333], heads=1, group=3, dim=dim, dtype=dtype, window=150, cap=4.0, page=8, seed=dim)
    _run([1000, 50], [70, 50], heads=1, group=7, dim=dim, dtype=dtype, page=24, window=300, seed=dim)
    _run([500], [499], heads=3, group=1, dim=dim, dtype=dtype, page=7, extra=5, seed=dim)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [H, B])
@pytest.mark.parametrize("dim", [64, 96, 128])
def test_chunks_of_middling_size(dim, dtype):
    """A few chunks over some hundred to some thousand keys: tiles of 32 rows, by the rule."""
    _run([1500, 800, 0, 2], [100, 60, 0, 2], heads=2, group=4, dim=dim, dtype=dtype, seed=dim)
    _run([2900, 450, 777], [33, 130, 1], heads=4, group=7, dim=dim, dtype=dtype, page=24, cap=5.0, extra=3, seed=dim)
    if dim == 64:
        _run([1100] * 9, [40] * 9, heads=8, group=4, dim=dim, dtype=dtype, seed=dim)  # more of them than CUs
    _run([3000, 100], [90, 100], heads=1, group=3, dim=dim, dtype=dtype, window=500, seed=dim)


@pytest.mark.gpu
@pytest.mark.parametrize("batch,tile", [(2, 32), (7, 128), (63, 256), (64, 32), (64, 128), (65, 128)])
def test_sequences_of_mixed_lengths(plan, batch, tile):
    """More tiles than CUs: up to 64 sequences are taken by their tiles' lengths, whatever their order; some
    have no new tokens, and some no keys."""
    plan(0, None, tile)
    rows = torch.randint(0, 40, (batch,), generator=gen(batch)) * 300 // (batch + 10)
    new = [0 if i % 5 == 3 else int(n) for i, n in enumerate(rows)]
    new[-1] = 700 if batch < 10 else 90
    lens = [n + int(p) for n, p in zip(new, torch.randint(0, 300, (batch,), generator=gen(1)))]
    _run(lens, new, heads=8, group=2, dim=128 if tile == 256 else 64, window=200 * (batch % 2), seed=batch)


@pytest.mark.gpu
@pytest.mark.parametrize("dim,dtype", [(64, H), (64, B), (96, B), (128, H), (128, B)])
def test_tiles_of_two_groups_of_waves(plan, monkeypatch, dim, dtype):
    """Blocks in turn: none, one, an even and an odd number of them, and rows that see those of one group only."""
    plan(0, None, 128)
    monkeypatch.setenv("PW4_ATTN_GROUPS", "2")
    _run([600, 257, 64, 400, 0, 65], [600, 129, 1, 90, 0, 65], heads=2, group=2, dim=dim, dtype=dtype, seed=dim)
    _run([900, 333, 128], [200, 333, 70], heads=1, group=3, dim=dim, dtype=dtype, window=30, cap=4.0, page=8, seed=dim)
    _run([500], [499], heads=3, group=1, dim=dim, dtype=dtype, page=7, extra=5, seed=dim)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
def test_chunks_of_whole_tiles(dim):
    """Two groups of waves by the rule."""
    _run([1500, 1300, 1200], [200, 200, 200], heads=8, group=4, dim=dim, window=1000, seed=dim)


@pytest.mark.gpu
@pytest.mark.parametrize("groups", [1, 2])
def test_infinite_values_with_groups_of_waves(plan, monkeypatch, groups):
    """A block of NaN in a key of either group's blocks reaches only the queries that see it."""
    plan(0, None, 128)
    monkeypatch.setenv("PW4_ATTN_GROUPS", str(groups))
    lens, new, dim = [400], 300, 64
    for j in (120, 190, 399):
        def edit(ks, vs):
            vs[0][j, 0, 3] = math.inf
            ks[0][j - 20, 0, 40] = math.nan

        kc, vc, tables, ks, vs = fp4_kv(lens, 16, 1, dim, B, 8, edit=edit)
        q = torch.randn(new, 2, dim, generator=gen(9)).to(B).to(DEV)
        out, lse = ops.paged_attention_fp4(q, kc, vc, tables, _i32(lens), offsets([new]).to(DEV), new, lens[0],
                                           return_lse=True)
        ref = attention_ref(q.cpu(), ks[0], vs[0], lens[0], new, dim ** -0.5, 0, 0.0)
        fine = torch.arange(100, 400) < j - 20  # the queries that see no key of NaN
        check_attention(out.cpu()[fine], lse.cpu()[fine], [r[fine] for r in ref], dim, lens[0], B)
        assert bool(out.cpu()[~fine].isnan().all()) and bool(lse.cpu()[~fine].isnan().all())


@pytest.mark.gpu
def test_magnitudes():
    """Blocks of very different exponents, and of zeros."""
    for dtype, lo, hi in ((B, -30, 30), (H, -10, 9)):
        def edit(ks, vs):
            g = gen(5)
            for x in [*ks, *vs]:
                scale = torch.randint(lo, hi, (*x.shape[:2], x.shape[2] // 32, 1), generator=g)
                x.copy_(torch.ldexp(x.unflatten(-1, (-1, 32)), scale).flatten(-2))
                x[::3, :, :32] = 0

        for new in (1, 40):
            lens, dim = [90], 128
            kc, vc, tables, ks, vs = fp4_kv(lens, 16, 1, dim, dtype, 3, edit=edit)
            q = torch.randn(new, 2, dim, generator=gen(4)).to(dtype).to(DEV)
            scale = 2.0 ** -(hi + 4)
            out, lse = ops.paged_attention_fp4(q, kc, vc, tables, _i32(lens), offsets([new]).to(DEV), new, 90,
                                               scale=scale, return_lse=True)
            check_attention(out, lse, attention_ref(q.cpu(), ks[0], vs[0], 90, new, scale, 0, 0.0), dim, 90, dtype)


@pytest.mark.gpu
def test_rows_past_the_last_sequence_are_empty():
    _run([50, 20], [3, 1], extra=7)
    _run([200], [120], extra=150)
    _run([], [], extra=4)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [8, 100])
def test_queries_before_the_first_key_are_empty(new):
    """Fewer tokens in the cache than new ones: the first queries stand before position 0."""
    lens, page, heads, dim = [new - 5], 16, 2, 64
    kc, vc, tables, ks, vs = fp4_kv(lens, page, heads, dim, B, 3)
    q = torch.randn(new, heads * 2, dim, generator=gen(4)).to(B).to(DEV)
    out, lse = ops.paged_attention_fp4(q, kc, vc, tables, _i32(lens), offsets([new]).to(DEV), new, lens[0], return_lse=True)
    assert bool((out[:5] == 0).all()) and bool((lse[:5] == -math.inf).all())
    ref = attention_ref(q[5:].cpu(), ks[0], vs[0], lens[0], lens[0], dim ** -0.5, 0, 0.0)
    check_attention(out[5:], lse[5:], ref, dim, lens[0], B)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 33])
def test_pages_behind_the_window_may_be_gone(new):
    """Table entries of -1, or of no page at all, behind every query's window."""
    lens, page, window = [640], 16, 100
    kc, vc, tables, ks, vs = fp4_kv(lens, page, 2, 128, B, 5)
    first = lens[0] - new - window + 1  # the oldest key that the first query sees
    tables[0, :first // page] = torch.tensor([-1, 10 ** 9] * 40, dtype=torch.int32, device=DEV)[:first // page]
    q = torch.randn(new, 8, 128, generator=gen(6)).to(B).to(DEV)
    out, lse = ops.paged_attention_fp4(q, kc, vc, tables, _i32(lens), offsets([new]).to(DEV), new, lens[0], window=window,
                                       return_lse=True)
    ref = attention_ref(q.cpu(), ks[0], vs[0], lens[0], new, 128 ** -0.5, window, 0.0)
    check_attention(out, lse, ref, 128, window, B)


@pytest.mark.gpu
@pytest.mark.parametrize("split,tile", [(None, None), (0, 256), (1, 128), (None, 32)])
@pytest.mark.parametrize("new,group", [(7, 1), (40, 1), (40, 4), (300, 2)])
@pytest.mark.parametrize("dim", [64, 96])
def test_values_of_nan_reach_only_the_queries_that_see_them(plan, new, group, dim, split, tile):
    """A block of NaN among the values makes the outputs of later queries NaN in that block, and no others':
    the queries of the same chunk that stand before it do not see it."""
    plan(split, 1 if split else None, tile)
    lens, page = [new + 50], 16
    j = lens[0] - new // 2  # inside the chunk

    def edit(ks, vs):
        vs[0][j, 0, 3] = math.inf

    kc, vc, tables, ks, vs = fp4_kv(lens, page, 1, dim, B, 8, edit=edit)
    assert bool(vs[0][j, 0, :32].isnan().all()) and not bool(vs[0][j, 0, 32:].isnan().any())
    q = torch.randn(new, group, dim, generator=gen(9)).to(B).to(DEV)
    for window in (0, 30):
        out, lse = ops.paged_attention_fp4(q, kc, vc, tables, _i32(lens), offsets([new]).to(DEV), new, lens[0],
                                           window=window, return_lse=True)
        ref = attention_ref(q.cpu(), ks[0], vs[0], lens[0], new, dim ** -0.5, window, 0.0)
        check_attention(out, lse, ref, dim, lens[0], B)


@pytest.mark.gpu
@pytest.mark.parametrize("split", [0, 1])
@pytest.mark.parametrize("new,tile", [(1, None), (7, None), (60, 128), (200, 256), (60, 32)])
def test_nan_scores_have_a_nan_lse(plan, new, tile, split):
    """A query of NaN, and a key with a block of NaN for the queries that see it: out and lse are NaN, and
    no other row's change."""
    plan(split, 1, tile)
    lens, page, dim = [new + 130], 16, 64
    j = lens[0] - 1 - (new - 1) // 2  # its queries: those from new - 1 - (new - 1) // 2 on
    kc, vc, tables, ks, vs = fp4_kv(lens, page, 2, dim, B, 8)
    q = torch.randn(new, 4, dim, generator=gen(9)).to(B)
    args = (_i32(lens), offsets([new]).to(DEV), new, lens[0])
    ref = attention_ref(q, ks[0], vs[0], lens[0], new, dim ** -0.5, 0, 0.0)

    def check(out, lse, bad):  # bad [new, 4]
        assert torch.equal(lse.cpu().isnan(), bad) and torch.equal(out.cpu().isnan().all(-1), bad)
        fine = ~bad
        check_attention(out.cpu()[fine], lse.cpu()[fine], [r[fine] for r in ref], dim, lens[0], B)

    bad = torch.zeros(new, 4, dtype=torch.bool)
    bad[new // 2, 1] = True
    broken = torch.where(bad[..., None], math.nan, q)
    check(*ops.paged_attention_fp4(broken.to(DEV), kc, vc, tables, *args, return_lse=True), bad)

    def edit(ks, vs):
        ks[0][j, 1, 5] = math.nan

    kc, vc, tables, _, _ = fp4_kv(lens, page, 2, dim, B, 8, edit=edit)
    bad = torch.zeros(new, 4, dtype=torch.bool)
    bad[new - 1 - (new - 1) // 2:, 2:] = True
    check(*ops.paged_attention_fp4(q.to(DEV), kc, vc, tables, *args, return_lse=True), bad)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 50])
def test_keys_of_nan_that_are_not_seen(new):
    """Blocks of NaN behind the window; what nothing has written is NaN as well."""
    lens, page, dim, window = [300], 16, 64, 64
    def edit(ks, vs):
        for j in range(0, lens[0] - new - window + 1, 7):
            ks[0][j], vs[0][j] = math.nan, math.inf

    kc, vc, tables, ks, vs = fp4_kv(lens, page, 1, dim, H, 8, edit=edit)
    ks[0], vs[0] = ks[0].nan_to_num(0.0), vs[0].nan_to_num(0.0)
    q = torch.randn(new, 2, dim, generator=gen(9)).to(H).to(DEV)
    out, lse = ops.paged_attention_fp4(q, kc, vc, tables, _i32(lens), offsets([new]).to(DEV), new, lens[0], window=window,
                                       return_lse=True)
    ref = attention_ref(q.cpu(), ks[0], vs[0], lens[0], new, dim ** -0.5, window, 0.0)
    check_attention(out, lse, ref, dim, lens[0], H)


@pytest.mark.gpu
def test_large_scores_do_not_overflow():
    """Scores of some thousand either way, and equal ones."""
    for dtype in (H, B):
        q = (torch.randn(3, 4, 64, generator=gen(1)) * 60).to(dtype).to(DEV)
        _run([200], [3], heads=1, group=4, dim=64, dtype=dtype, scale=1.0, q=q)
        _run([200], [3], heads=1, group=4, dim=64, dtype=dtype, q=torch.zeros_like(q))


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 70])
def test_query_strides(new):
    lens, heads, group, dim = [230, 71], 2, 4, 128
    hq = heads * group
    # a slice of a fused q|k|v projection, then one that 16-byte loads cannot read in place
    for shift in (0, 3):
        fused = torch.randn(2 * new, hq * dim + 2 * heads * dim + 8, generator=gen(2)).to(B).to(DEV)
        q = fused[:, shift:shift + hq * dim].view(2 * new, hq, dim)
        _run(lens, [new, new], heads=heads, group=group, dim=dim, q=q, seed=4)
    q = torch.randn(hq, 2 * new, dim, generator=gen(2)).to(B).to(DEV).transpose(0, 1)
    _run(lens, [new, new], heads=heads, group=group, dim=dim, q=q, seed=5)
    _run(lens, [new, new], heads=heads, group=group, dim=dim, q=q.transpose(1, 2).contiguous().transpose(1, 2), seed=5)


@pytest.mark.gpu
def test_wide_tables_and_table_strides():
    """A table of more columns than any row uses, rows apart, of garbage past the used ones."""
    lens, new = [100, 260], [1, 40]
    kc, vc, tables, ks, vs = fp4_kv(lens, 16, 2, 128, B, 1)
    wide = torch.randint(-2 ** 31, 2 ** 31 - 1, (2, 90), dtype=torch.int32, device=DEV)
    for b, l in enumerate(lens):
        wide[b, :-(-l // 16)] = tables[b, :-(-l // 16)]
    q = torch.randn(41, 4, 128, generator=gen(1)).to(B).to(DEV)
    args = (_i32(lens), offsets(new).to(DEV))
    a = ops.paged_attention_fp4(q, kc, vc, tables, *args, 40, 260)
    for w in (wide, wide[:, :80]):
        assert torch.equal(a, ops.paged_attention_fp4(q, kc, vc, w, *args, 40, 260))


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """A pool of more than 2^32 bytes whose sequence lies at its end."""
    page, heads, dim = 64, 8, 128
    pages = 2 ** 32 // (page * heads * row_bytes(dim)) + 64
    pool = torch.zeros(2, pages, page, heads, row_bytes(dim), dtype=torch.uint8, device=DEV)
    for new in (1, 40):
        lens = [150]
        kc, vc, tables, ks, vs = fp4_kv(lens, page, heads, dim, B, 4)
        far = tables.clone()
        for c in range(3):
            far[0, c] = pages - 1 - c
            pool[0, pages - 1 - c] = kc[int(tables[0, c])]
            pool[1, pages - 1 - c] = vc[int(tables[0, c])]
        q = torch.randn(new, heads, dim, generator=gen(1)).to(B).to(DEV)
        args = (_i32(lens), offsets([new]).to(DEV), new, 150)
        assert torch.equal(ops.paged_attention_fp4(q, kc, vc, tables, *args),
                           ops.paged_attention_fp4(q, pool[0], pool[1], far, *args))


@pytest.mark.gpu
@pytest.mark.parametrize("name", [-1, 10 ** 9, -2 ** 31])
@pytest.mark.parametrize("new", [1, 40])
def test_page_ids_outside_the_pool_read_its_last_page(new, name):
    lens, page = [130], 16
    kc, vc, tables, _, _ = fp4_kv(lens, page, 2, 64, B, 5, fill=0x21)
    q = torch.randn(new, 4, 64, generator=gen(6)).to(B).to(DEV)
    args = (_i32(lens), offsets([new]).to(DEV), new, lens[0])
    got = []
    for page_id in (name, kc.shape[0] - 1):
        tables[0, 2] = page_id
        got.append(ops.paged_attention_fp4(q, kc, vc, tables, *args))
    assert torch.equal(*got)


@pytest.mark.gpu
@pytest.mark.parametrize("split", [0, 1])
@pytest.mark.parametrize("most,tile", [(0, None), (1, None), (5, None), (40, 128), (90, 256), (40, 32), (90, 32)])
def test_queries_past_max_q_len_are_empty(plan, most, tile, split):
    plan(split, 1, tile)
    lens, new, dim = [300, 150, 2, 40], [100, 150, 2, 0], 64
    kc, vc, tables, ks, vs = fp4_kv(lens, 16, 2, dim, B, 3)
    q = torch.randn(sum(new) + 3, 4, dim, generator=gen(4)).to(B).to(DEV)
    cu = offsets(new)
    out, lse = ops.paged_attention_fp4(q, kc, vc, tables, _i32(lens), cu.to(DEV), most, max(lens), return_lse=True)
    computed = torch.zeros(q.shape[0], dtype=torch.bool)
    for b, n in enumerate(new):
        c0, m = int(cu[b]), min(n, most)
        if m == 0:
            continue
        computed[c0:c0 + m] = True
        ref = attention_ref(q[c0:c0 + n].cpu(), ks[b], vs[b], lens[b], n, dim ** -0.5, 0, 0.0)
        check_attention(out[c0:c0 + m], lse[c0:c0 + m], [r[:m] for r in ref], dim, lens[b], B)
    assert bool((out.cpu()[~computed] == 0).all()) and bool((lse.cpu()[~computed] == -math.inf).all())


@pytest.mark.gpu
@pytest.mark.parametrize("lens,new", [([3000, 900], [1, 1]), ([1200, 300], [200, 300])])
def test_repeats_streams_and_graphs(lens, new):
    """The same bits on every call: on another stream, and in a graph's replays between eager calls."""
    kc, vc, tables, _, _ = fp4_kv(lens, 16, 2, 128, B, 1)
    q = torch.randn(sum(new), 8, 128, generator=gen(1)).to(B).to(DEV)
    lens_t, cu = _i32(lens), offsets(new).to(DEV)

    def call():
        return ops.paged_attention_fp4(q, kc, vc, tables, lens_t, cu, max(new), 3000, return_lse=True)

    first = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = call()
        graph = torch.cuda.CUDAGraph()
    side.synchronize()
    with torch.cuda.graph(graph, stream=side):
        captured = call()
    for _ in range(3):
        for t in captured:
            t.fill_(7)
        graph.replay()
        eager = call()
        torch.cuda.synchronize()
        for a, b, c, d in zip(first, other, captured, eager):
            assert torch.equal(a, b) and torch.equal(a, c) and torch.equal(a, d)
    # a graph follows lengths that change on the device between replays
    lens_t.sub_(_i32([17, 0]))
    graph.replay()
    for a, b in zip(captured, call()):
        assert torch.equal(a, b)


def _good():
    kc, vc, tables, _, _ = fp4_kv([20], 16, 2, 64, B, 1)
    q = torch.zeros(1, 4, 64, dtype=B, device=DEV)
    return dict(q=q, k_cache=kc, v_cache=vc, block_tables=tables, seq_lens=_i32([20]), cu_q=offsets([1]).to(DEV),
                max_q_len=1, max_seq_len=20)


@pytest.mark.gpu
@pytest.mark.parametrize("change,message", [
    (lambda a: dict(q=a["q"].float()), "fp16 or bf16"),
    (lambda a: dict(q=a["q"][0]), "3-D"),
    (lambda a: dict(q=a["q"][:, :3]), "multiple of kv_heads"),
    (lambda a: dict(q=a["q"][..., :32]), "head_dim"),
    (lambda a: dict(q=a["q"].cpu()), "one CUDA device|CUDA tensors"),
    (lambda a: dict(v_cache=a["v_cache"][:-1]), "one shape"),
    (lambda a: dict(k_cache=a["k_cache"].bfloat16(), v_cache=a["v_cache"].bfloat16()), "uint8"),
    (lambda a: dict(k_cache=a["k_cache"][..., :17], v_cache=a["v_cache"][..., :17]), "contiguous"),
    (lambda a: dict(k_cache=a["k_cache"][..., :33], v_cache=a["v_cache"][..., :33]), "multiple of 32"),
    (lambda a: dict(k_cache=a["k_cache"][:, :8], v_cache=a["v_cache"][:, :8].clone()), "one shape"),
    (lambda a: dict(k_cache=a["k_cache"].transpose(1, 2), v_cache=a["v_cache"].transpose(1, 2)), "contiguous"),
    (lambda a: dict(block_tables=a["block_tables"].long()), "int32"),
    (lambda a: dict(seq_lens=a["seq_lens"].repeat(2)), "rows of block_tables"),
    (lambda a: dict(cu_q=a["cu_q"][:1]), "batch"),
    (lambda a: dict(window=-1), "window"),
    (lambda a: dict(softcap=-1.0), "softcap"),
    (lambda a: dict(scale=math.inf), "scale"),
    (lambda a: dict(max_seq_len=-1), "max_seq_len"),
])
def test_refusals(change, message):
    args = _good()
    ops.paged_attention_fp4(**args)
    args.update(change(args))
    with pytest.raises(RuntimeError, match=message):
        ops.paged_attention_fp4(**args)


@pytest.mark.gpu
def test_refuses_unaligned_pages():
    args = _good()
    n, size = args["k_cache"].shape[0], args["k_cache"][0].numel()
    raw = torch.zeros(n * (size + 16) + 64, dtype=torch.uint8, device=DEV)
    for first, apart in ((8, size), (0, size + 8), (0, size - 16)):
        cache = raw.as_strided(args["k_cache"].shape, (apart, *args["k_cache"].stride()[1:]), first)
        with pytest.raises(RuntimeError, match="aligned|overlap"):
            ops.paged_attention_fp4(**dict(args, k_cache=cache, v_cache=cache))


class _Args(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in ("q", "k_cache", "v_cache", "block_tables", "seq_lens", "cu_q", "out",
                                                "lse")]
                + [(n, ctypes.c_int64) for n in (
                    "num_tokens", "batch", "q_heads", "kv_heads", "head_dim", "num_pages", "page_size", "table_width",
                    "table_stride", "q_token_stride", "q_head_stride", "page_stride", "row_stride", "kv_head_stride",
                    "max_q_len", "max_seq_len", "window")]
                + [("scale", ctypes.c_float), ("softcap", ctypes.c_float), ("dtype", ctypes.c_int)])


def _lib():
    lib = pulsar_amd.capi()
    lib.pw4_paged_attention_fp4.argtypes = [ctypes.POINTER(_Args), ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p]
    lib.pw4_paged_attention_fp4_workspace_size.argtypes = [ctypes.POINTER(_Args)]
    lib.pw4_paged_attention_fp4_workspace_size.restype = ctypes.c_size_t
    return lib


def test_c_entry_refuses_before_any_launch():
    lib = _lib()
    good = dict(q=4096, k_cache=4096, v_cache=4096, block_tables=4096, seq_lens=4096, cu_q=4096, out=4096, num_tokens=1,
                batch=1, q_heads=4, kv_heads=2, head_dim=64, num_pages=4, page_size=16, table_width=2, table_stride=2,
                q_token_stride=256, q_head_stride=64, page_stride=16 * 2 * 34, max_q_len=1, max_seq_len=32, scale=1.0,
                dtype=1)

    def call(**change):
        return lib.pw4_paged_attention_fp4(ctypes.byref(_Args(**dict(good, **change))), None, 0, None)

    assert lib.pw4_paged_attention_fp4(None, None, 0, None) == -1
    assert call(dtype=2) == -1 and call(num_tokens=-1) == -1
    assert call(head_dim=40) == -2 and call(head_dim=288) == -2 and call(head_dim=0) == -2
    assert call(q_heads=3) == -2 and call(kv_heads=0) == -1 and call(table_stride=1) == -2
    assert call(softcap=math.nan) == -1 and call(scale=math.inf) == -1
    assert call(q=None) == -1 and call(k_cache=None) == -1 and call(cu_q=None) == -1
    assert call(q=4098) == -1 and call(v_cache=4104) == -1 and call(page_stride=16 * 2 * 34 + 8) == -1
    assert call(page_stride=16 * 2 * 34 - 16) == -2 and call(page_stride=-16) == -1 and call(page_stride=2 ** 31) == -2
    assert call(page_size=0) == -1 and call(page_size=2 ** 24) == -2 and call(max_seq_len=2 ** 40) == -2
    assert call(num_tokens=0, q=None) == 0
    # a sequence whose keys are split needs the workspace that it asks for
    big = _Args(**dict(good, table_width=10000, table_stride=10000, max_seq_len=100000))
    assert lib.pw4_paged_attention_fp4_workspace_size(ctypes.byref(big)) > 0
    assert lib.pw4_paged_attention_fp4(ctypes.byref(big), None, 0, None) == -3


def test_fake_kernel():
    q = torch.empty(5, 8, 64, dtype=B, device="meta")
    kc = torch.empty(4, 16, 2, 34, dtype=torch.uint8, device="meta")
    i = torch.empty(1, 2, dtype=torch.int32, device="meta")
    out, lse = ops.paged_attention_fp4(q, kc, kc, i, i[0, :1], i[0], 5, 32, return_lse=True)
    assert out.shape == q.shape and out.dtype == B and lse.shape == (5, 8) and lse.dtype == torch.float32


@pytest.mark.gpu
def test_opcheck():
    torch.library.opcheck(torch.ops.pulsar.paged_attention_fp4.default, tuple(_good().values()),
                          test_utils=("test_schema", "test_faketensor", "test_aot_dispatch_dynamic"))


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 100])
def test_no_sequences_and_a_far_bound(new):
    kc = torch.zeros(40, 16, 2, 34, dtype=torch.uint8, device=DEV)
    none = torch.zeros(0, 9000, dtype=torch.int32, device=DEV)
    q = torch.ones(new, 4, 64, dtype=B, device=DEV)
    out, lse = ops.paged_attention_fp4(q, kc, kc, none, none[:, 0].contiguous(), offsets([]).to(DEV), new, 9000 * 16,
                                       return_lse=True)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())


@pytest.mark.gpu
@pytest.mark.parametrize("split", [0, 1])
@pytest.mark.parametrize("tile,new", [(None, 1), (None, 7), (128, 40), (256, 150), (32, 40)])
@pytest.mark.parametrize("dim", [64, 96, 256])
def test_writes_stay_in_the_outputs_and_the_workspace(plan, dim, tile, new, split):
    """The C entry on buffers with a margin behind each."""
    plan(split, 1, tile)
    lens, group, heads = [900, 333, new, 61], 4, 2
    counts = [new, min(new, 40), new, 0]
    kc, vc, tables, _, _ = fp4_kv(lens, 16, heads, dim, B, 3)
    q = torch.randn(sum(counts) + 1, heads * group, dim, generator=gen(4)).to(B).to(DEV)
    lens_t, cu = _i32(lens), offsets(counts).to(DEV)
    want = ops.paged_attention_fp4(q, kc, vc, tables, lens_t, cu, new, 900, return_lse=True)
    out = torch.full((q.numel() + 64,), 3.0, dtype=B, device=DEV)
    lse = torch.full((q.shape[0] * q.shape[1] + 64,), 3.0, device=DEV)
    a = _Args(q=q.data_ptr(), k_cache=kc.data_ptr(), v_cache=vc.data_ptr(), block_tables=tables.data_ptr(),
              seq_lens=lens_t.data_ptr(), cu_q=cu.data_ptr(), out=out.data_ptr(), lse=lse.data_ptr(),
              num_tokens=q.shape[0], batch=4, q_heads=heads * group, kv_heads=heads, head_dim=dim,
              num_pages=kc.shape[0], page_size=16, table_width=tables.shape[1], table_stride=tables.stride(0),
              q_token_stride=q.stride(0), q_head_stride=q.stride(1), page_stride=kc.stride(0), max_q_len=new,
              max_seq_len=900, scale=dim ** -0.5, dtype=1)
    lib = _lib()
    size = lib.pw4_paged_attention_fp4_workspace_size(ctypes.byref(a))
    assert (size > 0) == (split == 1 and not (tile == 32 and dim < 256))  # (tiles of 32 rows are not split)
    ws = torch.full((size + 256,), 0x5a, dtype=torch.uint8, device=DEV)
    torch.cuda.synchronize()
    assert lib.pw4_paged_attention_fp4(ctypes.byref(a), ws.data_ptr(), size, None) == 0
    torch.cuda.synchronize()
    assert torch.equal(out[:q.numel()].view(q.shape), want[0]) and torch.equal(lse[:-64].view(want[1].shape), want[1])
    assert bool((out[q.numel():] == 3).all()) and bool((lse[-64:] == 3).all()) and bool((ws[size:] == 0x5a).all())


def test_the_host_rounds_to_the_nearest_code():
    """fp4_case itself: a value in range is off by half a step at most, halves go to even codes."""
    x = torch.linspace(-7, 7, 32 * 101)[torch.randperm(32 * 101, generator=gen(0))].view(101, 32)
    codes, exps, values = fp4_round(x)
    unit = torch.ldexp(torch.ones(101, dtype=torch.float64), exps[:, 0] - 127)[:, None]
    top = x.abs().amax(1, keepdim=True)
    assert bool((top >= 3.5 * unit).all()) and bool((top < 7 * unit).all())
    m = (x.double() / unit).abs()
    half = torch.where(m < 2, 0.25, torch.where(m < 4, 0.5, 1.0))
    assert bool(((values - x).abs() <= half * unit).all()) and bool((codes < 16).all())
    ties = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -5.0] + [0.0] * 22)
    assert fp4_round(ties)[2][:10].tolist() == [6.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, -0.0, -4.0]
    assert fp4_round(torch.zeros(32))[1].tolist() == [0]
    assert fp4_round(torch.full((32,), 65504.0), fp16=True)[2].tolist() == [6 * 2.0 ** 13] * 32
