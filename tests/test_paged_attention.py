"""paged_attention against its definition in 64 bits: head layouts, page sizes, windows, caps, chunk
and context lengths from none to some thousand, what unused slots hold, strides, streams, graphs and
refusals.  The bounds are derived in paged_case.check_attention."""

import ctypes
import math

import pytest
import torch

import pulsar_amd
from paged_case import DEV, attention_ref, check_attention, gen, offsets, paged_kv
from pulsar_amd import ops

H, B = torch.float16, torch.bfloat16


def _run(lens, new, *, heads=2, group=4, dim=128, page=16, dtype=B, window=0, cap=0.0, scale=None, layout="nhd",
         seed=0, q=None, extra=0, lse=True):
    """Runs one call and checks every sequence; returns (out, lse)."""
    kc, vc, tables, ks, vs = paged_kv(lens, page, heads, dim, dtype, seed, layout)
    t = sum(new) + extra
    if q is None:
        q = torch.randn(t, heads * group, dim, generator=gen(seed + 1)).to(dtype).to(DEV)
    cu = offsets(new)
    got = ops.paged_attention(q, kc, vc, tables, torch.tensor(lens, dtype=torch.int32, device=DEV), cu.to(DEV),
                              max(new + [0]), max(lens + [0]), scale=scale, window=window, softcap=cap, return_lse=lse)
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


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [H, B])
@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 63, 64, 65, 127, 129, 500, 1025])
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
@pytest.mark.parametrize("dim", [8, 16, 40, 64, 80, 96, 120, 128, 136, 192, 256])
@pytest.mark.parametrize("new", [1, 130])
def test_head_dims(dim, new, dtype):
    _run([333, 140], [new, new], heads=2, group=2, dim=dim, dtype=dtype, seed=dim)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [1, 7, 8, 16, 24, 32, 60, 64, 128, 256, 1000])
@pytest.mark.parametrize("new", [1, 40])
def test_page_sizes(page, new):
    """Pages that end inside a block of keys, and pages of many blocks."""
    _run([421, 64, 40], [new, new, new], page=page, seed=page)


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
@pytest.mark.parametrize("tile", [128, 256])
@pytest.mark.parametrize("dim,dtype", [(64, H), (128, B), (96, B), (256, H)])
def test_many_rows_whole_and_split(plan, dim, dtype, tile, split, units):
    plan(split, units, tile)
    _run([600, 257, 64, 400], [600, 129, 1, 90], heads=2, group=2, dim=dim, dtype=dtype, seed=dim)
    _run([900, 333], [200, 333], heads=1, group=3, dim=dim, dtype=dtype, window=150, cap=4.0, page=8, seed=dim)
    _run([1000, 50], [70, 50], heads=1, group=7, dim=dim, dtype=dtype, page=24, window=300, seed=dim)
    _run([500], [499], heads=3, group=1, dim=dim, dtype=dtype, page=7, extra=5, seed=dim)


@pytest.mark.gpu
@pytest.mark.parametrize("tile", [128, 256])
@pytest.mark.parametrize("split", [0, 1])
def test_nonfinite_values_in_wide_and_split_tiles(plan, tile, split):
    plan(split, 1, tile)
    lens, page, dim, new = [700], 16, 128, 400
    kc, vc, tables, ks, vs = paged_kv(lens, page, 1, dim, B, 8)
    for j, bad in ((310, math.nan), (480, math.inf), (650, -math.inf)):
        vs[0][j, 0, j % dim] = bad
        vc[int(tables[0, j // page]), j % page, 0, j % dim] = bad
    q = torch.randn(new, 2, dim, generator=gen(9)).to(B).to(DEV)
    for window in (0, 120):
        out, lse = ops.paged_attention(q, kc, vc, tables, torch.tensor(lens, dtype=torch.int32, device=DEV),
                                       offsets([new]).to(DEV), new, lens[0], window=window, return_lse=True)
        ref = attention_ref(q.cpu(), ks[0], vs[0], lens[0], new, dim ** -0.5, window, 0.0)
        check_attention(out, lse, ref, dim, lens[0], B)


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
    kc, vc, tables, ks, vs = paged_kv(lens, page, heads, dim, B, 3)
    q = torch.randn(new, heads * 2, dim, generator=gen(4)).to(B).to(DEV)
    out, lse = ops.paged_attention(q, kc, vc, tables, torch.tensor(lens, dtype=torch.int32, device=DEV),
                                   offsets([new]).to(DEV), new, lens[0], return_lse=True)
    assert bool((out[:5] == 0).all()) and bool((lse[:5] == -math.inf).all())
    ref = attention_ref(q[5:].cpu(), ks[0], vs[0], lens[0], lens[0], dim ** -0.5, 0, 0.0)
    check_attention(out[5:], lse[5:], ref, dim, lens[0], B)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 33])
def test_pages_behind_the_window_may_be_gone(new):
    """Table entries of -1, or of no page at all, behind every query's window."""
    lens, page, window = [640], 16, 100
    kc, vc, tables, ks, vs = paged_kv(lens, page, 2, 128, B, 5)
    first = lens[0] - new - window + 1  # the oldest key that the first query sees
    tables[0, :first // page] = torch.tensor([-1, 10 ** 9] * 40, dtype=torch.int32, device=DEV)[:first // page]
    q = torch.randn(new, 8, 128, generator=gen(6)).to(B).to(DEV)
    out, lse = ops.paged_attention(q, kc, vc, tables, torch.tensor(lens, dtype=torch.int32, device=DEV),
                                   offsets([new]).to(DEV), new, lens[0], window=window, return_lse=True)
    ref = attention_ref(q.cpu(), ks[0], vs[0], lens[0], new, 128 ** -0.5, window, 0.0)
    check_attention(out, lse, ref, 128, window, B)


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("new,group", [(40, 1), (40, 4), (300, 2)])
def test_nonfinite_values_reach_only_the_queries_that_see_them(bad, new, group):
    """A key whose value is not finite makes the outputs of later queries non-finite, and no others':
    the queries of the same chunk that stand before it do not see it."""
    lens, page, dim = [new + 50], 16, 64
    kc, vc, tables, ks, vs = paged_kv(lens, page, 1, dim, B, 8)
    j = lens[0] - new // 2  # inside the chunk
    vs[0][j, 0, 3] = bad
    vc[int(tables[0, j // page]), j % page, 0, 3] = bad
    q = torch.randn(new, group, dim, generator=gen(9)).to(B).to(DEV)
    out, lse = ops.paged_attention(q, kc, vc, tables, torch.tensor(lens, dtype=torch.int32, device=DEV),
                                   offsets([new]).to(DEV), new, lens[0], return_lse=True)
    ref = attention_ref(q.cpu(), ks[0], vs[0], lens[0], new, dim ** -0.5, 0, 0.0)
    check_attention(out, lse, ref, dim, lens[0], B)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 50])
def test_nonfinite_keys_that_are_not_seen(new):
    """Keys of NaN behind the window and after the query."""
    lens, page, dim, window = [300], 16, 64, 64
    kc, vc, tables, ks, vs = paged_kv(lens, page, 1, dim, H, 8)
    for j in range(0, lens[0] - new - window + 1, 7):
        kc[int(tables[0, j // page]), j % page] = math.nan
        vc[int(tables[0, j // page]), j % page] = math.inf
        ks[0][j], vs[0][j] = 0, 0
    q = torch.randn(new, 2, dim, generator=gen(9)).to(H).to(DEV)
    out, lse = ops.paged_attention(q, kc, vc, tables, torch.tensor(lens, dtype=torch.int32, device=DEV),
                                   offsets([new]).to(DEV), new, lens[0], window=window, return_lse=True)
    ref = attention_ref(q.cpu(), ks[0], vs[0], lens[0], new, dim ** -0.5, window, 0.0)
    check_attention(out, lse, ref, dim, lens[0], H)


@pytest.mark.gpu
def test_large_scores_do_not_overflow():
    """Scores of some thousand either way, and equal ones."""
    for dtype in (H, B):
        lens, new, dim = [200], [3], 64
        q = (torch.randn(3, 4, dim, generator=gen(1)) * 60).to(dtype).to(DEV)
        _run(lens, new, heads=1, group=4, dim=dim, dtype=dtype, scale=1.0, q=q)
        _run(lens, new, heads=1, group=4, dim=dim, dtype=dtype, q=torch.zeros_like(q))


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 70])
def test_layouts_and_strides(new):
    lens, heads, group, dim = [230, 71], 2, 4, 128
    _run(lens, [new, new], heads=heads, group=group, dim=dim, layout="hnd", seed=3)
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
    kc, vc, tables, ks, vs = paged_kv(lens, 16, 2, 128, B, 1)
    wide = torch.randint(-2 ** 31, 2 ** 31 - 1, (2, 90), dtype=torch.int32, device=DEV)
    for b, l in enumerate(lens):
        wide[b, :-(-l // 16)] = tables[b, :-(-l // 16)]
    q = torch.randn(41, 4, 128, generator=gen(1)).to(B).to(DEV)
    args = (torch.tensor(lens, dtype=torch.int32, device=DEV), offsets(new).to(DEV))
    a = ops.paged_attention(q, kc, vc, tables, *args, 40, 260)
    for w in (wide, wide[:, :80]):
        assert torch.equal(a, ops.paged_attention(q, kc, vc, w, *args, 40, 260))
        # bounds that are far above what the batch holds only change the split
        b = ops.paged_attention(q, kc, vc, w, *args, 41, 80 * 16)
        assert float((a.float() - b.float()).abs().max()) <= 2.0 ** -7 * float(a.float().abs().max())


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """A pool of more than 2^32 bytes whose sequence lies at its end."""
    page, heads, dim = 64, 8, 128
    pages = 2 ** 32 // (page * heads * dim * 2) + 64
    pool = torch.zeros(2, pages, page, heads, dim, dtype=B, device=DEV)
    for new in (1, 40):
        lens = [150]
        kc, vc, tables, ks, vs = paged_kv(lens, page, heads, dim, B, 4)
        far = tables.clone()
        for c in range(3):
            far[0, c] = pages - 1 - c
            pool[0, pages - 1 - c] = kc[int(tables[0, c])]
            pool[1, pages - 1 - c] = vc[int(tables[0, c])]
        q = torch.randn(new, heads, dim, generator=gen(1)).to(B).to(DEV)
        args = (torch.tensor(lens, dtype=torch.int32, device=DEV), offsets([new]).to(DEV), new, 150)
        assert torch.equal(ops.paged_attention(q, kc, vc, tables, *args), ops.paged_attention(q, pool[0], pool[1], far, *args))


@pytest.mark.gpu
@pytest.mark.parametrize("lens,new", [([3000, 900], [1, 1]), ([1200, 300], [200, 300])])
def test_repeats_streams_and_graphs(lens, new):
    """The same bits on every call: on another stream, and in a graph's replays between eager calls."""
    kc, vc, tables, _, _ = paged_kv(lens, 16, 2, 128, B, 1)
    q = torch.randn(sum(new), 8, 128, generator=gen(1)).to(B).to(DEV)
    lens_t, cu = torch.tensor(lens, dtype=torch.int32, device=DEV), offsets(new).to(DEV)

    def call():
        return ops.paged_attention(q, kc, vc, tables, lens_t, cu, max(new), 4096, return_lse=True)

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
    lens_t.sub_(torch.tensor([17, 0], dtype=torch.int32, device=DEV))
    graph.replay()
    for a, b in zip(captured, call()):
        assert torch.equal(a, b)


def _good():
    kc, vc, tables, _, _ = paged_kv([20], 16, 2, 64, B, 1)
    q = torch.zeros(1, 4, 64, dtype=B, device=DEV)
    return dict(q=q, k_cache=kc, v_cache=vc, block_tables=tables,
                seq_lens=torch.tensor([20], dtype=torch.int32, device=DEV), cu_q=offsets([1]).to(DEV), max_q_len=1,
                max_seq_len=20)


@pytest.mark.gpu
@pytest.mark.parametrize("change,message", [
    (lambda a: dict(q=a["q"].half()), "one dtype"),
    (lambda a: dict(q=a["q"].float()), "fp16 or bf16"),
    (lambda a: dict(q=a["q"][0]), "3-D"),
    (lambda a: dict(q=a["q"][:, :3]), "multiple of kv_heads"),
    (lambda a: dict(q=a["q"][..., :32]), "head_dim"),
    (lambda a: dict(q=a["q"].cpu()), "one CUDA device|CUDA tensors"),
    (lambda a: dict(v_cache=a["v_cache"][:-1]), "one shape"),
    (lambda a: dict(k_cache=a["k_cache"].float(), v_cache=a["v_cache"].float()), "one dtype"),
    (lambda a: dict(k_cache=a["k_cache"].transpose(2, 3).contiguous().transpose(2, 3),
                    v_cache=a["v_cache"].transpose(2, 3).contiguous().transpose(2, 3)), "last dimension"),
    (lambda a: dict(block_tables=a["block_tables"].long()), "int32"),
    (lambda a: dict(seq_lens=a["seq_lens"].repeat(2)), "rows of block_tables"),
    (lambda a: dict(cu_q=a["cu_q"][:1]), "batch"),
    (lambda a: dict(window=-1), "window"),
    (lambda a: dict(softcap=-1.0), "softcap"),
    (lambda a: dict(softcap=math.nan), "softcap"),
    (lambda a: dict(scale=math.inf), "scale"),
    (lambda a: dict(max_seq_len=-1), "max_seq_len"),
])
def test_refusals(change, message):
    args = _good()
    ops.paged_attention(**args)
    args.update(change(args))
    with pytest.raises(RuntimeError, match=message):
        ops.paged_attention(**args)


@pytest.mark.gpu
def test_refuses_unaligned_caches_and_odd_dims():
    args = _good()
    raw = torch.zeros(2 * args["k_cache"].numel() + 8, dtype=B, device=DEV)
    shape = args["k_cache"].shape
    n = args["k_cache"].numel()
    args.update(k_cache=raw[1:1 + n].view(shape), v_cache=raw[1 + n:1 + 2 * n].view(shape))
    with pytest.raises(RuntimeError, match="aligned"):
        ops.paged_attention(**args)
    odd = _good()
    odd.update(q=odd["q"][..., :60], k_cache=odd["k_cache"][..., :60], v_cache=odd["v_cache"][..., :60])
    with pytest.raises(RuntimeError, match="multiple of 8"):
        ops.paged_attention(**odd)


class _Args(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in ("q", "k_cache", "v_cache", "block_tables", "seq_lens", "cu_q", "out",
                                                "lse")]
                + [(n, ctypes.c_int64) for n in (
                    "num_tokens", "batch", "q_heads", "kv_heads", "head_dim", "num_pages", "page_size", "table_width",
                    "table_stride", "q_token_stride", "q_head_stride", "page_stride", "row_stride", "kv_head_stride",
                    "max_q_len", "max_seq_len", "window")]
                + [("scale", ctypes.c_float), ("softcap", ctypes.c_float), ("dtype", ctypes.c_int)])


def test_c_entry_refuses_before_any_launch():
    lib = pulsar_amd.capi()
    lib.pw4_paged_attention.argtypes = [ctypes.POINTER(_Args), ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p]
    lib.pw4_paged_attention_workspace_size.argtypes = [ctypes.POINTER(_Args)]
    lib.pw4_paged_attention_workspace_size.restype = ctypes.c_size_t

    def call(**change):
        a = dict(q=4096, k_cache=4096, v_cache=4096, block_tables=4096, seq_lens=4096, cu_q=4096, out=4096,
                 num_tokens=1, batch=1, q_heads=4, kv_heads=2, head_dim=64, num_pages=4, page_size=16, table_width=2,
                 table_stride=2, q_token_stride=256, q_head_stride=64, page_stride=2048, row_stride=128,
                 kv_head_stride=64, max_q_len=1, max_seq_len=32, scale=1.0, dtype=1)
        a.update(change)
        args = _Args(**a)
        return lib.pw4_paged_attention(ctypes.byref(args), None, 0, None)

    assert lib.pw4_paged_attention(None, None, 0, None) == -1
    assert call(dtype=2) == -1
    assert call(num_tokens=-1) == -1
    assert call(head_dim=60) == -2 and call(head_dim=264) == -2 and call(head_dim=0) == -2
    assert call(q_heads=3) == -2 and call(kv_heads=0) == -1
    assert call(table_stride=1) == -2
    assert call(softcap=-1.0) == -1 and call(softcap=math.nan) == -1
    assert call(q=None) == -1 and call(k_cache=None) == -1 and call(cu_q=None) == -1
    assert call(q=4098) == -1 and call(row_stride=132) == -1
    assert call(window=-1) == -1 and call(page_size=0) == -1
    assert call(max_seq_len=2 ** 40) == -2
    assert call(num_tokens=0, q=None) == 0
    # a sequence whose keys are split needs the workspace that it asks for
    big = _Args(q=4096, k_cache=4096, v_cache=4096, block_tables=4096, seq_lens=4096, cu_q=4096, out=4096,
                num_tokens=1, batch=1, q_heads=4, kv_heads=2, head_dim=64, num_pages=4, page_size=16,
                table_width=10000, table_stride=10000, q_token_stride=256, q_head_stride=64, page_stride=2048,
                row_stride=128, kv_head_stride=64, max_q_len=1, max_seq_len=100000, scale=1.0, dtype=1)
    if lib.pw4_paged_attention_workspace_size(ctypes.byref(big)) > 0:
        assert lib.pw4_paged_attention(ctypes.byref(big), None, 0, None) == -3


def test_fake_kernel():
    q = torch.empty(5, 8, 64, dtype=B, device="meta")
    kc = torch.empty(4, 16, 2, 64, dtype=B, device="meta")
    i = torch.empty(1, 2, dtype=torch.int32, device="meta")
    out, lse = ops.paged_attention(q, kc, kc, i, i[0, :1], i[0], 5, 32, return_lse=True)
    assert out.shape == q.shape and out.dtype == B and lse.shape == (5, 8) and lse.dtype == torch.float32


@pytest.mark.gpu
def test_opcheck():
    torch.library.opcheck(torch.ops.pulsar.paged_attention.default, tuple(_good().values()),
                          test_utils=("test_schema", "test_faketensor", "test_aot_dispatch_dynamic"))


def _one_key(values, dtype, n=1, **options):
    """lse of queries that see one key each, whose score before scale and cap is values[h] exactly: a
    head a value, the query 1 in one element and 0 else.  n > 1: the first query of a prompt of n."""
    heads, dim, page = len(values), 64, 16
    kc = torch.zeros(-(-n // page), page, heads, dim, dtype=dtype)
    kc[0, 0, :, 3] = values.to(dtype)
    q = torch.zeros(n, heads, dim, dtype=dtype)
    q[:, :, 3] = 1
    kc, q = kc.to(DEV), q.to(DEV)
    tables = torch.arange(kc.shape[0], dtype=torch.int32, device=DEV)[None]
    _, lse = ops.paged_attention(q, kc, torch.zeros_like(kc), tables, torch.tensor([n], dtype=torch.int32, device=DEV),
                                 offsets([n]).to(DEV), n, n, return_lse=True, **options)
    return lse[0].cpu().double()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [H, B])
@pytest.mark.parametrize("cap", [1e-3, 0.5, 30.0, 1e3, 1e6, 1e12, 3e38])
@pytest.mark.parametrize("n,tile", [(1, None), (70, 128), (300, 256)])
def test_softcap_of_any_size(plan, n, tile, cap, dtype):
    """The capped score of one key is its lse.  c tanh(s / c): s / c has a relative error of 2 eps, the
    tanh 8 (the hardware's exp2 and reciprocal at s / c = 1/2, its worst place), units of log2 and back
    5: 15 eps of the score; e^0 and its logarithm, whatever factor a sum is held with, some 20 eps."""
    plan(tile=tile)
    scale = 0.75
    s = torch.cat([torch.logspace(-6, 4, 31), -torch.logspace(-6, 4, 31), torch.zeros(1)]).to(dtype)
    got = _one_key(s, dtype, n, softcap=cap, scale=scale)
    c = float(torch.tensor(cap, dtype=torch.float32))
    want = c * torch.tanh(s.double() * scale / c)
    eps = 2.0 ** -24
    assert bool(((got - want).abs() <= (20 * want.abs() + 24) * eps).all()), float((got - want).abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("cap", [1e3, 1e5, 1e7])
@pytest.mark.parametrize("new", [1, 100])
def test_softcap_far_above_the_scores(new, cap):
    _run([400, 123], [new, new], cap=cap, seed=7)
    _run([90, 300], [new, new], heads=1, group=3, dim=80, cap=cap, dtype=H, seed=8)


def _filled(shape, dtype):
    """Leaves memory of 7s to the allocator, where the next tensor of this size is likely to lie."""
    return torch.full(shape, 7, dtype=dtype, device=DEV).data_ptr()


@pytest.mark.gpu
@pytest.mark.parametrize("split", [0, 1])
@pytest.mark.parametrize("most,tile", [(0, None), (1, None), (5, None), (40, 128), (90, 256)])
def test_queries_past_max_q_len_are_empty(plan, most, tile, split):
    """Of more new tokens than max_q_len the first ones are computed, at their places, and the others'
    rows are out 0 and lse -inf."""
    plan(split, 1, tile)
    lens, new, dim = [300, 150, 2, 40], [100, 150, 2, 0], 64
    kc, vc, tables, ks, vs = paged_kv(lens, 16, 2, dim, B, 3)
    q = torch.randn(sum(new) + 3, 4, dim, generator=gen(4)).to(B).to(DEV)
    cu = offsets(new)
    _filled(q.shape, B), _filled(q.shape[:2], torch.float32)
    out, lse = ops.paged_attention(q, kc, vc, tables, torch.tensor(lens, dtype=torch.int32, device=DEV), cu.to(DEV),
                                   most, max(lens), return_lse=True)
    computed = torch.zeros(q.shape[0], dtype=torch.bool)
    for b, n in enumerate(new):
        c0, m = int(cu[b]), min(n, most)
        if m == 0:
            continue
        computed[c0:c0 + m] = True
        out_ref = attention_ref(q[c0:c0 + n].cpu(), ks[b], vs[b], lens[b], n, dim ** -0.5, 0, 0.0)
        check_attention(out[c0:c0 + m], lse[c0:c0 + m], [r[:m] for r in out_ref], dim, lens[b], B)
    assert bool((out.cpu()[~computed] == 0).all()) and bool((lse.cpu()[~computed] == -math.inf).all())


@pytest.mark.gpu
@pytest.mark.parametrize("split", [0, 1])
@pytest.mark.parametrize("new,tile", [(1, None), (7, None), (60, 128), (200, 256)])
def test_nan_scores_have_a_nan_lse(plan, new, tile, split):
    """A query of NaN, and a key of NaN for the queries that see it: out and lse are NaN (-inf is the
    lse of a query that sees no key), and no other row's change."""
    plan(split, 1, tile)
    lens, page, dim = [new + 130], 16, 64
    kc, vc, tables, ks, vs = paged_kv(lens, page, 2, dim, B, 8)
    q = torch.randn(new, 4, dim, generator=gen(9)).to(B)
    args = (torch.tensor(lens, dtype=torch.int32, device=DEV), offsets([new]).to(DEV), new, lens[0])
    ref = attention_ref(q, ks[0], vs[0], lens[0], new, dim ** -0.5, 0, 0.0)

    def check(out, lse, bad):  # bad [new, 4]
        assert torch.equal(lse.cpu().isnan(), bad) and torch.equal(out.cpu().isnan().all(-1), bad)
        fine = ~bad
        check_attention(out.cpu()[fine], lse.cpu()[fine], [r[fine] for r in ref], dim, lens[0], B)

    bad = torch.zeros(new, 4, dtype=torch.bool)
    bad[new // 2, 1] = True
    broken = torch.where(bad[..., None], math.nan, q)
    check(*ops.paged_attention(broken.to(DEV), kc, vc, tables, *args, return_lse=True), bad)
    j = lens[0] - 1 - (new - 1) // 2  # its queries: those from new - 1 - (new - 1) // 2 on
    kc[int(tables[0, j // page]), j % page, 1, 5] = math.nan
    bad = torch.zeros(new, 4, dtype=torch.bool)
    bad[new - 1 - (new - 1) // 2:, 2:] = True
    check(*ops.paged_attention(q.to(DEV), kc, vc, tables, *args, return_lse=True), bad)


@pytest.mark.gpu
@pytest.mark.parametrize("split", [0, 1])
def test_nan_scores_only(plan, split):
    """Every score of a row NaN, in one piece or many."""
    plan(split, 1)
    kc, vc, tables, _, _ = paged_kv([700, 1], 16, 1, 128, H, 8)
    q = torch.full((2, 3, 128), math.nan, dtype=H, device=DEV)
    out, lse = ops.paged_attention(q, kc, vc, tables, torch.tensor([700, 1], dtype=torch.int32, device=DEV),
                                   offsets([1, 1]).to(DEV), 1, 700, return_lse=True)
    assert bool(out.isnan().all()) and bool(lse.isnan().all())


@pytest.mark.gpu
@pytest.mark.parametrize("split", [0, 1])
@pytest.mark.parametrize("window", [0, 21])
@pytest.mark.parametrize("group,tile", [(1, None), (4, None), (40, 128), (70, 256)])
def test_infinite_values_of_the_outermost_keys(plan, group, tile, window, split):
    """The first and the last key that a query sees hold an infinite value: its outputs there are that
    infinity, not NaN (the keys around them in a block take no part)."""
    plan(split, 1, tile)
    length, page, dim = 77, 16, 64
    first = length - window if window else 0
    for j, bad in ((length - 1, math.inf), (first, -math.inf)):
        kc, vc, tables, ks, vs = paged_kv([length], page, 1, dim, B, 8)
        vs[0][j, 0, 9] = bad
        vc[int(tables[0, j // page]), j % page, 0, 9] = bad
        q = torch.randn(1, group, dim, generator=gen(9)).to(B).to(DEV)
        out, lse = ops.paged_attention(q, kc, vc, tables, torch.tensor([length], dtype=torch.int32, device=DEV),
                                       offsets([1]).to(DEV), 1, length, window=window, return_lse=True)
        ref = attention_ref(q.cpu(), ks[0], vs[0], length, 1, dim ** -0.5, window, 0.0)
        check_attention(out, lse, ref, dim, length, B)
        assert bool((out[:, :, 9] == bad).all())


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["softcap", "scale"])
def test_refuses_what_32_bits_cannot_hold(name):
    with pytest.raises(RuntimeError, match=name):
        ops.paged_attention(**dict(_good(), **{name: 1e39}))


def test_c_entry_refuses_infinite_factors():
    lib = pulsar_amd.capi()
    lib.pw4_paged_attention.argtypes = [ctypes.POINTER(_Args), ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p]
    for change in (dict(softcap=math.inf), dict(scale=math.inf), dict(scale=-math.inf)):
        a = dict(num_tokens=0, q_heads=4, kv_heads=2, head_dim=64, page_size=16, scale=1.0, dtype=1)
        assert lib.pw4_paged_attention(ctypes.byref(_Args(**a)), None, 0, None) == 0
        assert lib.pw4_paged_attention(ctypes.byref(_Args(**dict(a, **change))), None, 0, None) == -1


def _workspace(**change):
    lib = pulsar_amd.capi()
    lib.pw4_paged_attention_workspace_size.argtypes = [ctypes.POINTER(_Args)]
    lib.pw4_paged_attention_workspace_size.restype = ctypes.c_size_t
    a = dict(q=4096, k_cache=4096, v_cache=4096, block_tables=4096, seq_lens=4096, cu_q=4096, out=4096, num_tokens=8,
             batch=8, q_heads=32, kv_heads=8, head_dim=128, num_pages=4, page_size=16, table_width=2048,
             table_stride=2048, q_token_stride=4096, q_head_stride=128, page_stride=16384, row_stride=1024,
             kv_head_stride=128, max_q_len=1, max_seq_len=32768, scale=1.0, dtype=1)
    a.update(change)
    return lib.pw4_paged_attention_workspace_size(ctypes.byref(_Args(**a)))


def test_the_split_goes_by_the_keys_that_a_window_leaves():
    """Workspace is asked for where the keys are split over workgroups: a tile sees `window` keys and
    its rows' spread, however long its sequence is."""
    chunks = dict(batch=2, num_tokens=200, max_q_len=100)
    for case in ({}, chunks, dict(chunks, kv_heads=2, q_heads=14, head_dim=64)):
        long = _workspace(**case)
        assert long > 0
        for window in (1, 128, 600):
            short = _workspace(**case, window=window)
            assert short == _workspace(**dict(case, max_seq_len=window + 150), window=window) == 0
        for window in (32768, 2 ** 31 - 1):
            assert _workspace(**case, window=window) == long
    assert _workspace(window=30000) > 0


@pytest.mark.gpu
@pytest.mark.parametrize("split", [None, 1])
@pytest.mark.parametrize("window", [1, 31, 128, 1000])
def test_windows_in_long_sequences(plan, window, split):
    """The newest tokens of long sequences, of which a window is seen: few rows, 128 and 256 rows."""
    plan(split, 1 if split else None)
    lens = [9001, 8000, 131]
    _run(lens, [1, 2, 3], heads=2, group=4, window=window, seed=window)
    _run(lens, [40, 1, 131], heads=1, group=3, dim=64, dtype=H, window=window, seed=window)
    plan(split, 1 if split else None, 256)
    _run(lens, [300, 77, 131], heads=1, group=2, dim=128, window=window, seed=window)


@pytest.mark.gpu
def test_one_element_views():
    """The stride of a dimension of one counts for nothing."""
    args = _good()
    want = ops.paged_attention(**args)
    got = ops.paged_attention(**dict(args, seq_lens=args["seq_lens"].repeat(2)[::2],
                                     block_tables=args["block_tables"].repeat(2, 1)[::2]))
    assert torch.equal(got, want)
    one = _good()
    one.update(seq_lens=torch.tensor([3], dtype=torch.int32, device=DEV))
    want = ops.paged_attention(**one)
    got = ops.paged_attention(**dict(one, block_tables=one["block_tables"].repeat_interleave(4, 1)[:, :4:4]))
    assert torch.equal(got, want)
    # caches of one page, whose strides between pages differ
    one.update(k_cache=one["k_cache"][:1], v_cache=one["v_cache"][:1], block_tables=one["block_tables"][:, :1] * 0)
    one["v_cache"] = one["v_cache"].as_strided(one["v_cache"].shape, (8, *one["v_cache"].stride()[1:]))
    assert ops.paged_attention(**one).shape == one["q"].shape


@pytest.mark.gpu
@pytest.mark.parametrize("name", [-1, 10 ** 9, -2 ** 31])
@pytest.mark.parametrize("new", [1, 40])
def test_page_ids_outside_the_pool_read_its_last_page(new, name):
    lens, page = [130], 16
    kc, vc, tables, _, _ = paged_kv(lens, page, 2, 64, B, 5, junk=1.0)
    q = torch.randn(new, 4, 64, generator=gen(6)).to(B).to(DEV)
    args = (torch.tensor(lens, dtype=torch.int32, device=DEV), offsets([new]).to(DEV), new, lens[0])
    got = []
    for page_id in (name, kc.shape[0] - 1):
        tables[0, 2] = page_id
        got.append(ops.paged_attention(q, kc, vc, tables, *args))
    assert torch.equal(*got)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [H, B])
@pytest.mark.parametrize("split", [0, 1])
def test_lse_of_two_keys(plan, dtype, split):
    """Scores below 2 that the products give exactly, two keys a query.  Each rounding of the lse as an
    even one: the exponents' arguments (fp16's are near 6, spaced 2^-21) 9.5e-8, exp2 7e-8, log2 of a
    sum below 2 4e-8, the maximum's sum with it 5e-8, the lse's own 7e-8: 1.5e-7 in the mean square."""
    plan(split, 1)
    heads, dim = 2048, 64
    s = (torch.rand(2, heads, generator=gen(3)) * 4 - 2).to(dtype)
    kc = torch.zeros(1, 16, heads, dim, dtype=dtype)
    kc[0, :2, :, 7] = s
    q = torch.zeros(1, heads, dim, dtype=dtype)
    q[:, :, 7] = 1
    kc, q = kc.to(DEV), q.to(DEV)
    _, lse = ops.paged_attention(q, kc, torch.zeros_like(kc), torch.zeros(1, 1, dtype=torch.int32, device=DEV),
                                 torch.tensor([2], dtype=torch.int32, device=DEV), offsets([1]).to(DEV), 1, 2,
                                 scale=1.0, return_lse=True)
    err = lse[0].cpu().double() - torch.logsumexp(s.double(), 0)
    assert float(err.square().mean().sqrt()) <= 1.5e-7 and float(err.abs().max()) <= 1e-6


def test_c_entry_refuses_more_rows_than_it_counts():
    lib = pulsar_amd.capi()
    lib.pw4_paged_attention.argtypes = [ctypes.POINTER(_Args), ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p]

    def call(tokens, most):  # refused before any launch: for the rows (-2), or else for want of memory for q (-1)
        a = dict(num_tokens=tokens, max_q_len=most, q_heads=8192, kv_heads=1, head_dim=8, page_size=16, scale=1.0, dtype=1)
        return lib.pw4_paged_attention(ctypes.byref(_Args(**a)), None, 0, None)

    assert call(2 ** 18, 2 ** 18) == -2 and call(2 ** 20, 2 ** 18) == -2
    assert call(2 ** 18, 2 ** 17) == -1 and call(2 ** 17, 2 ** 30) == -1


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 100])
def test_no_sequences_and_a_far_bound(new):
    """Nothing to split, whatever max_seq_len is."""
    kc = torch.zeros(40, 16, 2, 64, dtype=B, device=DEV)
    none = torch.zeros(0, 9000, dtype=torch.int32, device=DEV)
    q = torch.ones(new, 4, 64, dtype=B, device=DEV)
    out, lse = ops.paged_attention(q, kc, kc, none, none[:, 0].contiguous(), offsets([]).to(DEV), new, 9000 * 16,
                                   return_lse=True)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())


@pytest.mark.gpu
@pytest.mark.parametrize("split", [0, 1])
@pytest.mark.parametrize("tile,new", [(None, 1), (None, 7), (128, 40), (256, 150)])
@pytest.mark.parametrize("dim", [64, 96, 256])
def test_writes_stay_in_the_outputs_and_the_workspace(plan, dim, tile, new, split):
    """The C entry on buffers with a margin behind each."""
    plan(split, 1, tile)
    lens, group, heads = [900, 333, new, 61], 4, 2
    counts = [new, min(new, 40), new, 0]
    kc, vc, tables, _, _ = paged_kv(lens, 16, heads, dim, B, 3)
    q = torch.randn(sum(counts) + 1, heads * group, dim, generator=gen(4)).to(B).to(DEV)
    lens_t, cu = torch.tensor(lens, dtype=torch.int32, device=DEV), offsets(counts).to(DEV)
    want = ops.paged_attention(q, kc, vc, tables, lens_t, cu, new, 900, return_lse=True)
    out = torch.full((q.numel() + 64,), 3.0, dtype=B, device=DEV)
    lse = torch.full((q.shape[0] * q.shape[1] + 64,), 3.0, device=DEV)
    a = _Args(q=q.data_ptr(), k_cache=kc.data_ptr(), v_cache=vc.data_ptr(), block_tables=tables.data_ptr(),
              seq_lens=lens_t.data_ptr(), cu_q=cu.data_ptr(), out=out.data_ptr(), lse=lse.data_ptr(),
              num_tokens=q.shape[0], batch=4, q_heads=heads * group, kv_heads=heads, head_dim=dim,
              num_pages=kc.shape[0], page_size=16, table_width=tables.shape[1], table_stride=tables.stride(0),
              q_token_stride=q.stride(0), q_head_stride=q.stride(1), page_stride=kc.stride(0), row_stride=kc.stride(1),
              kv_head_stride=kc.stride(2), max_q_len=new, max_seq_len=900, scale=dim ** -0.5, dtype=1)
    lib = pulsar_amd.capi()
    lib.pw4_paged_attention.argtypes = [ctypes.POINTER(_Args), ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p]
    lib.pw4_paged_attention_workspace_size.argtypes = [ctypes.POINTER(_Args)]
    lib.pw4_paged_attention_workspace_size.restype = ctypes.c_size_t
    size = lib.pw4_paged_attention_workspace_size(ctypes.byref(a))
    assert (size > 0) == bool(split)
    ws = torch.full((size + 256,), 0x5a, dtype=torch.uint8, device=DEV)
    torch.cuda.synchronize()
    assert lib.pw4_paged_attention(ctypes.byref(a), ws.data_ptr(), size, None) == 0
    torch.cuda.synchronize()
    assert torch.equal(out[:q.numel()].view(q.shape), want[0]) and torch.equal(lse[:-64].view(want[1].shape), want[1])
    assert bool((out[q.numel():] == 3).all()) and bool((lse[-64:] == 3).all()) and bool((ws[size:] == 0x5a).all())
