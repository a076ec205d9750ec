"""paged_cache_append, paged_cache_append_fp4 and paged_cache_read_fp4 against their definitions.

A rotated element a c - b s is two exact products in fp64, summed there (2^-53 of the larger) and
rounded to fp32 (2^-24 of it) and to 16 bits (half a step of those, u = eps / 2): bound u |x| + 2^-23 of
|a c| + |b s|, and half the least subnormal of fp16.  In 4 bits the same element goes to a block: the codes
are equal to those of the 64-bit value but where that stands within 2^-22 of a border, which the tests'
inputs do not (they are checked for it)."""

import ctypes
import math

import pytest
import torch

import pulsar_amd
from fp4_case import fp4_round, new_pool, row_bytes, to_dev
from paged_case import DEV, gen
from pulsar_amd import ops

H, B = torch.float16, torch.bfloat16


def rotate_ref(x, rope, positions, interleaved):
    """x [T, heads, dim] rotated in 64 bits, and |a c| + |b s|, on the host."""
    x, rot = x.double().clone(), rope.shape[1]
    size = x.abs()
    half = rot // 2
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, half + i)
        c, s = rope[positions, i].double()[:, None], rope[positions, half + i].double()[:, None]
        xa, xb = x[..., a].clone(), x[..., b].clone()
        x[..., a], x[..., b] = xa * c - xb * s, xb * c + xa * s
        size[..., a] = (xa * c).abs() + (xb * s).abs()
        size[..., b] = (xb * c).abs() + (xa * s).abs()
    return x, size


def check16(got, want, size, dtype):
    u = torch.finfo(dtype).eps / 2
    bound = u * want.abs() + 1.01 * 2.0 ** -23 * size + (2.0 ** -25 if dtype == H else 0.0)
    assert bool(((got.cpu().double() - want).abs() <= bound).all())


def _case(t, hq, hkv, dim, rot, dtype, seed, most=5000):
    g = gen(seed)
    q, k, v = (torch.randn(t, h, dim, generator=g).to(dtype) for h in (hq, hkv, hkv))
    positions = torch.randint(0, most, (t,), generator=g)
    return q, k, v, positions, ops.rope_table(most, rot, 500000.0, device="cpu")


SHAPES = [  # tokens, q heads, kv heads, dim, rot
    (1, 32, 8, 128, 128), (7, 4, 1, 64, 64), (33, 14, 2, 64, 32), (5, 8, 8, 96, 96), (3, 3, 3, 256, 64),
    (200, 2, 1, 128, 128), (9, 7, 1, 192, 192), (4, 5, 5, 160, 160), (6, 1, 1, 32, 2), (2, 71, 1, 224, 56),
    (3000, 1, 1, 32, 32)]
SHAPES16 = SHAPES + [(5, 4, 2, 80, 80), (5, 4, 2, 80, 40), (4, 3, 1, 8, 8), (6, 2, 2, 40, 12), (3, 2, 1, 136, 136)]


def test_rope_table():
    t = ops.rope_table(200000, 6, 10000.0, device="cpu")
    assert t.shape == (200000, 6) and t.dtype == torch.float32
    p = torch.tensor([0.0, 1.0, 199999.0], dtype=torch.float64)
    for i in range(3):
        angle = p * 10000.0 ** (-2 * i / 6)
        want = torch.stack([angle.cos(), angle.sin()], 1)
        assert float((t[p.long()][:, [i, 3 + i]].double() - want).abs().max()) <= 2.0 ** -24 + 1e-10


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [H, B])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("t,hq,hkv,dim,rot", SHAPES16)
def test_append_16_bits(t, hq, hkv, dim, rot, interleaved, dtype):
    page, pages = 16, -(-t // 16) + 3
    q, k, v, positions, rope = _case(t, hq, hkv, dim, rot, dtype, t + dim)
    slots = torch.randperm(pages * page, generator=gen(1))[:t]
    slots[t // 2] = -1 if t > 1 else slots[t // 2]
    pool = torch.full((2, pages, page, hkv, dim), 3.0, dtype=dtype, device=DEV)
    out = ops.paged_cache_append(q.to(DEV), k.to(DEV), v.to(DEV), pool[0], pool[1], slots.to(DEV), rope.to(DEV),
                                 positions.to(DEV), interleaved)
    assert out.shape == q.shape and out.dtype == dtype
    check16(out, *rotate_ref(q, rope, positions, interleaved), dtype)
    there = slots >= 0
    flat = pool.cpu().view(2, -1, hkv, dim)
    want, size = rotate_ref(k, rope, positions, interleaved)
    check16(flat[0, slots[there]], want[there], size[there], dtype)
    assert torch.equal(flat[1, slots[there]], v[there])
    rest = torch.ones(pages * page, dtype=torch.bool)
    rest[slots[there]] = False
    assert bool((flat[:, rest] == 3).all())
    # keys and values alone are the same bits
    again = torch.full_like(pool, 3.0)
    assert ops.paged_cache_append(None, k.to(DEV), v.to(DEV), again[0], again[1], slots.to(DEV), rope.to(DEV),
                                  positions.to(DEV), interleaved) is None
    assert torch.equal(again, pool)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [H, B])
@pytest.mark.parametrize("t,hq,hkv,dim,rot", SHAPES)
def test_append_4_bits(t, hq, hkv, dim, rot, dtype):
    page, pages = 24, -(-t // 24) + 2
    q, k, v, positions, rope = _case(t, hq, hkv, dim, rot, dtype, t + dim)
    slots = torch.randperm(pages * page, generator=gen(1))[:t]
    if t > 1:
        slots[t // 2], slots[0] = -1, pages * page  # outside either way
    for interleaved in (False, True):
        pool = to_dev(new_pool(2, pages, page, hkv, dim, pad=1, fill=0xA5))
        before = pool.cpu()
        args = (slots.to(DEV), rope.to(DEV), positions.to(DEV), interleaved)
        out = ops.paged_cache_append_fp4(q.to(DEV), k.to(DEV), v.to(DEV), pool[0], pool[1], *args)
        check16(out, *rotate_ref(q, rope, positions, interleaved), dtype)
        there = (slots >= 0) & (slots < pages * page)
        after, host = pool.cpu(), before.clone()
        for plane, x in ((0, rotate_ref(k, rope, positions, interleaved)[0]), (1, v.double())):
            x = x.float()
            codes, exps, values = fp4_round(x, dtype == H)
            got = ops.paged_cache_read_fp4(pool[0], pool[1], slots.to(DEV), dtype)[plane].cpu()
            assert torch.equal(got[there].double(), values[there]) and bool((got[~there] == 0).all())
            for i in torch.nonzero(there)[:, 0].tolist():  # the bytes, where the layout puts them
                p, r = divmod(int(slots[i]), page)
                flat = host[plane, p].reshape(-1)
                for h in range(hkv):
                    at = (h * page + r) * (dim // 2)
                    flat[at:at + dim // 2] = (codes[i, h, 0::2] + 16 * codes[i, h, 1::2]).to(torch.uint8)
                    at = hkv * page * (dim // 2) + (h * page + r) * (dim // 32)
                    flat[at:at + dim // 32] = exps[i, h].to(torch.uint8)
                host[plane, p] = flat.view(page, hkv, -1)
                if t > 300 and i > 300:
                    break
        if t <= 300:
            assert torch.equal(after, host)
        # the pages' padding is left alone
        whole = pool.as_strided((2, pages, 16), (pool.stride(0), pool.stride(1), 1), pool.stride(1) - 16)
        assert bool((whole == 0xA5).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [H, B])
def test_blocks_of_every_kind(dtype):
    """Borders between codes, magnitudes from the least to the greatest, zeros, NaN and infinities."""
    dim, page = 64, 16
    rows = []
    grid = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0] * 4)
    for e in ((-24, -14, -3, 0, 5, 12) if dtype == H else (-133, -126, -60, 0, 60, 124)):
        rows.append(torch.ldexp(grid, torch.tensor(e)))
        rows.append(torch.ldexp(grid * torch.where(torch.arange(32) % 3 == 0, -1.0, 1.0), torch.tensor(e)))
    for top in (3.5, 6.9375, 7.0, 7.5):
        rows.append(torch.linspace(-top, top, 32))
    rows += [torch.zeros(32), -torch.zeros(32), torch.full((32,), torch.finfo(dtype).max),
             torch.full((32,), torch.finfo(dtype).tiny), torch.full((32,), torch.finfo(dtype).smallest_normal / 4)]
    for bad in (math.nan, math.inf, -math.inf):
        rows.append(torch.where(torch.arange(32) == 7, bad, torch.randn(32, generator=gen(1))))
    if len(rows) % 2:
        rows.append(torch.ones(32))
    x = torch.stack(rows).to(dtype).view(-1, 1, dim)
    t = x.shape[0]
    pool = to_dev(new_pool(2, -(-t // page), page, 1, dim))
    slots = torch.arange(t, device=DEV)
    ops.paged_cache_append_fp4(None, x.to(DEV), x.flip(0).to(DEV), pool[0], pool[1], slots)
    want = fp4_round(x, dtype == H)[2]
    k, v = ops.paged_cache_read_fp4(pool[0], pool[1], slots, dtype)
    assert torch.equal(k.cpu().double().nan_to_num(9e9), want.to(dtype).double().nan_to_num(9e9))
    assert torch.equal(v.cpu().double().nan_to_num(9e9), want.to(dtype).double().flip(0).nan_to_num(9e9))
    assert torch.equal(torch.signbit(k.cpu())[~want.isnan()], torch.signbit(want)[~want.isnan()])


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 16])
def test_layouts_strides_and_odd_addresses(bits):
    """Slices of a fused projection, other orders, rows that no vector load can take, caches in other layouts."""
    t, hq, hkv, dim, page = 20, 6, 2, 64, 8
    q, k, v, positions, rope = _case(t, hq, hkv, dim, dim, B, 3)
    slots = torch.randperm(64, generator=gen(1))[:t]
    op = ops.paged_cache_append if bits == 16 else ops.paged_cache_append_fp4

    def run(q, k, v, pool):
        out = op(q, k, v, pool[0], pool[1], slots.to(DEV), rope.to(DEV), positions.to(DEV))
        return out.cpu(), pool.cpu()

    def pool():
        if bits == 16:
            return torch.zeros(2, 8, page, hkv, dim, dtype=B, device=DEV)
        return to_dev(new_pool(2, 8, page, hkv, dim, fill=0))

    want = run(q.to(DEV), k.to(DEV), v.to(DEV), pool())
    for shift in (0, 1):
        fused = torch.zeros(t, (hq + 2 * hkv) * dim + 8, dtype=B, device=DEV)[:, shift:shift + (hq + 2 * hkv) * dim]
        fused.copy_(torch.cat([x.flatten(1) for x in (q, k, v)], 1))
        parts = [p.unflatten(1, (-1, dim)) for p in fused.split((hq * dim, hkv * dim, hkv * dim), 1)]
        for a, b in zip(want, run(*parts, pool())):
            assert torch.equal(a, b)
    heads_first = [x.transpose(0, 1).contiguous().to(DEV).transpose(0, 1) for x in (q, k, v)]
    dims_first = [x.transpose(1, 2).contiguous().to(DEV).transpose(1, 2) for x in (q, k, v)]
    for parts in (heads_first, dims_first):
        for a, b in zip(want, run(*parts, pool())):
            assert torch.equal(a, b)
    if bits == 16:
        hnd = torch.zeros(2, 8, hkv, page, dim, dtype=B, device=DEV).transpose(2, 3)
        odd = torch.zeros(2 * 8 * page * hkv * dim + 1, dtype=B, device=DEV)[1:].view(2, 8, page, hkv, dim)
        for p in (hnd, odd):
            for a, b in zip(want, run(q.to(DEV), k.to(DEV), v.to(DEV), p)):
                assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 16])
def test_positions_outside_the_table(bits):
    """Such a token is not stored, and its query is 0; the others are as ever.  A table of no rows knows none."""
    t, dim, page = 6, 64, 8
    q, k, v, positions, rope = _case(t, 2, 1, dim, dim, B, 5, most=50)
    op = ops.paged_cache_append if bits == 16 else ops.paged_cache_append_fp4
    fresh = (lambda: torch.zeros(2, 2, page, 1, dim, dtype=B, device=DEV)) if bits == 16 else (
        lambda: to_dev(new_pool(2, 2, page, 1, dim, fill=0)))
    slots = torch.arange(t, device=DEV)
    want = fresh()
    good = op(q.to(DEV), k.to(DEV), v.to(DEV), want[0], want[1], slots, rope.to(DEV), positions.to(DEV))
    wrong = positions.clone()
    wrong[1], wrong[3], wrong[4] = -1, 50, 2 ** 40
    got = fresh()
    out = op(q.to(DEV), k.to(DEV), v.to(DEV), got[0], got[1], slots, rope.to(DEV), wrong.to(DEV))
    bad = torch.tensor([1, 3, 4])
    fine = torch.tensor([0, 2, 5])
    assert bool((out[bad] == 0).all()) and torch.equal(out[fine], good[fine])
    part = fresh()
    op(q.to(DEV), k.to(DEV), v.to(DEV), part[0], part[1], torch.where(torch.isin(slots, bad.to(DEV)), -1, slots),
       rope.to(DEV), positions.to(DEV))
    assert torch.equal(got, part)
    none = fresh()
    out = op(q.to(DEV), k.to(DEV), v.to(DEV), none[0], none[1], slots, rope[:0].to(DEV), positions.to(DEV))
    assert bool((out == 0).all()) and not bool(none.any())
    # nothing to rotate by: queries and keys pass
    same = fresh()
    out = op(q.to(DEV), k.to(DEV), v.to(DEV), same[0], same[1], slots, rope[:, :0].to(DEV).contiguous(), positions.to(DEV))
    assert torch.equal(out.cpu(), q)


@pytest.mark.gpu
def test_writes_past_32_bits():
    page, heads, dim = 64, 8, 128
    for bits in (16, 4):
        row = 2 * dim if bits == 16 else row_bytes(dim)
        pages = 2 ** 32 // (page * heads * row) + 64
        k, v = (torch.randn(3, heads, dim, generator=gen(i)).to(B).to(DEV) for i in (1, 2))
        slots = torch.tensor([pages * page - 1, 5, (pages - 10) * page], device=DEV)
        if bits == 16:
            pool = torch.zeros(2, pages, page, heads, dim, dtype=B, device=DEV)
            ops.paged_cache_append(None, k, v, pool[0], pool[1], slots)
            flat = pool.view(2, -1, heads, dim)
            assert torch.equal(flat[0, slots], k) and torch.equal(flat[1, slots], v)
        else:
            pool = torch.zeros(2, pages, page, heads, row, dtype=torch.uint8, device=DEV)
            ops.paged_cache_append_fp4(None, k, v, pool[0], pool[1], slots)
            got = ops.paged_cache_read_fp4(pool[0], pool[1], slots, B)
            for a, b in zip(got, (k, v)):
                assert torch.equal(a.cpu().double(), fp4_round(b.cpu())[2])
        assert int((pool.view(2, pages, -1)[:, :, :64] != 0).any(-1).sum()) <= 6
        del pool


@pytest.mark.gpu
def test_nothing_to_do():
    pool = torch.zeros(2, 4, 8, 2, 64, dtype=B, device=DEV)
    none = torch.zeros(0, 2, 64, dtype=B, device=DEV)
    slots = torch.zeros(0, dtype=torch.int64, device=DEV)
    rope = ops.rope_table(8, 64)
    assert ops.paged_cache_append(none, none, none, pool[0], pool[1], slots, rope, slots).shape == (0, 2, 64)
    fp4 = to_dev(new_pool(2, 4, 8, 2, 64))
    assert ops.paged_cache_append_fp4(none, none, none, fp4[0], fp4[1], slots, rope, slots).shape == (0, 2, 64)
    assert [x.shape for x in ops.paged_cache_read_fp4(fp4[0], fp4[1], slots, H)] == [(0, 2, 64)] * 2
    # a pool without pages takes nothing
    one = torch.ones(1, 2, 64, dtype=B, device=DEV)
    ops.paged_cache_append(None, one, one, pool[0, :0], pool[1, :0], torch.zeros(1, dtype=torch.int64, device=DEV))
    got = ops.paged_cache_read_fp4(fp4[0, :0], fp4[1, :0], torch.zeros(1, dtype=torch.int64, device=DEV), B)
    assert not bool(got[0].any())


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 16])
def test_streams_and_graphs(bits):
    """The same bits on another stream and in a graph's replays, which follow slots that change on the device."""
    t, dim, page = 40, 128, 16
    q, k, v, positions, rope = (x.to(DEV) for x in _case(t, 4, 2, dim, dim, B, 7))
    op = ops.paged_cache_append if bits == 16 else ops.paged_cache_append_fp4
    pool = torch.zeros(2, 8, page, 2, dim, dtype=B, device=DEV) if bits == 16 else to_dev(new_pool(2, 8, page, 2, dim, fill=0))
    slots = torch.randperm(128, generator=gen(1))[:t].to(DEV)

    def call():
        return op(q, k, v, pool[0], pool[1], slots, rope, positions)

    first = call()
    want = pool.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        pool.zero_()
        other = call()
        graph = torch.cuda.CUDAGraph()
    side.synchronize()
    assert torch.equal(pool, want) and torch.equal(first, other)
    with torch.cuda.graph(graph, stream=side):
        captured = call()
    for _ in range(3):
        pool.zero_()
        captured.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(pool, want) and torch.equal(captured, first)
        slots.copy_(slots.flip(0).clone())
        pool.zero_()
        call()
        want = pool.clone()


def _good(bits):
    pool = torch.zeros(2, 4, 8, 2, 64, dtype=B, device=DEV) if bits == 16 else to_dev(new_pool(2, 4, 8, 2, 64, fill=0))
    x = torch.zeros(3, 2, 64, dtype=B, device=DEV)
    return dict(q=torch.zeros(3, 4, 64, dtype=B, device=DEV), k=x, v=x.clone(), k_cache=pool[0], v_cache=pool[1],
                slots=torch.arange(3, device=DEV), rope=ops.rope_table(9, 64), positions=torch.arange(3, device=DEV))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("change,message", [
    (lambda a: dict(q=a["q"].half()), "one dtype"),
    (lambda a: dict(k=a["k"].float(), v=a["v"].float()), "fp16 or bf16"),
    (lambda a: dict(v=a["v"][:, :1]), "3-D"),
    (lambda a: dict(k=a["k"][:, :1], v=a["v"][:, :1]), "kv_heads"),
    (lambda a: dict(k=a["k"][..., :32], v=a["v"][..., :32]), "head_dim"),
    (lambda a: dict(q=a["q"][:2]), "q must be"),
    (lambda a: dict(q=a["q"].cpu()), "one CUDA device"),
    (lambda a: dict(slots=a["slots"].int()), "int64"),
    (lambda a: dict(slots=a["slots"][:2]), "slots must be"),
    (lambda a: dict(positions=a["positions"][:2]), "positions must be"),
    (lambda a: dict(positions=a["positions"].int()), "int64"),
    (lambda a: dict(positions=None), "together"),
    (lambda a: dict(rope=None), "together"),
    (lambda a: dict(rope=None, positions=None), "needs rope"),
    (lambda a: dict(rope=a["rope"].double()), "fp32"),
    (lambda a: dict(rope=a["rope"][:, ::2]), "contiguous"),
    (lambda a: dict(rope=a["rope"][:, :63].contiguous()), "even"),
    (lambda a: dict(rope=torch.zeros(9, 66, device=DEV)), "even|head_dim"),
    (lambda a: dict(v_cache=a["v_cache"][:-1]), "one shape"),
    (lambda a: dict(k_cache=a["k_cache"].float(), v_cache=a["v_cache"].float()), "one dtype|uint8"),
])
def test_refusals(bits, change, message):
    op = ops.paged_cache_append if bits == 16 else ops.paged_cache_append_fp4
    args = _good(bits)
    op(**args)
    args.update(change(args))
    with pytest.raises(RuntimeError, match=message):
        op(**args)


@pytest.mark.gpu
def test_read_refusals():
    a = _good(4)
    args = (a["k_cache"], a["v_cache"], a["slots"])
    with pytest.raises(RuntimeError, match="fp16 or bf16"):
        ops.paged_cache_read_fp4(*args, torch.float32)
    with pytest.raises(RuntimeError, match="int64"):
        ops.paged_cache_read_fp4(*args[:2], a["slots"].int(), B)
    with pytest.raises(RuntimeError, match="uint8"):
        ops.paged_cache_read_fp4(a["k"][None], a["v"][None], a["slots"], B)


class _Args(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in ("q", "k", "v", "q_out", "k_cache", "v_cache", "slots", "positions", "rope")]
                + [(n, ctypes.c_int64) for n in (
                    "num_tokens", "q_heads", "kv_heads", "head_dim", "rot", "rope_rows", "q_token_stride", "q_head_stride",
                    "k_token_stride", "k_head_stride", "v_token_stride", "v_head_stride", "num_pages", "page_size",
                    "page_stride", "row_stride", "kv_head_stride")]
                + [("interleaved", ctypes.c_int), ("dtype", ctypes.c_int)])


def test_c_entries_refuse_before_any_launch():
    lib = pulsar_amd.capi()
    for f in (lib.pw4_paged_cache_append, lib.pw4_paged_cache_append_fp4):
        f.argtypes = [ctypes.POINTER(_Args), ctypes.c_void_p]
        fp4 = f is lib.pw4_paged_cache_append_fp4
        good = dict(q=4096, k=4096, v=4096, q_out=4096, k_cache=4096, v_cache=4096, slots=4096, positions=4096, rope=4096,
                    num_tokens=1, q_heads=4, kv_heads=2, head_dim=64, rot=64, rope_rows=9, q_token_stride=256,
                    q_head_stride=64, k_token_stride=128, k_head_stride=64, v_token_stride=128, v_head_stride=64,
                    num_pages=4, page_size=16, page_stride=16 * 2 * 34 if fp4 else 2048, row_stride=128, kv_head_stride=64,
                    dtype=1)

        def call(**change):
            return f(ctypes.byref(_Args(**dict(good, **change))), None)

        assert f(None, None) == -1
        assert call(dtype=2) == -1 and call(num_tokens=-1) == -1 and call(page_size=0) == -1 and call(head_dim=0) == -1
        assert call(head_dim=60) == -2 and call(head_dim=264) == -2 and call(rot=63) == -2 and call(rot=66) == -2
        assert call(num_pages=2 ** 31) == -2 and call(num_pages=2 ** 28) == -2 and call(rope_rows=2 ** 31) == -2
        assert call(k=None) == -1 and call(slots=None) == -1 and call(v_cache=None) == -1 and call(q_out=None) == -1
        assert call(rope=None) == -1 and call(positions=None) == -1 and call(positions=None, rope=None) == -1
        assert call(k=4097) == -1 and call(q_out=4104) == -1 and call(rope=4098) == -1
        assert call(num_tokens=0, k=None, v=None) == 0
        if fp4:
            assert call(head_dim=40, rot=40) == -2 and call(k_cache=4104) == -1
            assert call(page_stride=16 * 2 * 34 - 16) == -2 and call(page_stride=16 * 2 * 34 + 8) == -1
            assert call(page_size=2 ** 24, num_pages=1) == -2
    r = lib.pw4_paged_cache_read_fp4
    r.argtypes = [ctypes.c_void_p] * 5 + [ctypes.c_int64] * 6 + [ctypes.c_int, ctypes.c_void_p]

    def read(k_cache=4096, slots=4096, out=4096, t=1, heads=2, dim=64, pages=4, page=16, stride=16 * 2 * 34, dtype=1):
        return r(k_cache, 4096, slots, out, 4096, t, heads, dim, pages, page, stride, dtype, None)

    assert read(dtype=2) == -1 and read(t=-1) == -1 and read(dim=48) == -2 and read(dim=288) == -2 and read(page=0) == -1
    assert read(k_cache=None) == -1 and read(slots=None) == -1 and read(out=4104) == -1 and read(stride=40) == -1
    assert read(stride=16) == -2 and read(pages=2 ** 28) == -2 and read(t=0, slots=None) == 0


def test_fake_kernels():
    q, k = torch.empty(5, 8, 64, dtype=B, device="meta"), torch.empty(5, 2, 64, dtype=B, device="meta")
    i = torch.empty(5, dtype=torch.int64, device="meta")
    rope = torch.empty(9, 64, device="meta")
    c16, c4 = torch.empty(4, 16, 2, 64, dtype=B, device="meta"), torch.empty(4, 16, 2, 34, dtype=torch.uint8, device="meta")
    for op, c in ((ops.paged_cache_append, c16), (ops.paged_cache_append_fp4, c4)):
        assert op(q, k, k, c, c, i, rope, i).shape == q.shape
        assert op(None, k, k, c, c, i) is None
    assert [x.shape for x in ops.paged_cache_read_fp4(c4, c4, i, H)] == [(5, 2, 64)] * 2


@pytest.mark.gpu
def test_opcheck():
    utils = ("test_schema", "test_faketensor", "test_aot_dispatch_dynamic")
    torch.library.opcheck(torch.ops.pulsar.paged_cache_append.default, tuple(_good(16).values()), test_utils=utils)
    torch.library.opcheck(torch.ops.pulsar.paged_cache_append_fp4.default, tuple(_good(4).values()), test_utils=utils)
    a = _good(4)
    torch.library.opcheck(torch.ops.pulsar.paged_cache_read_fp4.default, (a["k_cache"], a["v_cache"], a["slots"], B),
                          test_utils=utils)


@pytest.mark.gpu
@pytest.mark.parametrize("dim,rot", [(32, 16), (64, 16), (64, 48), (96, 48), (128, 16), (128, 112), (160, 144), (176, 80),
                                     (224, 96), (256, 208)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotations_that_end_inside_blocks(dim, rot, interleaved):
    """Vectors of a block of 32 stand with their mates, or where the head has them: the block's exponent is of both."""
    t, page = 37, 20
    q, k, v, positions, rope = _case(t, 5, 3, dim, rot, B, dim + rot)
    k = (k * torch.exp2(torch.randint(-6, 7, k.shape, generator=gen(3)).float())).to(B)  # blocks that differ
    slots = torch.randperm(3 * page, generator=gen(1))[:t]
    args = (slots.to(DEV), rope.to(DEV), positions.to(DEV), interleaved)
    want, size = rotate_ref(k, rope, positions, interleaved)
    pool = torch.zeros(2, 3, page, 3, dim, dtype=B, device=DEV)
    check16(ops.paged_cache_append(q.to(DEV), k.to(DEV), v.to(DEV), pool[0], pool[1], *args),
            *rotate_ref(q, rope, positions, interleaved), B)
    check16(pool[0].view(-1, 3, dim)[slots.to(DEV)], want, size, B)
    if dim % 32:
        return
    four = to_dev(new_pool(2, 3, page, 3, dim))
    ops.paged_cache_append_fp4(None, k.to(DEV), v.to(DEV), four[0], four[1], *args)
    got = ops.paged_cache_read_fp4(four[0], four[1], slots.to(DEV), B)
    assert torch.equal(got[0].cpu().double(), fp4_round(want.float())[2])
    assert torch.equal(got[1].cpu().double(), fp4_round(v)[2])


@pytest.mark.gpu
def test_more_tokens_than_a_launch_has_workgroups():
    """2^24 workgroups of 256 threads are more than one launch may have."""
    t, page = (1 << 24) + 3, 64
    pages = -(-t // page)
    slots = torch.arange(t, device=DEV).flip(0)
    k = torch.arange(t, device=DEV).remainder(2039).half()[:, None, None].expand(t, 1, 8)
    v = torch.arange(t, device=DEV).remainder(1021).half()[:, None, None].expand(t, 1, 8)
    pool = torch.zeros(2, pages, page, 1, 8, dtype=H, device=DEV)  # heads of 8: one element at a time
    ops.paged_cache_append(None, k, v, pool[0], pool[1], slots)
    flat = pool.view(2, -1, 1, 8)[:, :t].flip(1)
    assert torch.equal(flat[0], k) and torch.equal(flat[1], v)
    del pool, flat
    four = torch.zeros(2, pages, page * 32, dtype=torch.uint8, device=DEV)[:, :, :page * 17].unflatten(2, (page, 1, 17))
    k4, v4 = ((x % 4)[:, :, :1].expand(t, 1, 32) for x in (k, v))  # exact in 4 bits
    ops.paged_cache_append_fp4(None, k4, v4, four[0], four[1], slots)
    got = ops.paged_cache_read_fp4(four[0], four[1], slots, H)
    assert torch.equal(got[0], k4) and torch.equal(got[1], v4)


def test_rope_table_refusals():
    for positions, rot in ((4, 3), (-1, 4), (4, -2)):
        with pytest.raises(ValueError, match="rope_table"):
            ops.rope_table(positions, rot, device="cpu")
    assert ops.rope_table(0, 4, device="cpu").shape == (0, 4) and ops.rope_table(3, 0, device="cpu").shape == (3, 0)
