"""Blocks of 4-bit floats at the end of their type's range: what is finite is held as something finite.

A block's exponent ends where 6 * 2^e still fits the type: at 13 for fp16, 6 * 2^13 = 49152, and at 125 for bf16,
6 * 2^125 = 1.5 * 2^127.  Up to 7 * 2^e an element is off by 2^e at most; above, it is cut off to 6 * 2^e."""

import math

import pytest
import torch

from fp4_case import fp4_round, new_pool, to_dev
from paged_case import DEV, attention_ref, check_attention, gen, offsets
from pulsar_amd import ops

H, B = torch.float16, torch.bfloat16
LAST = {H: 13, B: 125}


def held(x, dtype):
    """The values that blocks hold, in 64 bits.  (bf16's last exponent is fp16's, 2^112 further up.)"""
    far = LAST[dtype] - 13
    return torch.ldexp(fp4_round(torch.ldexp(x.double(), torch.tensor(-far)), True)[2], torch.tensor(far))


def near_the_end(dtype, g):
    """Rows [n, 32] whose largest magnitudes go up to the type's greatest value."""
    most = torch.finfo(dtype).max
    unit = 2.0 ** LAST[dtype]
    rows = [torch.full((32,), most, dtype=torch.float64), torch.full((32,), -most, dtype=torch.float64)]
    for top in (3.49 * unit, 3.5 * unit, 6.0 * unit, 6.9 * unit, 6.97 * unit, 7.0 * unit, 7.5 * unit, most):
        x = (2 * torch.rand(32, generator=g, dtype=torch.float64) - 1) * top
        x[int(torch.randint(32, (1,), generator=g))] = top
        rows.append(x)
    return torch.stack(rows).clamp(-most, most).to(dtype)


def test_the_reference_is_finite_and_near():
    for dtype in (H, B):
        x = near_the_end(dtype, gen(1)).double()
        unit = 2.0 ** LAST[dtype]
        v = held(x, dtype)
        assert bool(v.isfinite().all()) and bool(v.to(dtype).isfinite().all()) and torch.equal(v.to(dtype).double(), v)
        assert bool(((v - x).abs() <= torch.where(x.abs() <= 7 * unit, unit, x.abs() - 6 * unit)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("shift", [0, 1])  # 1: one element at a time
@pytest.mark.parametrize("dtype", [H, B])
def test_finite_blocks_stay_finite(dtype, shift):
    x = near_the_end(dtype, gen(1)).view(-1, 1, 64)
    t = x.shape[0]
    pool = to_dev(new_pool(2, 1, 16, 1, 64))
    slots = torch.arange(t, device=DEV)
    flat = torch.zeros(2, t * 64 + 8, dtype=dtype, device=DEV)[:, shift:shift + t * 64]
    k, v = flat.view(2, t, 1, 64).unbind()
    k.copy_(x)
    v.copy_(x.flip(0))
    ops.paged_cache_append_fp4(None, k, v, pool[0], pool[1], slots)
    got = ops.paged_cache_read_fp4(pool[0], pool[1], slots, dtype)
    assert torch.equal(got[0].cpu().double(), held(x, dtype))
    assert torch.equal(got[1].cpu().double(), held(x, dtype).flip(0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [H, B])
def test_blocks_of_every_kind(dtype):
    """Borders between codes, magnitudes from the least to the greatest, zeros, NaN and infinities."""
    least = torch.finfo(dtype).smallest_normal
    grid = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0] * 4, dtype=torch.float64)
    rows = []
    for e in ((-24, -14, -3, 0, 5, 12, 13) if dtype == H else (-133, -126, -60, 0, 60, 124, 125)):
        for sign in (1.0, torch.where(torch.arange(32) % 3 == 0, -1.0, 1.0)):
            rows.append(torch.ldexp(grid * sign, torch.tensor(e)))
    rows += [torch.linspace(-top, top, 32, dtype=torch.float64) for top in (3.5, 6.9375, 7.0, 7.5)]
    rows += [torch.full((32,), x, dtype=torch.float64) for x in (0.0, -0.0, torch.finfo(dtype).max, least, least / 4)]
    rows += [torch.where(torch.arange(32) == 7, bad, torch.randn(32, generator=gen(1)).double())
             for bad in (math.nan, math.inf, -math.inf)]
    x = torch.stack(rows).to(dtype).view(-1, 1, 64)
    t = x.shape[0]
    # far from the end both references are fp4_round's; bf16's least magnitudes have its exponent's own limit
    want = fp4_round(x, dtype == H)[2]
    far = x.double().unflatten(-1, (2, 32)).abs().amax(-1, keepdim=True) > 2.0 ** 100
    if dtype == B:
        want = torch.where(far.expand(-1, -1, -1, 32).flatten(-2) & ~want.isnan(), held(x.double().nan_to_num(0.0, 0.0, 0.0), dtype), want)
    assert bool((want.isfinite() == x.double().unflatten(-1, (2, 32)).isfinite().all(-1, keepdim=True).expand(-1, -1, -1, 32).flatten(-2)).all())
    pool = to_dev(new_pool(2, -(-t // 16), 16, 1, 64))
    slots = torch.arange(t, device=DEV)
    ops.paged_cache_append_fp4(None, x.to(DEV), x.flip(0).to(DEV), pool[0], pool[1], slots)
    k, v = (y.cpu() for y in ops.paged_cache_read_fp4(pool[0], pool[1], slots, dtype))
    for got, w in ((k, want.to(dtype)), (v, want.to(dtype).flip(0))):
        assert torch.equal(got.isnan(), w.isnan()) and torch.equal(got[~w.isnan()], w[~w.isnan()])
        assert torch.equal(torch.signbit(got[~w.isnan()]), torch.signbit(w[~w.isnan()])) and not bool(got.isinf().any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [H, B])
def test_rotated_keys_past_the_type(dtype):
    """A rotation makes magnitudes of up to sqrt(2) times its elements': more than the blocks hold, and than fp16."""
    g = gen(2)
    most = torch.finfo(dtype).max if dtype == H else 1.4 * 2.0 ** 127
    x = ((2 * torch.rand(12, 1, 64, generator=g, dtype=torch.float64) - 1).sign() * most).to(dtype)
    rope = ops.rope_table(300, 64, device="cpu")
    positions = torch.randint(0, 300, (12,), generator=g)
    c, s = rope[positions].double()[:, None].split(32, -1)
    a, b = x.double().split(32, -1)
    turned = torch.cat([a * c - b * s, b * c + a * s], -1).float()
    assert bool(turned.isfinite().all()) and bool((turned.abs() > 7 * 2.0 ** LAST[dtype]).any())
    pool = to_dev(new_pool(2, 1, 16, 1, 64))
    slots = torch.arange(12, device=DEV)
    ops.paged_cache_append_fp4(None, x.to(DEV), x.to(DEV), pool[0], pool[1], slots, rope.to(DEV), positions.to(DEV))
    got = ops.paged_cache_read_fp4(pool[0], pool[1], slots, dtype)
    assert torch.equal(got[0].cpu().double(), held(turned, dtype))
    assert torch.equal(got[1].cpu().double(), held(x, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 40, 200])
@pytest.mark.parametrize("dtype", [H, B])
def test_attention_over_a_great_value_is_finite(dtype, new):
    """The mean of values of which one is near the type's end, at either end of the sequence."""
    n, dim = 200, 64
    g = gen(3)
    k, q = torch.randn(n, 1, dim, generator=g).to(dtype), torch.randn(new, 2, dim, generator=g).to(dtype)
    great = near_the_end(dtype, g).view(-1, 1, dim)
    for at in (0, n - 1):
        for x in great:
            v = torch.zeros(n, 1, dim, dtype=dtype)
            v[at] = x
            pool = to_dev(new_pool(2, -(-n // 16), 16, 1, dim))
            ops.paged_cache_append_fp4(None, k.to(DEV), v.to(DEV), pool[0], pool[1], torch.arange(n, device=DEV))
            tables = torch.arange(pool.shape[1], dtype=torch.int32, device=DEV)[None]
            out = ops.paged_attention_fp4(q.to(DEV), pool[0], pool[1], tables,
                                          torch.tensor([n], dtype=torch.int32, device=DEV), offsets([new]).to(DEV), new, n,
                                          scale=0.0)
            assert bool(out.isfinite().all())
            ref = attention_ref(q, held(k, dtype), held(v, dtype), n, new, 0.0, 0, 0.0)
            check_attention(out, None, ref, dim, n, dtype)
