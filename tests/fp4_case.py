"""Blocks of 4-bit floats on the host, by their definition, and pools of them for the tests."""

from __future__ import annotations

import math

import torch

from paged_case import DEV, gen

STEPS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def fp4_round(x: torch.Tensor, fp16: bool = False):
    """(codes, exponent bytes, values in 64 bits) of x [..., dim], as given in any float type: each block of
    32 on its own."""
    grid = torch.tensor(STEPS, dtype=torch.float64)
    b = x.double().unflatten(-1, (-1, 32))
    bad = ~b.isfinite().all(-1)
    safe = torch.where(bad[..., None], 0.0, b)
    mant, exp = torch.frexp(safe.abs().amax(-1))  # the largest is mant * 2^exp, mant in [1/2, 1)
    e = torch.where(mant == 0, torch.tensor(-127), exp - 3 + (mant >= 0.875).int()).clamp(-127, 13 if fp16 else 127)
    unit = torch.ldexp(torch.ones_like(mant), e)[..., None]
    m = (safe.abs() / unit).clamp(max=6.0)
    dist = (m[..., None] - grid).abs()
    near = dist.amin(-1, keepdim=True)
    # of two codes as near the even one
    code = torch.where(dist == near, torch.arange(8) + 100 * (torch.arange(8) % 2), 1000).amin(-1) % 100
    sign = torch.signbit(safe)
    values = grid[code] * unit * torch.where(sign, -1.0, 1.0)
    values = torch.where(bad[..., None], math.nan, values)
    return (code + 8 * sign).flatten(-2), torch.where(bad, 255, e + 127), values.flatten(-2)


def row_bytes(dim: int) -> int:
    return dim // 2 + dim // 32


def new_pool(planes: int, pages: int, page: int, heads: int, dim: int, pad: int = 0, fill: int = 0xFF) -> torch.Tensor:
    """A host pool [planes, pages, page, heads, row] of `fill`, its pages at multiples of 16 bytes, `pad` more
    of them apart."""
    size = page * heads * row_bytes(dim)
    flat = torch.full((planes, pages, -(-size // 16) * 16 + 16 * pad), fill, dtype=torch.uint8)
    return flat[:, :, :size].unflatten(2, (page, heads, row_bytes(dim)))


def to_dev(pool: torch.Tensor) -> torch.Tensor:
    """The same on the device, strides kept."""
    planes, pages = pool.shape[:2]
    whole = pool.as_strided((planes, pages, pool.stride(1)), (pool.stride(0), pool.stride(1), 1))
    return whole.to(DEV).as_strided(pool.shape, pool.stride())


def fp4_kv(lens, page, heads, dim, dtype, seed, slack=3, pad=0, fill=0xFF, edit=None):
    """(k_cache, v_cache, tables, k rows, v rows): paged_case.paged_kv in 4 bits; rows are the values held,
    [len, heads, dim] in dtype (exact).  `edit(ks, vs)` may change keys and values before they are rounded.
    Slots that nothing is written to hold `fill` (0xFF: NaN)."""
    g = gen(seed)
    held = [-(-l // page) for l in lens]
    pages, width = sum(held) + slack, max(held + [1])
    order = torch.randperm(pages, generator=g)
    pool = new_pool(2, pages, page, heads, dim, pad, fill)
    tables = torch.full((len(lens), width), -1, dtype=torch.int32)
    raw = [[torch.randn(l, heads, dim, generator=g) for l in lens] for _ in range(2)]
    if edit is not None:
        edit(*raw)
    rows, at = ([], []), 0
    for b, l in enumerate(lens):
        mine = order[at:at + held[b]]
        at += held[b]
        tables[b, :held[b]] = mine.int()
        j = torch.arange(l)
        for plane in range(2):
            codes, exps, values = fp4_round(raw[plane][b], dtype == torch.float16)
            rows[plane].append(values.to(dtype))
            flat = pool[plane].as_strided((pages, page * heads * row_bytes(dim)), (pool.stride(1), 1))
            cut = page * heads * dim // 2
            packed = (codes[..., 0::2] + 16 * codes[..., 1::2]).to(torch.uint8)
            flat[:, :cut].view(pages, heads, page, dim // 2)[mine[j // page], :, j % page] = packed
            flat[:, cut:].view(pages, heads, page, dim // 32)[mine[j // page], :, j % page] = exps.to(torch.uint8)
    dev = to_dev(pool)
    return dev[0], dev[1], tables.to(DEV), rows[0], rows[1]
