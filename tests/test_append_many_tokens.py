"""The append of more tokens than one launch has workgroups for, by vectors."""

import pytest
import torch

from fp4_case import new_pool, to_dev
from paged_case import DEV, gen
from pulsar_amd import ops

B = torch.bfloat16


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 4])
def test_more_tokens_than_a_launch_has_workgroups(bits):
    """2^24 workgroups of 256 threads are more than one launch may have; heads of 256 go two tokens to a workgroup.
    Most tokens have no slot; those that do, and the queries, are as in a call of these alone."""
    t, heads, dim, page = (1 << 25) + 5, 4, 256, 16
    g = gen(bits)
    some = torch.randint(0, t, (300,), generator=g)
    edges = torch.tensor([0, 1, (1 << 23) - 1, 1 << 23, (1 << 24) - 1, 1 << 24, (1 << 24) + 1, (1 << 25) - 1, 1 << 25, t - 1])
    some = torch.cat([some, edges]).unique()
    n = some.numel()
    base = torch.randn(t * 8 + heads * dim, generator=torch.Generator(DEV).manual_seed(1), device=DEV, dtype=torch.bfloat16)
    k = base.as_strided((t, heads, dim), (8, dim, 1))  # a token's elements are the last one's, 8 on
    v = base[:heads * dim].flip(0).view(1, heads, dim).expand(t, heads, dim)
    q = base.as_strided((t, 1, dim), (8, dim, 1))
    pages = -(-n // page) + 1
    slots = torch.full((t,), -1, dtype=torch.int64, device=DEV)
    places = torch.randperm(pages * page, generator=g)[:n].to(DEV)
    some = some.to(DEV)
    slots[some] = places
    positions = torch.arange(t, device=DEV).remainder(50)
    rope = ops.rope_table(50, dim)

    def fresh():
        if bits == 16:
            return torch.full((2, pages, page, heads, dim), 3.0, dtype=B, device=DEV)
        return to_dev(new_pool(2, pages, page, heads, dim, fill=0xA5))

    op = ops.paged_cache_append if bits == 16 else ops.paged_cache_append_fp4
    want, got = fresh(), fresh()
    few = op(q[some], k[some], v[some], want[0], want[1], places, rope, positions[some])
    out = op(q, k, v, got[0], got[1], slots, rope, positions)
    assert torch.equal(got, want) and torch.equal(out[some], few)
    # and without queries and a rotation
    want, got = fresh(), fresh()
    op(None, k[some], v[some], want[0], want[1], places)
    op(None, k, v, got[0], got[1], slots)
    assert torch.equal(got, want)
