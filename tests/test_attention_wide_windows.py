"""Windows as wide as 32 bits hold, of sequences with fewer keys than new tokens: the first queries stand before
the first key, so that a window's lower end lies below -2^31."""

import math

import pytest
import torch

from fp4_case import fp4_kv
from paged_case import DEV, attention_ref, check_attention, gen, offsets, paged_kv
from pulsar_amd import ops

B = torch.bfloat16


@pytest.mark.gpu
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 2, 2 ** 31 - 100, 2 ** 30])
@pytest.mark.parametrize("new,before", [(4, 3), (9, 5), (100, 7), (100, 60), (700, 300)])
@pytest.mark.parametrize("bits", [4, 16])
def test_windows_of_32_bits(bits, new, before, window):
    lens, heads, dim = [new - before], 2, 128
    kc, vc, tables, ks, vs = (fp4_kv if bits == 4 else paged_kv)(lens, 16, heads, dim, B, 3)
    q = torch.randn(new, heads * 2, dim, generator=gen(4)).to(B).to(DEV)
    attention = ops.paged_attention_fp4 if bits == 4 else ops.paged_attention
    out, lse = attention(q, kc, vc, tables, torch.tensor(lens, dtype=torch.int32, device=DEV), offsets([new]).to(DEV), new,
                         lens[0], window=window, return_lse=True)
    assert bool((out[:before] == 0).all()) and bool((lse[:before] == -math.inf).all())
    ref = attention_ref(q[before:].cpu(), ks[0], vs[0], lens[0], lens[0], dim ** -0.5, 0, 0.0)
    check_attention(out[before:], lse[before:], ref, dim, lens[0], B)
