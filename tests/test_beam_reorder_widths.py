"""beam_reorder of states that allow different widths of copy in one call."""

import pytest
import torch

from paged_case import DEV, gen
from pulsar_amd import ops


@pytest.mark.gpu
@pytest.mark.parametrize("odd", [1, 2, 3, 4, 6, 8, 12, 16, 20, 40, 16384 + 8, 2 * 16384 + 2, 3 * 16384 + 5])
def test_rows_of_every_length_beside_wide_ones(odd):
    """Rows of `odd` bytes, and views whose addresses are so odd, beside rows of whole vectors, in any order."""
    g = gen(odd)
    rows = torch.tensor([4, 4, -1, 0, 5, 2, 3], dtype=torch.int32)
    there = ((rows >= 0) & (rows < 5))[:, None]
    wide = torch.randint(0, 256, (5, 4096), generator=g).to(torch.uint8).to(DEV)
    narrow = torch.randint(0, 256, (5, odd), generator=g).to(torch.uint8).to(DEV)
    shifted = torch.randint(0, 256, (5 * 64 + 16,), generator=g).to(torch.uint8).to(DEV)[odd % 16:][:5 * 64].view(5, 64)
    last = torch.randint(-9, 9, (5, 17), generator=g).to(DEV)  # rows of 8 bytes more than whole vectors
    for states in ([wide, narrow, shifted, last], [narrow, wide], [last, shifted, wide, narrow, last, wide, narrow, wide, last]):
        for s, o in zip(states, ops.beam_reorder(states, rows.to(DEV))):
            assert torch.equal(o.cpu(), torch.where(there, s.cpu()[rows.clamp(0, 4).long()], 0))


def _time(call):
    call()
    best = 1e9
    for _ in range(10):
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        call()
        end.record()
        torch.cuda.synchronize()
        best = min(best, start.elapsed_time(end))
    return best


@pytest.mark.gpu
def test_a_flag_does_not_slow_down_what_stands_beside_it():
    """A state is copied by its own width: a byte a row beside 1 GB, and a history of odd length, take their own
    time more and not a multiple of the whole.  (The least of ten; a factor of two is left for the card.)"""
    rows = torch.arange(32, dtype=torch.int32, device=DEV).flip(0).contiguous()
    big = torch.zeros(32, 1 << 23, dtype=torch.int32, device=DEV)
    flag = torch.zeros(32, dtype=torch.bool, device=DEV)
    history = torch.zeros(32, 501, dtype=torch.int64, device=DEV)
    alone = _time(lambda: ops.beam_reorder([big], rows))
    for others in ([flag], [history], [flag, history]):
        assert _time(lambda: ops.beam_reorder([big, *others], rows)) < 2 * alone
