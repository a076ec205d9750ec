"""paged_cache_free of more rows than one launch has workgroups for."""

import pytest
import torch

from paged_case import DEV
from pulsar_amd import ops


@pytest.mark.gpu
def test_more_rows_than_a_launch_has_workgroups():
    """2^24 workgroups of 256 threads are more than one launch may have.  Entries outside the tables, and rows that
    are named twice, are passed over."""
    n, rows = (1 << 24) + 3, 40
    refs = torch.ones(rows, dtype=torch.int32, device=DEV)
    tables = torch.arange(rows, dtype=torch.int32, device=DEV)[:, None].repeat(1, 2)
    tables[:, 1] = -1
    lens = torch.full((rows,), 5, dtype=torch.int32, device=DEV)
    which = torch.full((n,), -1, dtype=torch.int32, device=DEV)
    gone = [0, 7, 8, 20, 30, 39]
    for row, at in zip(gone, (0, (1 << 22) - 1, 1 << 22, 1 << 23, (1 << 24) - 1, n - 1)):
        which[at] = row
    which[100], which[1 << 24] = 39, 0
    ops.paged_cache_free(refs, tables, lens, which)
    left = torch.tensor([r not in gone for r in range(rows)])
    assert torch.equal(refs.cpu(), left.int()) and torch.equal(lens.cpu(), 5 * left.int())
    assert torch.equal(tables.cpu()[:, 0], torch.where(left, torch.arange(rows), -1).int())
