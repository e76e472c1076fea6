"""Calls of the operators of serving at the limits that their documentation names, and beyond, on the GPU."""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def test_wide_tables_of_the_selection():
    """16384 blocks in a row of the table are taken, one more is a ValueError, whatever the tensors."""
    from moba_amd import paged_select_blocks
    q, sums = torch.zeros((3, 2, 64), dtype=BF16, device="cuda"), torch.zeros((4, 1, 64), device="cuda")
    for page, block in ((16, 16), (16, 48), (256, 512)):
        widest = 16384 * (block // page)
        table = torch.zeros((1, widest + 1), dtype=torch.int32, device="cuda")
        for query in (q, torch.stack([q, q], -1)[..., 0]):
            got = paged_select_blocks(query, sums, table[:, :widest], ints(100), ints(0, 3), page, block, 2)
            assert got.shape == (3, 2, 2) and got.max() == 99 // block
            with pytest.raises(ValueError, match="16384 blocks"):
                paged_select_blocks(query, sums, table, ints(100), ints(0, 3), page, block, 2)
