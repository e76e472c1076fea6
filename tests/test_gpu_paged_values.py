"""paged_attention on the GPU: values that are not finite, and batches of more work than the chip takes at once."""

import pytest
import torch

from paged_reference import Batch, attended, check_attention

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("old,new,heads", [([3000], [1], 4), ([700, 2500], [1, 3], 6), ([2000, 5, 900], [40, 1, 50], 8),
                                           ([9000], [160], 8)])
def test_infinite_values_in_any_run(old, new, heads, dtype):
    """An infinite value is the sum's in every row that sees it, whichever of the runs that the keys are cut into it lies in: the
    last, the first, one between, and beside other rows' infinities of the other sign."""
    from moba_amd import paged_attention
    batch = Batch(old, new, 64, 2, 64, dtype, False, seed=21)
    q, = batch.tensors(heads)
    length, values = old[0] + new[0], batch.pages[1]
    for element, position, sign in ((3, old[0], 1), (4, 0, -1), (5, length // 2, 1), (6, old[0] - 1, -1), (6, 7, -1)):
        values[int(batch.table[0, position // 64]), :, position % 64, element] = sign * float("inf")
    got = paged_attention(q.cuda(), batch.cache(), *batch.index())
    want = attended(batch, q)[0]
    assert torch.equal(want.isinf().any(0).any(0).nonzero().flatten(), torch.tensor([3, 4, 5, 6])) and not want.isnan().any()
    check_attention(batch, got, q)
