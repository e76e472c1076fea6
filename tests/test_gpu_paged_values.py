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


def scores_that_are_not_finite(d, dtype):
    """(batch, queries): infinite keys and queries, NaN among the queries, for few rows and for many."""
    batch = Batch([300, 50, 7, 1200], [6, 60, 1, 2], 16, 2, d, dtype, False, seed=14)
    q, = batch.tensors(6)
    for b, position, head, sign in ((0, 303, 0, 1), (1, 80, 1, -1), (0, 17, 1, 1), (2, 3, 0, -1), (3, 1100, 0, 1)):
        batch.pages[0][int(batch.table[b, position // 16]), head, position % 16, 9] = sign * float("inf")
    q[2, 1, 4], q[20, 5, 0], q[40, 2, 3], q[41, 0, 8] = float("nan"), float("inf"), float("nan"), -float("inf")
    return batch, q


def finite_bound(batch, q, want):
    """Of rows whose result is finite, half a step and what 32 bits allow, by the sizes of the elements that are finite: an infinite
    one gives no term of a finite sum."""
    pages = batch.pages
    batch.pages = [x.where(x.isfinite(), 0) for x in pages]
    slack = attended(batch, q.where(q.isfinite(), 0))[1]
    batch.pages = pages
    return torch.finfo(q.dtype).eps / 2 * 1.001 * want.abs() + slack + 2.0 ** -25


@pytest.mark.parametrize("d,dtype", [(128, BF16), (64, BF16), (128, FP16), (64, FP16)])
def test_finite_rows_beside_scores_that_are_not(d, dtype):
    """Every row within its own bound: one that saw a key more or less would not be."""
    from moba_amd import paged_attention
    batch, q = scores_that_are_not_finite(d, dtype)
    got = paged_attention(q.cuda(), batch.cache(), *batch.index()).cpu().double()
    want = attended(batch, q)[0]
    assert want.isnan().any() and want.isfinite().any((1, 2)).all()
    assert torch.equal(got.isnan(), want.isnan()) and not want.isinf().any()
    off, fine = (got - want).abs(), want.isfinite()
    bad = fine & ~(off <= finite_bound(batch, q, want))
    assert not bad.any(), bad.nonzero()[:5].tolist()


def among(short, count, long, at):
    return [short + i % 7 for i in range(at)] + [long] + [short + i % 5 for i in range(count - at - 1)]


LARGE = [  # more groups of rows than the chip has places for a key/value head, and than four times as many: old, new, page, heads, kv heads, d, dtype, quantized
    (among(90, 65, 9000, 40), [1] * 65, 64, 16, 8, 128, BF16, True),
    (among(90, 257, 9000, 3), [1] * 257, 16, 8, 8, 64, BF16, True),
    (among(60, 33, 5000, 32), [1] * 33, 32, 8, 8, 128, FP16, False),
    (among(60, 129, 5000, 0), [1, 2, 0] * 43, 32, 8, 8, 128, BF16, False),
    (among(300, 17, 5000, 5), [1] * 17, 64, 32, 32, 128, FP16, True),
    (among(40, 66, 5000, 65), [1, 2] * 33, 64, 32, 32, 64, BF16, True),
    (among(40, 3, 3000, 1), [1] * 3, 16, 512, 256, 64, FP16, False),
    (among(40, 9, 3000, 4), [1] * 9, 16, 256, 256, 64, BF16, True),
    (among(40, 9, 700, 4), [33, 2, 20, 40, 33, 1, 5, 9, 17], 32, 512, 256, 64, BF16, True),   # two groups of few rows
    (among(20, 6, 900, 2), [130, 40, 35, 160, 33, 129], 16, 128, 128, 64, BF16, False),       # many rows
    (among(20, 18, 900, 7), [33, 35] * 9, 16, 128, 128, 64, FP16, False),
    (among(20, 3, 900, 1), [70, 70, 300], 64, 128, 128, 128, BF16, True),
    (among(20, 10, 700, 9), [65, 1, 66] * 3 + [70], 64, 128, 128, 128, FP16, True),
]


@pytest.mark.parametrize("old,new,page,heads,kv_heads,d,dtype,quantized", LARGE)
def test_more_work_than_one_round(old, new, page, heads, kv_heads, d, dtype, quantized):
    from moba_amd import paged_attention
    print("large", len(old), max(old), new[:6], page, heads, kv_heads, d, dtype, quantized, flush=True)
    batch = Batch(old, new, page, kv_heads, d, dtype, quantized, seed=len(old) + kv_heads, pad_rows=1)
    q, = batch.tensors(heads)
    cache, index = batch.cache(), batch.index()
    got = paged_attention(q.cuda(), cache, *index)
    check_attention(batch, got, q)
    assert torch.equal(got, paged_attention(q.cuda(), cache, *index, max_new=max(new)))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_scales_of_pages_that_nobody_names(dtype, bad):
    """The first page of the pool, which is read in the place of pages that are none, and all others that no table names."""
    from moba_amd import paged_attention
    batch = Batch([200, 70, 9, 33, 0], [1, 6, 1, 40, 90], 32, 2, 128, dtype, True, seed=5, spare=4)
    batch.table[0, 2], batch.table[3, 0], batch.table[4, 1] = -1, 10 ** 6, -1
    free = sorted(set(range(batch.pages[0].shape[0])) - set(batch.table.flatten().tolist()))
    if free[0] != 0:                                      # (page 0's part goes to a free one)
        batch.table[batch.table == 0] = free[-1]
        for x in (*batch.pages, *batch.scales):
            x[free[-1]] = x[0]
        free = [0] + free[:-1]
    q, = batch.tensors(8)
    for x in batch.scales:
        x[free] = bad
    for x in batch.pages:
        x[free] = float("nan")
    check_attention(batch, paged_attention(q.cuda(), batch.cache(), *batch.index()), q)
