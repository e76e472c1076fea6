"""paged_prefix_attention on the GPU in the precision that it promises for few rows, which the bounds for many rows are too wide to hold it to."""

import pytest
import torch

from prefix_precision import cases, exact_batch, exact_queries, is_within, wanted

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,dtype,quantized", [(d, dtype, quantized) for d in (64, 128) for dtype in (torch.bfloat16, torch.float16)
                                               for quantized in (True, False)])
def test_few_rows(d, dtype, quantized):
    """Groups and sequences of up to 256 rows (128 with 16-bit pages and heads of 128), alone and beside a group of more."""
    from moba_amd import paged_prefix_attention
    for i, (old, new, rep) in enumerate(cases(d, quantized)):
        for beside in (False, True):
            print("few rows", d, dtype, quantized, len(old), new[:7], rep, beside, flush=True)
            groups, members = [0, len(old)], len(old)
            if beside:
                old, new, groups = old + [70, 64], new + [300, 1], groups + [members + 2]
            batch = exact_batch(old, new, 16, 2, d, dtype, quantized, seed=i + d)
            batch.table[:members, :6] = batch.table[0, :6].clone()
            if beside:
                batch.table[members:, :4] = batch.table[members, :4].clone()
            q = exact_queries(batch, 2 * rep)
            index = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (groups, [96, 64][:len(groups) - 1])]
            got = paged_prefix_attention(q.cuda(), batch.cache(), *batch.index(), *index)
            want, bound = wanted(batch, q)
            rows = sum(new[:members])
            good = is_within(got, want, bound)[:rows]
            assert good.all(), (new[:members], rep, beside, (~good).nonzero()[:5].tolist(),
                                ((got.cpu().double() - want).abs() / bound)[:rows].max().item())
