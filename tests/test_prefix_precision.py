"""The bound that holds paged_prefix_attention to its precision for few rows: that of many rows is outside (no GPU)."""

import pytest
import torch

from prefix_precision import cases, exact_batch, exact_queries, is_within, limit, wanted


@pytest.mark.parametrize("d,dtype,quantized", [(64, torch.bfloat16, True), (128, torch.bfloat16, True), (64, torch.bfloat16, False),
                                               (128, torch.bfloat16, False), (64, torch.float16, False), (128, torch.float16, False)])
def test_one_element_is_told_apart(d, dtype, quantized):
    """Results of probabilities that are rounded once -- planted here -- do not pass, those of exact ones do."""
    count = 0
    for old, new, rep in cases(d, quantized):
        assert sum(new) * rep <= limit(d, quantized)
        batch = exact_batch(old, new, 16, 1, d, dtype, quantized, seed=count + d)
        batch.table[:, :6] = batch.table[0, :6].clone()
        q = exact_queries(batch, rep)
        want, bound = wanted(batch, q)
        assert is_within(want.to(dtype), want, bound).all()
        planted = wanted(batch, q, one_element=True)[0].to(dtype)
        assert (~is_within(planted, want, bound)).sum() > 4, (old, new, rep)
        count += 1
    assert count >= 7
