"""What the operators of serving refuse for its size, before anything is launched (no GPU)."""

import pytest
import torch

I32 = torch.int32


def meta(*shape):
    return torch.empty(shape, dtype=I32, device="meta")


def test_large_tables_are_refused():
    """2^31 entries of a table, or pages of a pool (tensors without memory)."""
    from moba_amd import PagePool, paged_release, paged_reserve
    with pytest.raises(ValueError, match="2\\^31"):
        PagePool(meta(1 << 31), meta(1), 16)
    pool = PagePool(meta((1 << 31) - 1), meta(1), 16)
    for sequences, wide in ((8192, 1 << 18), (1, 1 << 31), (2, 1 << 30)):
        for call in (paged_reserve, paged_release):
            rows = (4,) if call is paged_reserve else ()
            with pytest.raises(ValueError, match="2\\^31"):
                call(pool, meta(sequences, wide), meta(sequences), meta(sequences), *rows)
            with pytest.raises(RuntimeError, match="AMD GPU"):
                call(pool, meta(sequences, wide - 1), meta(sequences), meta(sequences), *rows)
