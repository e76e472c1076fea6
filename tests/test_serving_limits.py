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


def test_wide_tables_are_refused():
    """Rows of 2^31 pages and more, by every operator on the cache."""
    from moba_amd import (PagedKVCache, paged_append, paged_attention, paged_block_attention, paged_key_sums, paged_prefix_attention,
                          paged_select_blocks)
    cache = PagedKVCache.empty(3, 2, 64, 16, dtype=torch.bfloat16, device="meta")
    q, kv, sums = (torch.empty(s, device="meta").to(d) for s, d in (((5, 4, 64), torch.bfloat16), ((5, 2, 64), torch.bfloat16),
                                                                    ((3, 2, 64), torch.float32)))
    calls = (lambda *i: paged_append(cache, kv, kv, *i), lambda *i: paged_attention(q, cache, *i),
             lambda *i: paged_prefix_attention(q, cache, *i, meta(2), meta(1)), lambda *i: paged_key_sums(cache, sums, *i, 5),
             lambda *i: paged_select_blocks(q, sums, *i, 16, 1 << 24, 3), lambda *i: paged_block_attention(q, cache, meta(5, 4, 3), *i, 32))
    for call in calls:
        with pytest.raises(ValueError, match="2\\^31"):
            call(meta(1, 1 << 31), meta(1), meta(2))
        with pytest.raises(RuntimeError, match="AMD GPU"):
            call(meta(1, 9), meta(1), meta(2))


def test_the_lists_of_long_pieces_are_bounded():
    """The workspace of the attention over chosen blocks: lists of up to 512 MiB beside the rows' parts, however many rows there are."""
    from moba_amd import _lib
    size = _lib.load().moba_paged_block_attention_workspace_bytes
    for tokens in (1 << 17, 1 << 20, (1 << 24) - 1):
        for d, cache8 in ((64, 1), (128, 0)):
            short, long = (size(tokens, 1, 32, 8, d, 64, pages, 64, 64, cache8) for pages in (1024, 4096))
            assert 0 < short < 1 << 29 and 0 < long - short <= 1 << 29, (tokens, d, short, long)
    assert size((1 << 24) - 1, 1, 128, 1, 64, 64, 4096, 64, 64, 1) > 0     # (2^26 units)
