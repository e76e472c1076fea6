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


def test_one_block_for_many_rows():
    """2^26 rows and more of a table of one block (the query's tokens are one token's)."""
    from moba_amd import paged_select_blocks
    tokens, heads, page = (1 << 20) + 5, 64, 256
    q = torch.ones((1, heads, 64), dtype=BF16, device="cuda").expand(tokens, -1, -1)
    table, sums = torch.zeros((1, 4100), dtype=torch.int32, device="cuda"), torch.zeros((1, 1, 64), device="cuda")
    for rows in (tokens, tokens - 9):      # (the last nine belong to no sequence)
        got = paged_select_blocks(q, sums, table, ints(rows), ints(0, rows), page, 4100 * page, 2)
        assert got.shape == (tokens, heads, 2)
        assert (got[:rows, :, 0] == 0).all() and (got[:rows, :, 1] == -1).all() and (got[rows:] == -1).all()


def test_key_sums_of_many_rows():
    """Rows beyond 2^25 waves' pages: a sequence of 2^26 new tokens, most of whose pages the table names wrongly, and a short one."""
    from moba_amd import PagedKVCache, paged_key_sums
    page, heads, long = 16, 8, 1 << 26
    g = torch.Generator().manual_seed(1)
    k = torch.randn((6, heads, page, 64), generator=g).to(BF16).cuda()
    cache = PagedKVCache(k, torch.zeros_like(k))
    table = torch.full((2, long // page), -1, dtype=torch.int32, device="cuda")
    table[0, 0], table[0, 12345], table[0, -1], table[1, 0], table[1, 1] = 4, 2, 0, 3, 1
    sums = torch.full((6, heads, 64), 7.5, device="cuda")
    paged_key_sums(cache, sums, table, ints(long, 21), ints(0, long, long + 21), long + 21)
    for id, held in ((4, 16), (2, 16), (0, 16), (3, 16), (1, 5)):
        part = k[id, :, :held].double()
        assert ((sums[id].double() - part.sum(1)).abs() <= 18 * 2.0 ** -24 * part.abs().sum(1)).all(), id
    assert (sums[5] == 7.5).all()


def test_large_tables():
    """2^31 entries and more are no table of a pool's."""
    from moba_amd import PagePool, paged_release, paged_reserve
    pool = PagePool.full(4, 16)
    table, lengths = torch.empty((8192, 1 << 18), dtype=torch.int32, device="cuda"), torch.zeros(8192, dtype=torch.int32, device="cuda")
    for call in (lambda: paged_reserve(pool, table, lengths, lengths, 4), lambda: paged_release(pool, table, lengths, lengths)):
        with pytest.raises(ValueError, match="2\\^31"):
            call()


def test_wide_tables():
    """Rows of 2^31 pages and more are refused by every operator on the cache."""
    import moba_amd as m
    cache = m.PagedKVCache.empty(3, 2, 64, 16, dtype=BF16)
    q, kv, sums = torch.zeros((5, 4, 64), dtype=BF16, device="cuda"), torch.zeros((5, 2, 64), dtype=BF16, device="cuda"), cache.key_sums()
    blocks = torch.zeros((5, 4, 3), dtype=torch.int32, device="cuda")
    index = (torch.empty((1, 1 << 31), dtype=torch.int32, device="cuda"), ints(5), ints(0, 5))
    for call in (lambda: m.paged_append(cache, kv, kv, *index), lambda: m.paged_attention(q, cache, *index),
                 lambda: m.paged_prefix_attention(q, cache, *index, ints(0, 1), ints(0)), lambda: m.paged_key_sums(cache, sums, *index, 5),
                 lambda: m.paged_select_blocks(q, sums, *index, 16, 1 << 24, 3), lambda: m.paged_block_attention(q, cache, blocks, *index, 32)):
        with pytest.raises(ValueError, match="2\\^31"):
            call()


@pytest.mark.parametrize("quantized", [True, False])
def test_block_attention_in_several_launches(quantized):
    """More lists of blocks than a launch's workspace takes: the same as pieces of the tokens, each in one launch."""
    from moba_amd import PagedKVCache, _lib, paged_block_attention
    heads, kv_heads, page, d = 64, 8, 16, 64
    old, new, pages = (20000, 300), (13000, 5000), 2400
    g = torch.Generator(device="cuda").manual_seed(2)
    k, v = (torch.randn((pages + 400, kv_heads, page, d), generator=g, device="cuda") for _ in range(2))
    if quantized:
        cache = PagedKVCache(*(x.to(torch.float8_e4m3fn) for x in (k, v)), *(torch.rand((pages + 400, kv_heads), generator=g, device="cuda") for _ in range(2)))
    else:
        cache = PagedKVCache(k.to(BF16), v.to(BF16))
    table = torch.full((2, pages), -1, dtype=torch.int32, device="cuda")
    ids = torch.randperm(pages + 400, generator=g, device="cuda").int()
    table[0], table[1, :400] = ids[:pages], ids[pages:]
    tokens = sum(new)
    q = torch.randn((tokens, heads, d), generator=g, device="cuda").to(BF16)
    at = torch.cat([torch.arange(o, o + n, device="cuda") for o, n in zip(old, new)]) // page
    blocks = torch.full((tokens, heads, 64), -1, dtype=torch.int32, device="cuda")
    for i in (0, 17, 63):
        blocks[..., i] = (torch.rand((tokens, heads), generator=g, device="cuda") * (at + 1)[:, None]).int()
    size = _lib.load().moba_paged_block_attention_workspace_bytes
    assert size(tokens, 2, heads, kv_heads, d, page, pages, page, 64, quantized) < 1 << 30
    got = paged_block_attention(q, cache, blocks, table, ints(old[0] + new[0], old[1] + new[1]), ints(0, new[0], tokens), page)
    row = 0
    for b in range(2):
        for first in range(0, new[b], 4000):
            n = min(4000, new[b] - first)
            part = paged_block_attention(q[row:row + n], cache, blocks[row:row + n], table[b:b + 1], ints(old[b] + first + n), ints(0, n), page)
            assert torch.equal(got[row:row + n], part), (b, first)
            row += n
    assert row == tokens
