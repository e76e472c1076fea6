"""paged_key_sums, paged_select_blocks and paged_block_attention on the GPU against their definitions in 64 bits."""

import pytest
import torch

from paged_reference import Batch
from rotary_reference import frequencies
from serving_reference import check_chosen, check_against, chosen_attended, held, key_sums, selected

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def some_blocks(batch, heads, n, block_size, own=True):
    """[rows, heads, n]: random blocks up to a row's own, in any order, some of them twice, some that are none."""
    g, out = batch.g, torch.full((batch.rows, heads, n), -1, dtype=torch.int32)
    for row, at in enumerate(batch.positions()):
        if at is None:
            out[row] = 0
            continue
        last = at // block_size
        out[row] = torch.randint(-1, last + 1, (heads, n), generator=g).int()
        if own:
            out[row, :, n // 2] = last
        out[row, 0, 0] = last + 1                     # beyond the row's own
    return out


# ---- sums
@pytest.mark.parametrize("old,new,page,kv_heads,d,dtype,quantized", [
    ([0], [1], 64, 1, 128, BF16, True), ([0], [1], 16, 3, 64, FP16, False), ([63, 64, 65, 0, 5], [1, 1, 1, 0, 200], 64, 8, 128, BF16, True),
    ([63, 64, 65, 0, 5], [1, 1, 1, 0, 200], 32, 5, 64, BF16, True), ([7, 250, 300], [500, 9, 1], 256, 2, 128, FP16, False),
    ([7, 250, 300], [500, 9, 1], 128, 2, 64, BF16, False), ([16 * i for i in range(80)], [1, 0, 17, 2] * 20, 16, 2, 128, FP16, True),
    ([0, 3], [3000, 70], 16, 1, 64, FP16, True)])
def test_sums(old, new, page, kv_heads, d, dtype, quantized):
    from moba_amd import paged_key_sums
    print("sums", old[:6], new[:6], page, kv_heads, d, dtype, quantized, flush=True)
    batch = Batch(old, new, page, kv_heads, d, dtype, quantized, seed=page + d)
    for b, (o, c) in enumerate(zip(old, new)):            # behind a sequence's end: whatever
        if (o + c) % page and c:
            batch.pages[0][int(batch.table[b, (o + c) // page]), :, (o + c) % page:] = float("nan")
    sums = torch.full((batch.pages[0].shape[0], kv_heads, d), 7.5, device="cuda")
    paged_key_sums(batch.cache(), sums, *batch.index(), batch.rows)
    want = key_sums(batch)
    for page, x in enumerate(sums.cpu()):
        if page in want:
            assert bool(((x.double() - want[page][0]).abs() <= want[page][1] + 2.0 ** -149).all()), page
        else:
            assert bool((x == 7.5).all()), page
    again = torch.zeros_like(sums)
    paged_key_sums(batch.cache(), again, *batch.index(), batch.rows + 100)
    assert all(torch.equal(sums[p], again[p]) for p in want)


def test_sums_of_tables_that_do_not_fit():
    from moba_amd import paged_key_sums
    batch = Batch([100, 30, 5], [30, 2, 40], 16, 2, 64, BF16, True, seed=2)
    batch.table[0, 6], batch.table[1, 1], batch.table[2, 1] = -1, batch.pages[0].shape[0], 2 ** 31 - 1
    cache, (table, lengths, cu) = batch.cache(), batch.index()
    sums = torch.zeros((batch.pages[0].shape[0], 2, 64), device="cuda")
    paged_key_sums(cache, sums, table, lengths, cu, batch.rows)
    want = key_sums(batch)
    for page, x in enumerate(sums.cpu()):
        assert bool(((x.double() - want[page][0]).abs() <= want[page][1]).all()) if page in want else not x.any()
    for n in (0, -7, 2 ** 31 - 1, 10 ** 6):
        paged_key_sums(cache, sums, table, torch.full_like(lengths, n), cu, batch.rows)
    for bad in ((5, 0, 9, 1), (-7, 900, 3, 3), (2 ** 31 - 1, -2 ** 31, 0, 70)):
        paged_key_sums(cache, sums, table, lengths, ints(*bad), batch.rows)
    paged_key_sums(cache, sums, table, lengths, cu, 0)
    torch.cuda.synchronize()
    # a value that is not finite is a sum that is not
    batch.pages[0][int(batch.table[0, 7]), 1, 3, 5] = float("nan")
    paged_key_sums(batch.cache(), sums, table, lengths, cu, batch.rows)
    assert sums[int(batch.table[0, 7])].isnan().nonzero().tolist() == [[1, 5]]


# ---- selection
@pytest.mark.parametrize("old,new,page,block,topk,heads,kv_heads,d,dtype,wide", [
    ([0], [1], 64, 64, 1, 4, 1, 128, BF16, 0), ([0], [1], 16, 64, 5, 2, 2, 64, FP16, 0), ([5000], [1], 64, 64, 7, 8, 2, 128, BF16, 0),
    ([5000], [1], 64, 512, 3, 32, 8, 128, BF16, 0), ([5000, 100, 4095, 0], [3, 0, 1, 9], 16, 48, 12, 6, 2, 64, FP16, 0),
    ([5000, 100, 4095, 0], [3, 0, 1, 9], 32, 256, 64, 6, 3, 128, FP16, 3), ([20000], [2], 16, 16, 24, 5, 1, 64, BF16, 900),
    ([900, 1000], [40, 130], 16, 32, 6, 4, 2, 128, BF16, 0), ([16 * i for i in range(70)], [1, 0, 2] * 23 + [1], 16, 16, 4, 4, 2, 64, BF16, 0),
    ([40000, 300], [1, 1], 64, 2048, 9, 4, 2, 128, BF16, 0), ([140000], [1], 256, 4096, 12, 4, 1, 64, FP16, 0)])
def test_select(old, new, page, block, topk, heads, kv_heads, d, dtype, wide):
    from moba_amd import paged_select_blocks
    print("select", old[:6], new[:6], page, block, topk, heads, kv_heads, d, dtype, wide, flush=True)
    batch = Batch(old, new, page, kv_heads, 64, dtype, False, seed=page + d + topk, pad_rows=2, noise=0.0)
    if wide:
        batch.table = torch.cat([batch.table, torch.full((len(old), wide), -1, dtype=torch.int32)], 1)
    sums = torch.randn((batch.pages[0].shape[0], kv_heads, d), generator=batch.g)
    q = torch.randn((batch.rows, heads, d), generator=batch.g).to(dtype)
    want = selected(q, sums, batch.table, batch.lengths, batch.cu, page, block, topk)
    got = paged_select_blocks(q.cuda(), sums.cuda(), *batch.index(), page, block, topk)
    assert got.dtype == torch.int32 and torch.equal(got.cpu(), want), (got.cpu() != want).nonzero()[:5]


@pytest.mark.parametrize("page,block,length", [(16, 16, 700), (16, 32, 3000), (16, 16, 20000), (32, 96, 30000)])
def test_equal_scores(page, block, length):
    """Few different sums, and all the same: of equal products the lowest block."""
    from moba_amd import paged_select_blocks
    batch = Batch([length], [3], page, 2, 64, BF16, False, seed=1, noise=0.0)
    q, = batch.tensors(6)
    for kinds in (1, 2, 7):
        values = torch.randn((kinds, 2, 64), generator=batch.g)
        sums = values[torch.randint(0, kinds, (batch.pages[0].shape[0],), generator=batch.g)]
        if block > page:     # (blocks of the same pages: their sums are formed alike)
            each, row = block // page, batch.table[0]
            whole = row[:len(row) // each * each].view(-1, each)
            used = whole[(whole >= 0).all(1)]
            sums[used.flatten().long()] = values[torch.randint(0, kinds, (used.shape[0], 1), generator=batch.g).expand(-1, each).flatten()]
        want = selected(q, sums, batch.table, batch.lengths, batch.cu, page, block, 9)
        got = paged_select_blocks(q.cuda(), sums.cuda(), *batch.index(), page, block, 9)
        assert torch.equal(got.cpu(), want), kinds
    assert paged_select_blocks(q.cuda(), torch.zeros_like(sums).cuda(), *batch.index(), page, block, 9)[0, 0, :8].tolist() == list(range(8))


def test_select_what_is_not_finite():
    from moba_amd import paged_select_blocks
    batch = Batch([2000], [2], 16, 2, 64, BF16, False, seed=5, noise=0.0)
    q, = batch.tensors(4)
    sums = torch.randn((batch.pages[0].shape[0], 2, 64), generator=batch.g)
    flat = batch.table[0].tolist()
    sums[flat[3], 0, 5], sums[flat[9], 0, 1], sums[flat[40], 1, 2] = float("nan"), float("inf"), -float("inf")
    sums[flat[50]], sums[flat[51]] = 1e38, -1e38
    want = selected(q, sums, batch.table, batch.lengths, batch.cu, 16, 16, 6)
    assert torch.equal(paged_select_blocks(q.cuda(), sums.cuda(), *batch.index(), 16, 16, 6).cpu(), want)
    q[0, 0, 3] = float("nan")          # all NaN: the lowest
    got = paged_select_blocks(q.cuda(), sums.cuda(), *batch.index(), 16, 16, 6).cpu()
    assert got[0, 0].tolist() == [0, 1, 2, 3, 4, 125] and torch.equal(got[1:], want[1:])


def test_select_of_tables_that_do_not_fit():
    from moba_amd import paged_select_blocks
    batch = Batch([400, 30, 0], [5, 2, 40], 16, 2, 64, BF16, False, seed=6, pad_rows=3)
    batch.table[0, 4], batch.table[0, 7], batch.table[0, 9] = -1, batch.pages[0].shape[0], 2 ** 31 - 1
    q, = batch.tensors(4)
    sums = torch.randn((batch.pages[0].shape[0], 2, 64), generator=batch.g)
    table, lengths, cu = batch.index()
    for lens in ([405, 32, 40], [405, -3, 0], [3, 1, 5], [100000, 32, 2 ** 31 - 1]):
        for rows in ([0, 5, 7, 47], [0, 0, 50, 50], [10, 12, 12, 30]):
            want = selected(q, sums, batch.table, lens, rows, 16, 48, 4)
            got = paged_select_blocks(q.cuda(), sums.cuda(), table, ints(*lens), ints(*rows), 16, 48, 4)
            assert torch.equal(got.cpu(), want), (lens, rows)
    for bad in ((5, 0, 9, 1), (-7, 900, 3, 3), (2 ** 31 - 1, -2 ** 31, 0, 70)):
        paged_select_blocks(q.cuda(), sums.cuda(), table, lengths, ints(*bad), 16, 48, 4)
    torch.cuda.synchronize()
    assert (paged_select_blocks(q.cuda(), sums.cuda(), table[:0], lengths[:0], cu[:1], 16, 48, 4) == -1).all()
    assert paged_select_blocks(q[:0].cuda(), sums.cuda(), table, lengths, cu, 16, 48, 4).shape == (0, 4, 4)


def test_select_in_several_launches(monkeypatch):
    """More scores than a launch's workspace takes: wide tables, many rows."""
    from moba_amd import paged_select_blocks
    wide, heads = 16000, 64
    batch = Batch([700], [90], 16, 1, 64, BF16, False, seed=8, noise=0.0)
    batch.table = torch.cat([batch.table, torch.full((1, wide - batch.table.shape[1]), -1, dtype=torch.int32)], 1)
    q, = batch.tensors(heads)
    sums = torch.randn((batch.pages[0].shape[0], 1, 64), generator=batch.g)
    got = paged_select_blocks(q.cuda(), sums.cuda(), *batch.index(), 16, 16, 5)
    narrow = batch.table[:, :60].contiguous()
    assert torch.equal(got, paged_select_blocks(q.cuda(), sums.cuda(), narrow.cuda(), *batch.index()[1:], 16, 16, 5))
    want = selected(q[:3], sums, narrow, [703], [0, 3], 16, 16, 5)
    assert torch.equal(got[:3].cpu(), want)


# ---- attention
CASES = [  # old, new, page, block, n, heads, kv heads, head_dim, dtype, quantized, rows behind
    ([0], [1], 64, 64, 1, 4, 1, 128, BF16, True, 0),
    ([0], [1], 16, 32, 3, 1, 1, 64, FP16, False, 0),
    ([4096], [1], 64, 256, 5, 32, 8, 128, BF16, True, 0),
    ([4095], [1], 64, 256, 5, 32, 8, 128, BF16, False, 0),
    ([127, 128, 129, 31, 32, 0, 15, 16], [1] * 8, 16, 16, 4, 6, 2, 128, FP16, True, 0),
    ([127, 128, 129, 31, 32, 0, 15, 16], [1] * 8, 32, 96, 2, 6, 2, 64, BF16, True, 3),
    ([300, 5, 2000, 77], [1, 0, 3, 8], 16, 48, 7, 12, 4, 128, BF16, True, 2),
    ([300, 5, 2000, 77], [1, 0, 3, 8], 64, 128, 7, 12, 4, 128, FP16, False, 2),
    ([50, 0, 1000], [20, 33, 5], 16, 32, 6, 7, 1, 64, FP16, True, 0),               # more rows than a unit has
    ([50, 0, 1000], [20, 33, 5], 16, 32, 6, 40, 1, 64, BF16, False, 0),             # more heads on one than a unit has rows
    ([10 * i for i in range(70)], [1, 2, 0, 1, 1] * 14, 16, 16, 3, 4, 2, 64, BF16, True, 0),
    ([40000, 100], [1, 1], 64, 1024, 20, 8, 2, 128, BF16, True, 0),                 # several runs
    ([30000], [2], 16, 16, 64, 4, 4, 64, FP16, False, 0),
    ([90000], [1], 16, 16, 30, 4, 1, 64, BF16, True, 0),                            # more blocks than a window has
    ([100] * 300, [1] * 300, 16, 32, 2, 8, 8, 64, BF16, True, 0),                   # more units than the chip has places
    ([20000, 70], [2, 1], 16, 16, 64, 16, 1, 128, BF16, True, 0),                   # longer lists than LDS has room for
    ([20000], [2], 16, 16, 64, 16, 1, 64, FP16, False, 0),
]


@pytest.mark.parametrize("old,new,page,block,n,heads,kv_heads,d,dtype,quantized,behind", CASES)
def test_blocks(old, new, page, block, n, heads, kv_heads, d, dtype, quantized, behind):
    from moba_amd import paged_block_attention
    print("blocks", old[:6], new[:6], page, block, n, heads, kv_heads, d, dtype, quantized, behind, flush=True)
    batch = Batch(old, new, page, kv_heads, d, dtype, quantized, seed=page + d + len(old), pad_rows=behind)
    q, = batch.tensors(heads)
    blocks = some_blocks(batch, heads, n, block)
    args = (q.cuda(), batch.cache(), blocks.cuda(), *batch.index(), block)
    got = paged_block_attention(*args)
    check_chosen(batch, got, q, blocks, block)
    assert torch.equal(got, paged_block_attention(*args))          # the same bits every time
    if len(old) < 20:
        check_chosen(batch, paged_block_attention(*args, scaling=-0.3), q, blocks, block, -0.3)


@pytest.mark.parametrize("quantized", [True, False])
def test_all_blocks_are_all_keys(quantized):
    from moba_amd import paged_attention, paged_block_attention
    batch = Batch([500, 31, 64], [1, 3, 2], 16, 2, 128, BF16, quantized, seed=5)
    q, = batch.tensors(8)
    blocks = torch.arange(17, dtype=torch.int32).expand(6, 8, 17)
    got = paged_block_attention(q.cuda(), batch.cache(), blocks.cuda(), *batch.index(), 32)
    check_chosen(batch, got, q, blocks, 32)
    want, slack = chosen_attended(batch, q, blocks, 32)
    check_against(paged_attention(q.cuda(), batch.cache(), *batch.index()), want, slack, BF16)


@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("d", [64, 128])
def test_large_scores_and_scales(quantized, d):
    from moba_amd import paged_block_attention
    batch = Batch([700, 40, 200], [1, 3, 20], 16, 2, d, BF16, quantized, seed=2)
    if quantized:
        for s in batch.scales:
            s *= torch.rand(s.shape, generator=batch.g) + 0.5
            s[::5] *= -1
            s[3::7] = 0
        batch.scales[1] *= 2.0 ** torch.randint(-60, 60, batch.scales[1].shape, generator=batch.g).float()
    else:
        batch.pages[1][::2] *= 2.0 ** 40
    q = batch.tensors(4)[0] * 30
    blocks = some_blocks(batch, 4, 5, 48)
    for scaling in (None, -0.1, 0.0, 1.0):
        got = paged_block_attention(q.cuda(), batch.cache(), blocks.cuda(), *batch.index(), 48, scaling=scaling)
        check_chosen(batch, got, q, blocks, 48, scaling)


@pytest.mark.parametrize("quantized", [True, False])
def test_values_that_are_not_finite(quantized):
    """They reach the rows that have chosen them, and no others of the same unit."""
    from moba_amd import paged_block_attention
    nan = float("nan")
    for d, dtype in ((128, BF16), (64, FP16)):
        batch = Batch([320, 70, 9], [1, 6, 1], 32, 2, d, dtype, quantized, seed=3)
        for b, (o, c) in enumerate(zip(batch.old, batch.new)):                     # behind the end
            last = int(batch.table[b, (o + c) // 32])
            if last >= 0:
                for x in batch.pages:
                    x[last, :, (o + c) % 32:] = nan
        q, = batch.tensors(6)
        blocks = some_blocks(batch, 6, 2, 64)
        blocks[0] = torch.tensor([[0, 5], [1, 5], [2, 5], [0, 1], [3, 4], [-1, 2]])
        run = lambda: paged_block_attention(q.cuda(), batch.cache(), blocks.cuda(), *batch.index(), 64)  # noqa: E731
        check_chosen(batch, run(), q, blocks, 64)
        batch.pages[1][int(batch.table[0, 2]), 0, 3, 5] = nan if quantized else float("inf")     # a value of block 1
        batch.pages[0][int(batch.table[0, 6]), 1, 3, 5] = nan                                    # a key of block 3
        got = run()
        check_chosen(batch, got, q, blocks, 64)
        assert got[0, 4].isnan().all() and got[0, [0, 2, 3, 5]].isfinite().all()
        assert not got[0, 1].isfinite().all()


@pytest.mark.parametrize("quantized", [True, False])
def test_tables_that_do_not_fit(quantized):
    from moba_amd import paged_block_attention
    batch = Batch([100, 0, 300, 40, 200], [2, 20, 1, 3, 50], 16, 2, 64, BF16, quantized, seed=4, pad_rows=4)
    batch.table[4, 3], batch.table[4, 9] = -7, 2 ** 30
    batch.table[0, 1], batch.table[0, 4], batch.table[1], batch.table[2, 5:] = -1, batch.pages[0].shape[0], 2 ** 31 - 1, -2 ** 31
    q, = batch.tensors(4)
    blocks = some_blocks(batch, 4, 5, 32)
    blocks[:, 1, 1], blocks[:, 2, 2], blocks[:, 3, 0] = 2 ** 31 - 1, -2 ** 31, 10 ** 6
    cache, (table, lengths, cu) = batch.cache(), batch.index()
    got = paged_block_attention(q.cuda(), cache, blocks.cuda(), table, lengths, cu, 32)
    check_chosen(batch, got, q, blocks, 32)
    assert not got[2:22].any() and not got[-4:].any()
    assert not paged_block_attention(q.cuda(), cache, torch.full_like(blocks, -1).cuda(), table, lengths, cu, 32).any()
    for n in (0, -5):
        assert not paged_block_attention(q.cuda(), cache, blocks.cuda(), table, torch.full_like(lengths, n), cu, 32).any()
    for n in (1, 2 ** 31 - 1):
        paged_block_attention(q.cuda(), cache, blocks.cuda(), table, torch.full_like(lengths, n), cu, 32)
    for bad in ((0, 5, 1, 9, 2, 60), (-7, 900, 0, 0, 3, 3), (2 ** 31 - 1, -2 ** 31, 0, 1, 2, 3)):
        paged_block_attention(q.cuda(), cache, blocks.cuda(), table, lengths, ints(*bad), 32)
    torch.cuda.synchronize()
    cut = Batch([100], [2], 16, 2, 64, BF16, quantized, seed=5)
    cut.table = cut.table[:, :3].contiguous()                   # 48 of 102 tokens, the second block is half there
    q, = cut.tensors(4)
    blocks = torch.tensor([0, 1, 3], dtype=torch.int32).expand(2, 4, 3)
    check_chosen(cut, paged_block_attention(q.cuda(), cut.cache(), blocks.cuda(), *cut.index(), 32), q, blocks, 32)


def test_views_and_nothing():
    from moba_amd import paged_block_attention, paged_key_sums, paged_select_blocks
    batch = Batch([100, 30], [1, 4], 16, 2, 128, BF16, True, seed=6)
    q = batch.tensors(6)[0].cuda()
    cache, (table, lengths, cu) = batch.cache(), batch.index()
    sums = cache.key_sums()
    paged_key_sums(cache, sums, table, lengths, cu, 5)
    wide = torch.full((2, 2 * table.shape[1]), -1, dtype=torch.int32, device="cuda")
    wide[:, ::2] = table
    again = torch.zeros_like(sums)
    paged_key_sums(cache, again, wide[:, ::2], lengths, cu, 5)
    assert torch.equal(sums, again)
    blocks = paged_select_blocks(q, sums, table, lengths, cu, 16, 32, 3)
    want = paged_block_attention(q, cache, blocks, table, lengths, cu, 32)
    odd = torch.empty(q.numel() + 1, dtype=BF16, device="cuda")[1:].view_as(q).copy_(q)
    for view in (torch.cat([q, q[:, :2]], 1)[:, :6], q.transpose(0, 1).contiguous().transpose(0, 1), torch.stack([q, q], -1)[..., 0], odd):
        assert torch.equal(paged_select_blocks(view, sums, table, lengths, cu, 16, 32, 3), blocks)
        assert torch.equal(paged_block_attention(view, cache, blocks, table, lengths, cu, 32), want)
    assert torch.equal(paged_select_blocks(q, sums.transpose(1, 2).contiguous().transpose(1, 2), wide[:, ::2], lengths, cu, 16, 32, 3), blocks)
    spread = torch.stack([blocks, blocks], -1)[..., 0]
    assert torch.equal(paged_block_attention(q, cache, spread, wide[:, ::2], lengths, cu, 32), want)
    assert paged_block_attention(q[:0], cache, blocks[:0], table, lengths, cu, 32).shape == (0, 6, 128)
    assert not paged_block_attention(q, cache, blocks, table[:0], lengths[:0], cu[:1], 32).any()


def test_a_cache_of_more_than_2_31_elements():
    from moba_amd import PagedKVCache, paged_block_attention, paged_key_sums, paged_select_blocks
    E4M3 = torch.float8_e4m3fn
    pages = 2 ** 31 // (8 * 256 * 128) + 2
    zeros = lambda: torch.zeros((pages, 8, 256, 128), dtype=E4M3, device="cuda")  # noqa: E731
    cache = PagedKVCache(zeros(), zeros(), *(torch.ones((pages, 8), device="cuda") for _ in range(2)))
    for i, page in enumerate((pages - 1, 0)):
        cache.v_pages[page] = torch.full((8, 256, 128), 2.0 + 2 * i, device="cuda").to(E4M3)
        cache.k_pages[page] = torch.full((8, 256, 128), 1.0 - i, device="cuda").to(E4M3)
    table, sums = ints(pages - 1, 0).view(1, 2), cache.key_sums()
    paged_key_sums(cache, sums, table, ints(512), ints(0, 512), 512)
    assert (sums[pages - 1] == 256).all() and not sums[0].any()
    q = torch.ones((1, 8, 128), dtype=BF16, device="cuda")
    blocks = paged_select_blocks(q, sums, table, ints(512), ints(0, 1), 256, 256, 2)
    assert (blocks == ints(0, 1)).all()
    assert (paged_block_attention(q * 0, cache, blocks, table, ints(512), ints(0, 1), 256) == 3).all()
    assert (paged_block_attention(q, cache, blocks[..., :1].contiguous(), table, ints(512), ints(0, 1), 256) == 2).all()


def test_graph_and_streams():
    """A captured step -- sums, selection, attention -- follows lengths and rows; two at once have workspaces of their own."""
    from moba_amd import paged_block_attention, paged_key_sums, paged_select_blocks
    batches = [Batch([1000, 50, 63, 400], [1, 1, 1, 1], 16, 2, 128, BF16, True, seed=8), Batch([3000, 500], [2, 2], 16, 2, 128, BF16, True, seed=9)]

    def step(q, cache, sums, table, lengths, cu):
        paged_key_sums(cache, sums, table, lengths, cu, q.shape[0])
        blocks = paged_select_blocks(q, sums, table, lengths, cu, 16, 64, 4)
        return blocks, paged_block_attention(q, cache, blocks, table, lengths, cu, 64)

    args, graphs, outs = [], [], []
    for batch in batches:
        cache = batch.cache()
        sums = torch.randn((batch.pages[0].shape[0], 2, 128), generator=batch.g).cuda()
        args.append((batch.tensors(8)[0].cuda(), cache, sums, *batch.index()))
        step(*args[-1])
    torch.cuda.synchronize()
    for a in args:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step(*a))
    want_other = step(*args[1])
    side = torch.cuda.Stream()
    for i, (lens, rows) in enumerate((([1001, 51, 64, 401], [0, 1, 2, 3, 4]), ([1, 51, 64, 390], [0, 1, 2, 3, 4]),
                                      ([900, 51, 0, 401], [0, 2, 3, 3, 4]), ([30, 30, 60, 300], [0, 0, 0, 4, 4]))):
        args[0][4].copy_(torch.tensor(lens))
        args[0][5].copy_(torch.tensor(rows))
        torch.cuda.synchronize()
        side.wait_stream(torch.cuda.current_stream())
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
            eager_other = step(*args[1])
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs[0], step(*args[0]))), i
        assert all(torch.equal(a, b) and torch.equal(c, b) for a, b, c in zip(outs[1], want_other, eager_other)), i


@pytest.mark.parametrize("quantized", [False, True])
def test_serving(quantized):
    """As they are used together: pages reserved, prompts with a common beginning and then tokens appended, their key sums kept, the
    blocks chosen and attended -- and all of the keys, the common ones once -- drafted tokens taken back; every step against the
    definitions, and generation against the packed operator on the whole sequence."""
    from moba_amd import (PagedKVCache, PagePool, moba_attn_varlen_gqa, paged_append, paged_block_attention, paged_key_sums,
                          paged_prefix_attention, paged_release, paged_reserve, paged_select_blocks)
    from serving_reference import check_prefix
    heads, kv_heads, d, page, block, topk, b = 4, 2, 128, 16, 32, 3, 3
    g = torch.Generator().manual_seed(4)
    cache = PagedKVCache.empty(60, kv_heads, d, page, dtype=BF16 if not quantized else torch.float8_e4m3fn)
    pool, sums = PagePool.full(60, page), cache.key_sums()
    table, lengths = torch.full((b, 20), -1, dtype=torch.int32, device="cuda"), ints(0, 0, 0)
    inv_freq = frequencies(d // 2, "cuda")
    history = [[] for _ in range(b)]     # of every sequence: (q, k, v) rows

    def run(new, rows):
        cu, owners, positions, slots = paged_reserve(pool, table, lengths, ints(*new), rows)
        q, k, v = (torch.randn((rows, h, d), generator=g).to(BF16).cuda() for h in (heads, kv_heads, kv_heads))
        turned = paged_append(cache, k, v, table, lengths, cu, inv_freq, q)
        paged_key_sums(cache, sums, table, lengths, cu, rows)
        if not quantized:                # the slots are where the tokens went
            live = slots[:sum(new)]
            assert torch.equal(cache.v_pages.transpose(1, 2).flatten(0, 1)[live], v[:sum(new)])
            flat = cache.k_pages.transpose(1, 2).flatten(0, 1)[live]
            for i, owner in enumerate(owners[:sum(new)].tolist()):
                assert positions[i] == len(history[owner])
                history[owner].append((turned[i], flat[i], v[i]))
        return turned, cu

    def state(new, cu, rows):
        batch = Batch([0] * b, new, page, kv_heads, d, BF16, quantized)
        batch.pages, batch.scales = [cache.k_pages.cpu(), cache.v_pages.cpu()], [None, None]
        if quantized:
            batch.scales = [cache.k_scales.cpu(), cache.v_scales.cpu()]
        batch.table, batch.lengths, batch.cu, batch.rows = table.cpu(), lengths.cpu(), cu.cpu(), rows
        batch.old = [n - m for n, m in zip(lengths.tolist(), new)]
        return batch

    run([70, 0, 0], 70)                          # the common beginning, in sequence 0 ...
    table[1:, :4] = table[:1, :4]                # ... 64 tokens of which the others share
    lengths[1:] = 64
    history[1], history[2] = list(history[0][:64]), list(history[0][:64])
    for new in ([1, 40, 90], [1, 1, 1], [3, 2, 1], [1, 1, 1]):
        turned, cu = run(new, sum(new) + 1)
        batch = state(new, cu, sum(new) + 1)
        blocks = paged_select_blocks(turned, sums, table, lengths, cu, page, block, topk)
        assert torch.equal(blocks.cpu(), selected(turned.cpu(), sums.cpu(), batch.table, batch.lengths, batch.cu, page, block, topk))
        for s in range(b):                       # the sums are those of the pages
            there, k, _ = held(batch, s, int(lengths[s]))
            for i in range(-(-int(lengths[s]) // page)):
                part = k[i * page:(i + 1) * page]
                off = (sums[int(batch.table[s, i])].cpu().double() - part.sum(0)).abs()
                assert bool((off <= (page + 2) * 2.0 ** -24 * part.abs().sum(0)).all())
        out = paged_block_attention(turned, cache, blocks, table, lengths, cu, block)
        check_chosen(batch, out, turned.cpu(), blocks.cpu(), block)
        check_prefix(batch, [(0, 3)], paged_prefix_attention(turned, cache, table, lengths, cu, ints(0, 3), ints(64)), turned.cpu())
        if not quantized:
            packed = [torch.stack([row[i] for rows in history for row in rows]) for i in range(3)]
            ends = [0] + [sum(len(r) for r in history[:i + 1]) for i in range(b)]
            # (the operator for whole prompts rounds the means: only where both choose the same blocks is the attention the same)
            plain = moba_attn_varlen_gqa(*packed, ints(*ends), max(lengths.tolist()), block, topk)
            at, near = 0, []
            for s, n in enumerate(new):
                near.append((plain[ends[s + 1] - n:ends[s + 1]].float() - out[at:at + n].float()).abs().amax(-1) < 2e-2)
                at += n
            assert torch.cat(near).float().mean() > 0.9
    before = pool.free_count.item()
    paged_release(pool, table, lengths, ints(40, 64, 66))       # drafted tokens rejected, a sequence back to what it shares
    assert lengths.tolist() == [40, 64, 66] and pool.free_count.item() > before
    table[1:, :4], lengths[1:] = -1, 0                          # (theirs to give back is only what lies behind)
    paged_release(pool, table, lengths, ints(0, 0, 0))
    assert (table[0] == -1).all()
