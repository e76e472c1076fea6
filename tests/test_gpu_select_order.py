"""paged_select_blocks: which blocks a token gets does not depend on what else is in the batch."""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("each", [1, 3, 5, 8, 12, 16, 24, 33, 40, 64, 65, 150])
def test_a_choice_is_the_tokens_own(each, d):
    """Pages whose sums cancel but for what 64 bits lose, so that the order of the additions decides: the same blocks for a token by
    itself, and beside few and many others, in front of it and behind, in tables of any width."""
    from moba_amd import paged_select_blocks
    page, heads, kv_heads, count = 16, 4, 2, 40
    g = torch.Generator().manual_seed(each + d)
    sums = torch.randn((count, each, kv_heads, d), generator=g)
    some = each // 3
    large = torch.randn((count, some, kv_heads, d), generator=g) * 2.0 ** 52
    for block in range(count):        # large ones, their negatives, and small ones, anywhere in the block
        at = torch.randperm(each, generator=g)
        sums[block, at[:some]], sums[block, at[some:2 * some]] = large[block], -large[block]
    table = torch.arange(count * each, dtype=torch.int32)[None].repeat(600, 1).cuda()
    sums = sums.flatten(0, 1).cuda()
    q = torch.randn((600, heads, d), generator=g).to(BF16).cuda()
    lengths = [(1 + (7 * i) % count) * each * page - i % page for i in range(600)]
    lengths[0] = count * each * page
    call = lambda first, end, wide: paged_select_blocks(q[first:end], sums, table[first:end, :wide], ints(lengths[first:end]),  # noqa: E731
                                                        ints(list(range(end - first + 1))), page, page * each, 9)
    wide = count * each
    want = call(0, 600, wide)
    assert want[0, :, -1].tolist() == [count - 1] * heads
    for first, end in ((0, 1), (0, 2), (0, 40), (0, 150), (7, 8), (599, 600), (500, 600), (30, 400)):
        assert torch.equal(call(first, end, wide), want[first:end]), (first, end)
    broad = torch.cat([table, torch.full((600, 50 * each), -1, dtype=torch.int32, device="cuda")], 1)
    assert torch.equal(paged_select_blocks(q, sums, broad, ints(lengths), ints(list(range(601))), page, page * each, 9), want)
    # as one sequence's new tokens, all of which see whole blocks up to the last
    tokens = min(600, each * page)
    one = lambda first, end: paged_select_blocks(q[:end - first], sums, table[:1], ints([count * each * page - tokens + end]),  # noqa: E731
                                                 ints([0, end - first]), page, page * each, 9)
    piece = one(0, tokens)
    single = torch.cat([paged_select_blocks(q[i:i + 1], sums, table[:1], ints([count * each * page - tokens + i + 1]), ints([0, 1]), page,
                                            page * each, 9) for i in range(0, tokens, 29)])
    assert torch.equal(piece[::29], single)
