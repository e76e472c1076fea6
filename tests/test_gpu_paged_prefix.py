"""paged_prefix_attention on the GPU against softmax attention of every sequence by itself, in 64 bits."""

import pytest
import torch

from paged_reference import Batch
from serving_reference import check_prefix

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def share(batch, groups, shared):
    """The sequences of a group name the same pages for its first tokens; (cu_groups, shared) on the device."""
    for (first, end), tokens in zip(groups, shared):
        pages = tokens // batch.page
        batch.table[first:end, :pages] = batch.table[first, :pages].clone()
    cu = [g[0] for g in groups] + [groups[-1][1]]
    return tuple(torch.tensor(x, dtype=torch.int32, device="cuda") for x in (cu, shared))


CASES = [  # groups (first, end), shared, old, new, page, heads, kv heads, head_dim, dtype, quantized, rows behind
    ([(0, 1)], [0], [5], [1], 64, 4, 1, 128, BF16, True, 0),
    ([(0, 2)], [64], [64, 100], [1, 1], 64, 4, 1, 128, BF16, True, 0),
    ([(0, 2)], [64], [64, 100], [1, 1], 16, 1, 1, 64, FP16, False, 0),
    ([(0, 4)], [4096], [4096, 4097, 4500, 5000], [1] * 4, 64, 32, 8, 128, BF16, True, 0),
    ([(0, 4)], [4096], [4096, 4097, 4500, 5000], [1] * 4, 64, 32, 8, 128, BF16, False, 0),
    ([(0, 3), (3, 4), (4, 8)], [1008, 200, 64], [1008, 1010, 1100, 300, 64, 65, 80, 3000], [1, 2, 0, 1, 1, 3, 1, 1], 16, 6, 2, 64, FP16, True, 3),
    ([(0, 3), (3, 4), (4, 8)], [1008, 208, 64], [1008, 1010, 1100, 300, 64, 65, 80, 3000], [1, 2, 0, 1, 1, 3, 1, 1], 16, 6, 2, 64, BF16, False, 0),
    ([(1, 3), (3, 6)], [512, 2048], [3, 600, 512, 2048, 2500, 2049, 77], [1, 1, 5, 1, 1, 1, 2], 256, 8, 2, 128, FP16, True, 0),   # some outside
    ([(0, 40)], [320], [320 + 7 * i for i in range(40)], [1] * 40, 64, 8, 2, 128, BF16, True, 0),      # many rows together, few apart
    ([(0, 40)], [320], [320 + 7 * i for i in range(40)], [1] * 40, 32, 8, 2, 128, FP16, False, 0),
    ([(0, 40)], [320], [320 + 7 * i for i in range(40)], [1] * 40, 32, 10, 2, 64, FP16, True, 0),
    ([(0, 3), (3, 5)], [700, 130], [700, 704, 900, 130, 130], [200, 1, 40, 129, 3], 4 * 16, 8, 2, 128, BF16, True, 5),   # many rows in both
    ([(0, 3), (3, 5)], [704, 128], [704, 704, 900, 128, 130], [200, 1, 40, 129, 3], 64, 6, 2, 64, BF16, False, 0),
    ([(i, i + 2) for i in range(0, 80, 2)], [64 + 16 * i for i in range(40)], [64 + 16 * (i // 2) for i in range(80)], [1] * 80, 16, 4, 2, 64,
     BF16, True, 0),                                                                               # more sequences than a wave has lanes
    ([(0, 2)], [40000], [40000, 40100], [1, 2], 64, 8, 2, 128, BF16, True, 0),                     # several runs of the shared keys
    ([(0, 2)], [48], [48, 60], [1, 1], 16, 4, 2, 64, BF16, True, 0),                               # less than a tile is shared
    ([(0, 3), (3, 5)], [640, 128], [700, 640, 900, 128, 4000], [300, 40, 1, 170, 12], 64, 33, 3, 128, BF16, True, 4),   # rows of many runs
    ([(0, 3), (3, 5)], [640, 128], [700, 640, 900, 128, 9000], [300, 40, 1, 170, 12], 64, 33, 3, 64, FP16, False, 4),
]


@pytest.mark.parametrize("groups,shared,old,new,page,heads,kv_heads,d,dtype,quantized,behind", CASES)
def test_prefix(groups, shared, old, new, page, heads, kv_heads, d, dtype, quantized, behind):
    from moba_amd import paged_prefix_attention
    print("prefix", groups[:4], shared[:4], old[:6], new[:6], page, heads, kv_heads, d, dtype, quantized, behind, flush=True)
    batch = Batch(old, new, page, kv_heads, d, dtype, quantized, seed=page + d + len(old), pad_rows=behind)
    index = share(batch, groups, shared)
    q, = batch.tensors(heads)
    args = (q.cuda(), batch.cache(), *batch.index(), *index)
    got = paged_prefix_attention(*args)
    check_prefix(batch, groups, got, q)
    assert torch.equal(got, paged_prefix_attention(*args))          # the same bits every time
    check_prefix(batch, groups, paged_prefix_attention(*args, scaling=-0.2), q, -0.2)


@pytest.mark.parametrize("quantized", [True, False])
def test_more_is_shared_than_a_sequence_has(quantized):
    """Tokens of a group that lie before the shared keys' end see those up to themselves: the same table under all sequences."""
    from moba_amd import paged_prefix_attention
    for new in ([3, 1, 40, 0], [30, 1, 70, 2]):
        old = [500 - new[0], 100, 300, 20]
        batch = Batch(old, new, 16, 2, 64, BF16, quantized, seed=3)
        batch.table[:] = batch.table[0].clone()
        q, = batch.tensors(8)
        for shared in (64, 320, 500, 10 ** 6, 2 ** 31 - 1):
            index = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 4], [shared])]
            check_prefix(batch, [(0, 4)], paged_prefix_attention(q.cuda(), batch.cache(), *batch.index(), *index), q)


@pytest.mark.parametrize("quantized", [True, False])
def test_values_that_are_not_finite(quantized):
    """They reach the rows that see them, in the shared keys and in a sequence's own."""
    from moba_amd import paged_prefix_attention
    for d, dtype, new in ((128, BF16, [1, 3, 2]), (64, FP16, [20, 9, 30])):
        batch = Batch([256 - new[0], 300, 200], new, 32, 2, d, dtype, quantized, seed=4)
        batch.table[:, :6] = batch.table[0, :6].clone()
        index = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 3], [192])]
        used = set(batch.table.flatten().tolist())
        for page in set(range(batch.pages[0].shape[0])) - used:
            batch.pages[0][page], batch.pages[1][page] = float("nan"), float("nan")
        q, = batch.tensors(6)
        check_prefix(batch, [(0, 3)], paged_prefix_attention(q.cuda(), batch.cache(), *batch.index(), *index), q)
        batch.pages[1][int(batch.table[1, 9]), 1, 4, 5] = float("nan")          # sequence 1's own
        check_prefix(batch, [(0, 3)], paged_prefix_attention(q.cuda(), batch.cache(), *batch.index(), *index), q)
        batch.pages[0][int(batch.table[0, 2]), 0, 3, 7] = float("nan")          # everybody's
        got = paged_prefix_attention(q.cuda(), batch.cache(), *batch.index(), *index)
        check_prefix(batch, [(0, 3)], got, q)
        assert got[:, :3].isnan().all() and got[:new[0], 3:].isfinite().all()


@pytest.mark.parametrize("quantized", [True, False])
def test_tables_that_do_not_fit(quantized):
    """Entries that are no page, lengths beyond the table, groups that are none: rows that see nothing are zeros, and nothing outside
    the tensors is touched."""
    from moba_amd import paged_prefix_attention
    batch = Batch([100, 130, 300, 40, 200], [2, 20, 1, 3, 50], 16, 2, 64, BF16, quantized, seed=4)
    groups, shared = [(0, 2), (2, 4)], [96, 32]
    index = share(batch, groups, shared)
    batch.table[0:2, 2], batch.table[0:2, 4] = -1, batch.pages[0].shape[0]
    batch.table[1, 8:], batch.table[2, 5:] = 2 ** 31 - 1, -2 ** 31
    q, = batch.tensors(4)
    cache, (table, lengths, cu) = batch.cache(), batch.index()
    check_prefix(batch, groups, paged_prefix_attention(q.cuda(), cache, table, lengths, cu, *index), q)
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    for groups in ([5, 0, 5], [-3, 900, 2], [2 ** 31 - 1, 0, -2 ** 31], [3, 3, 3], [0, 5, 2]):
        for shared in ([64, 64], [-5, 2 ** 31 - 1], [10 ** 6, 0]):
            paged_prefix_attention(q.cuda(), cache, table, lengths, cu, ints(*groups), ints(*shared))
    for bad in ([0, 5, 1, 9, 2, 60], [-7, 900, 0, 0, 3, 3], [2 ** 31 - 1, -2 ** 31, 0, 1, 2, 3]):
        paged_prefix_attention(q.cuda(), cache, table, lengths, ints(*bad), *index)
    for length in (0, -5, 2 ** 31 - 1):
        got = paged_prefix_attention(q.cuda(), cache, table, torch.full_like(lengths, length), cu, *index)
        assert length > 0 or not got.any()
    torch.cuda.synchronize()
    # groups of nothing, and none at all: the attention of the sequences
    from moba_amd import paged_attention
    want = paged_attention(q.cuda(), cache, table, lengths, cu)
    empty = ints()
    assert torch.equal(paged_prefix_attention(q.cuda(), cache, table, lengths, cu, ints(0), empty), want)
    check_prefix(batch, [], paged_prefix_attention(q.cuda(), cache, table, lengths, cu, ints(2, 2), ints(64)), q)


@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("d", [64, 128])
def test_large_scores_and_scales(quantized, d):
    """Scores of hundreds, scales of every size beside each other, negative and zero softmax scales."""
    from moba_amd import paged_prefix_attention
    batch = Batch([700, 640, 800, 200], [1, 3, 35, 4], 16, 2, d, BF16, quantized, seed=2)
    index = share(batch, [(0, 3), (3, 4)], [640, 128])
    if quantized:
        batch.scales[1] *= 2.0 ** torch.randint(-60, 60, batch.scales[1].shape, generator=batch.g).float()
    else:
        batch.pages[1][::2] *= 2.0 ** 40
    q = batch.tensors(4)[0] * 30
    for scaling in (None, -0.1, 0.0, 1.0):
        got = paged_prefix_attention(q.cuda(), batch.cache(), *batch.index(), *index, scaling=scaling)
        check_prefix(batch, [(0, 3), (3, 4)], got, q, scaling)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_any_scales(dtype):
    """Scales that paged_append does not make: no powers of two, negative ones, zero."""
    from moba_amd import paged_prefix_attention
    batch = Batch([300, 340, 390], [1, 3, 70], 16, 2, 128, dtype, True, seed=7)
    index = share(batch, [(0, 3)], [256])
    for s in batch.scales:
        s *= torch.rand(s.shape, generator=batch.g) + 0.5
        s[::5] *= -1
        s[3::7] = 0
    q, = batch.tensors(8)
    for scaling in (None, -0.05):
        got = paged_prefix_attention(q.cuda(), batch.cache(), *batch.index(), *index, scaling=scaling)
        check_prefix(batch, [(0, 3)], got, q, scaling)


@pytest.mark.parametrize("d,dtype,quantized", [(64, BF16, True), (64, FP16, False), (128, FP16, True), (128, BF16, False)])
@pytest.mark.parametrize("members,new,heads", [(9, 4, 1), (33, 1, 1), (16, 1, 4), (100, 1, 2), (70, 3, 1), (130, 2, 2)])
def test_members(members, new, heads, d, dtype, quantized):
    """Groups of few and of more sequences than a wave has lanes, some without new tokens; rows around those that a workgroup takes."""
    from moba_amd import paged_prefix_attention
    count = [0 if i % 7 == 3 else new for i in range(members)]
    batch = Batch([192 + 5 * (i % 9) for i in range(members)] + [30], count + [1], 16, 1, d, dtype, quantized, seed=members + d)
    index = share(batch, [(0, members)], [192])
    q, = batch.tensors(heads)
    check_prefix(batch, [(0, members)], paged_prefix_attention(q.cuda(), batch.cache(), *batch.index(), *index), q)


def test_a_cache_of_more_than_2_31_elements():
    from moba_amd import PagedKVCache, paged_prefix_attention
    E4M3 = torch.float8_e4m3fn
    pages = 2 ** 31 // (8 * 256 * 128) + 2
    zeros = lambda: torch.zeros((pages, 8, 256, 128), dtype=E4M3, device="cuda")  # noqa: E731
    cache = PagedKVCache(zeros(), zeros(), *(torch.ones((pages, 8), device="cuda") for _ in range(2)))
    for i, page in enumerate((pages - 1, 0, pages - 2)):
        cache.v_pages[page] = torch.full((8, 256, 128), 2.0 + 2 * i, device="cuda").to(E4M3)
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    q = torch.ones((2, 8, 128), dtype=BF16, device="cuda")
    got = paged_prefix_attention(q, cache, ints(pages - 1, 0, pages - 1, pages - 2).view(2, 2), ints(512, 512), ints(0, 1, 2), ints(0, 2), ints(256))
    assert (got[0] == 3).all() and (got[1] == 4).all()


def test_views_and_nothing():
    from moba_amd import paged_prefix_attention
    batch = Batch([100, 130], [1, 4], 16, 2, 128, BF16, True, seed=6)
    index = share(batch, [(0, 2)], [96])
    q = batch.tensors(6)[0].cuda()
    cache, (table, lengths, cu) = batch.cache(), batch.index()
    want = paged_prefix_attention(q, cache, table, lengths, cu, *index)
    odd = torch.empty(q.numel() + 1, dtype=BF16, device="cuda")[1:].view_as(q).copy_(q)
    for view in (torch.cat([q, q[:, :2]], 1)[:, :6], q.transpose(0, 1).contiguous().transpose(0, 1), torch.stack([q, q], -1)[..., 0], odd):
        assert torch.equal(paged_prefix_attention(view, cache, table, lengths, cu, *index), want)
    wide = torch.full((2, 2 * table.shape[1]), -1, dtype=torch.int32, device="cuda")
    wide[:, ::2] = table
    assert torch.equal(paged_prefix_attention(q, cache, wide[:, ::2], lengths, cu, *index), want)
    spread = torch.stack([index[0], index[0]], 1)[:, 0]
    assert torch.equal(paged_prefix_attention(q, cache, table, lengths, cu, spread, index[1]), want)
    assert paged_prefix_attention(q[:0], cache, table, lengths, cu, *index).shape == (0, 6, 128)


def test_graph_and_streams():
    """A captured call follows the index tensors, the groups among them; another call at the same time on another stream."""
    from moba_amd import paged_prefix_attention
    batch = Batch([1000, 1050, 1063, 400], [1, 1, 1, 1], 64, 2, 128, BF16, True, seed=8)
    groups, shared = share(batch, [(0, 3), (3, 4)], [960, 320])
    other = Batch([3000, 3005], [20, 20], 64, 2, 128, BF16, True, seed=9)
    o_index = share(other, [(0, 2)], [2048])
    q, oq = batch.tensors(8)[0].cuda(), other.tensors(8)[0].cuda()
    cache, (table, lengths, cu) = batch.cache(), batch.index()
    o_args = (oq, other.cache(), *other.index(), *o_index)
    want_other = paged_prefix_attention(*o_args)
    torch.cuda.synchronize()
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged_prefix_attention(q, cache, table, lengths, cu, groups, shared)
    with torch.cuda.graph(second):
        out_other = paged_prefix_attention(*o_args)
    side = torch.cuda.Stream()
    for i, (lens, rows, cut, front) in enumerate((([1001, 1051, 1064, 401], [0, 1, 2, 3, 4], [0, 3, 4], [960, 320]),
                                                  ([1001, 970, 1064, 2], [0, 1, 2, 3, 4], [0, 2, 2], [960, 0]),
                                                  ([1001, 1051, 0, 401], [0, 2, 3, 3, 4], [0, 3, 4], [64, 64]),
                                                  ([300, 300, 300, 300], [0, 0, 0, 4, 4], [1, 4, 4], [256, 64]))):
        lengths.copy_(torch.tensor(lens))
        cu.copy_(torch.tensor(rows))
        groups.copy_(torch.tensor(cut))
        shared.copy_(torch.tensor(front))
        torch.cuda.synchronize()
        side.wait_stream(torch.cuda.current_stream())
        graph.replay()
        with torch.cuda.stream(side):
            second.replay()
            eager_other = paged_prefix_attention(*o_args)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        assert torch.equal(out, paged_prefix_attention(q, cache, table, lengths, cu, groups, shared)), i
        assert torch.equal(out_other, want_other) and torch.equal(eager_other, want_other), i
