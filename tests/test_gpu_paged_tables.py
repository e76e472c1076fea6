"""paged_reserve and paged_release on the GPU against a plain loop over the sequences."""

import random

import pytest
import torch

from serving_reference import released, reserved

pytestmark = pytest.mark.gpu


def ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def pool_of(free, count, page):
    from moba_amd import PagePool
    return PagePool(ints(free), ints([count]), page)


def case(sequences, wide, page, pages, seed, most=None):
    """(free, count, table, lengths, new, keep): sequences that hold some pages of a shuffled pool."""
    rng = random.Random(seed)
    ids = list(range(pages))
    rng.shuffle(ids)
    table, lengths = [[-1] * wide for _ in range(sequences)], []
    for row in table:
        length = rng.choice((0, 1, page - 1, page, page + 1, rng.randint(0, wide * page)))
        length = min(length, wide * page, len(ids) // 2 * page)
        for i in range(-(-length // page)):
            row[i] = ids.pop()
        lengths.append(length)
    new = [rng.choice((0, 1, 1, 1, 5, page, rng.randint(0, most or 2 * page))) for _ in range(sequences)]
    keep = [rng.choice((0, n, n, n + 3, rng.randint(0, n))) for n in lengths]
    return ids + [0] * (pages - len(ids)), len(ids), table, lengths, new, keep


def check_reserve(free, count, table, lengths, new, rows, page, view=lambda t: t):
    from moba_amd import paged_reserve
    pool, t, n = pool_of(free, count, page), view(ints(table)), ints(lengths)
    got = paged_reserve(pool, t, n, ints(new), rows)
    want = reserved(free, count, table, lengths, new, rows, page)
    assert [x.dtype for x in got] == [torch.int32] * 3 + [torch.int64]
    for name, g, w in zip(("count", "table", "lengths", "cu_new", "owners", "positions", "slots"), (pool.free_count[0], t, n, *got), want):
        assert torch.equal(g.cpu().long(), torch.tensor(w, dtype=torch.long).view(g.shape)), name
    assert pool.free_pages.tolist() == free
    return pool, t, n


def check_release(free, count, table, lengths, keep, page, view=lambda t: t):
    from moba_amd import paged_release
    pool, t, n = pool_of(free, count, page), view(ints(table)), ints(lengths)
    assert paged_release(pool, t, n, ints(keep)) is None
    want = released(free, count, table, lengths, keep, page)
    for name, g, w in zip(("free", "count", "table", "lengths"), (pool.free_pages, pool.free_count[0], t, n), want):
        assert torch.equal(g.cpu().long(), torch.tensor(w, dtype=torch.long).view(g.shape)), name


@pytest.mark.parametrize("sequences,wide,page,pages", [(1, 1, 16, 1), (1, 40, 64, 50), (7, 9, 16, 40), (64, 12, 32, 600), (63, 30, 256, 700),
                                                       (1023, 4, 16, 3000), (1025, 3, 128, 2000), (2500, 5, 64, 6000), (8192, 2, 16, 12000)])
def test_tables(sequences, wide, page, pages):
    for seed in range(3):
        free, count, table, lengths, new, keep = case(sequences, wide, page, pages, seed)
        print("tables", sequences, wide, page, pages, seed, flush=True)
        enough = sum(new)
        for rows in (enough + 5, enough // 2, 0):
            check_reserve(free, count, table, lengths, new, rows, page)
        check_reserve(free, count // 3, table, lengths, new, enough, page)      # fewer pages than are wanted
        check_reserve(free, 0, table, lengths, new, enough, page)
        check_release(free, count, table, lengths, keep, page)
        check_release(free, count, table, lengths, [0] * sequences, page)


def test_long_prompts():
    """More rows than the first launch places, more pages than it has threads."""
    free, count, table, lengths, _, _ = case(3, 9000, 16, 30000, 5)
    lengths, table = [0, 77, 0], [[-1] * 9000, [7, 8, 9, 10, 11] + [-1] * 8995, [-1] * 9000]
    new = [50000, 4096, 20001]
    check_reserve(free, count, table, lengths, new, sum(new) + 3, 16)
    check_reserve(free, 1200, table, lengths, new, sum(new), 16)
    check_reserve(free, count, table, lengths, [1, 2, 4094], 4097, 16)
    check_reserve(free, count, table, lengths, [1, 2, 8190], 8193, 16)
    check_reserve(free, count, table, lengths, [1, 2, 8189], 8192, 16)
    for row in table:
        row[:5000] = random.Random(1).sample(range(30000), 5000)
    check_release(free, 20000, table, [80000, 77, 31999], [17, 80, 0], 16)


@pytest.mark.parametrize("lengths,keep", [([144000, 143999, 144000], [0, 0, 0]), ([144000, 0, 9, 130000], [17, 0, 0, 16]), ([16] * 5000 + [100000], [0] * 5001),
                                          ([1, 0, 33] * 2000 + [100000], [0, 0, 17] * 2000 + [99])])
def test_many_pages_back(lengths, keep):
    """More than one step takes, of long sequences, of many short ones, and of both; some entries name no page."""
    rng = random.Random(len(lengths))
    wide = max(-(-n // 16) for n in lengths)
    held = [-(-n // 16) for n in lengths]
    ids = rng.sample(range(30000), sum(held))
    table = []
    for n in held:
        row = [ids.pop() if rng.random() < 0.9 else rng.choice((-1, 30000, 2 ** 31 - 1, -2 ** 31)) for _ in range(n)]
        table.append(row + [-1] * (wide - n))
    check_release([5] * 30000, 100, table, lengths, keep, 16)
    check_release([5] * 30000, 29000, table, lengths, keep, 16)


def test_no_rows():
    """Without rows nobody gets tokens; sequences that want none are as they were."""
    check_reserve([3, 2, 1, 0], 4, [[-1, -1], [9, -1]], [0, 16], [1, 0], 0, 16)
    check_reserve([3, 2, 1, 0], 4, [[-1, -1], [9, -1]], [0, 16], [0, 0], 0, 16)


def test_a_captured_prompt():
    """Many rows: the second launch's workspace is the graph's own."""
    from moba_amd import paged_release, paged_reserve
    free, count, table, lengths, _, _ = case(3, 1000, 16, 2500, 5)
    pool, t, n, wanted = pool_of(free, count, 16), ints(table), ints(lengths), ints([0, 0, 0])
    kept = n.clone()
    paged_reserve(pool_of(free, count, 16), t.clone(), n.clone(), wanted, 9000)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged_reserve(pool, t, n, wanted, 9000)
        full = t.clone()
        paged_release(pool, t, n, kept)
    for new in ([5000, 16, 3000], [0, 0, 0], [1, 9000, 1], [4095, 2, 0]):
        wanted.copy_(torch.tensor(new))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        _, after, _, *want = reserved(free, count, table, lengths, new, 9000, 16)
        assert all(x.tolist() == w for x, w in zip(out, want)) and full.tolist() == after, new
        assert t.tolist() == table and n.tolist() == lengths and pool.free_count.tolist() == [count], new


def test_what_does_not_fit():
    free = list(range(20))
    row = [3, -1, 99, 4]
    # beyond the table's row; by more than 31 bits; negative lengths and numbers
    for lengths, new in (([64], [1]), ([60], [5]), ([1], [2 ** 31 - 1]), ([2 ** 31 - 1], [2 ** 31 - 1]), ([-5], [3]), ([2], [-9]),
                         ([10 ** 6], [0]), ([10 ** 6], [1]), ([17], [10]), ([33], [3])):
        check_reserve(free, 20, [row], lengths, new, 70, 16)
    # counts that are none
    for count in (-3, 21, 2 ** 31 - 1):
        check_reserve(free, count, [row] * 2, [16, 5], [20, 20], 40, 16)
        check_release(free, count, [row], [60], [5], 16)
    # entries that name no page, lengths beyond the row, more pages than the pool has places
    check_release(free, 3, [row, [1, 2, 5, 6]], [10 ** 6, 2 ** 31 - 1], [0, 17], 16)
    check_release(free, 18, [[1, 2, 5, 6]], [64], [0], 16)
    check_release(free, 3, [row], [-4], [3], 16)
    check_release(free, 3, [row], [40], [-4], 16)
    check_reserve(free, 20, [[-1] * 4, [-1] * 4, [-1] * 4], [0, 0, 0], [70, 17, 64], 81, 16)


def test_taken_back():
    """A release that undoes a reserve leaves everything as it was; and the pages come out again in the same order."""
    from moba_amd import paged_release, paged_reserve
    free, count, table, lengths, new, _ = case(40, 20, 32, 500, 9)
    pool, t, n, wanted = pool_of(free, count, 32), ints(table), ints(lengths), ints(new)
    before = [x.clone() for x in (pool.free_pages, pool.free_count, t, n)]
    first = [x.clone() for x in (*paged_reserve(pool, t, n, wanted, sum(new)), t)]
    paged_release(pool, t, n, before[3])
    assert all(torch.equal(a, b) for a, b in zip(before, (pool.free_pages, pool.free_count, t, n)))
    again = [*paged_reserve(pool, t, n, wanted, sum(new)), t]
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_views():
    from moba_amd import PagePool, paged_release, paged_reserve
    free, count, table, lengths, new, keep = case(9, 6, 16, 60, 11)
    wide = lambda t: torch.cat([t, t], 1)[:, :6]  # noqa: E731
    check_reserve(free, count, table, lengths, new, sum(new), 16, wide)
    check_release(free, count, table, lengths, keep, 16, wide)
    pool, t, n = pool_of(free, count, 16), ints(table), ints(lengths)
    spread = ints([x for v in new for x in (v, 99)])[::2]
    got = paged_reserve(pool, t, n, spread, sum(new))
    assert got[0].tolist() == reserved(free, count, table, lengths, new, sum(new), 16)[3]
    for wrong in (ints(table).T.contiguous().T, ints(table)[:1].expand(9, -1)):
        with pytest.raises(ValueError):
            paged_reserve(pool, wrong, n, spread, 5)
        with pytest.raises(ValueError):
            paged_release(pool, wrong, n, spread)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    cu, owners, positions, slots = paged_reserve(pool, none.view(0, 3), none, none, 4)
    assert cu.tolist() == [0] and owners.tolist() == [-1] * 4 and positions.tolist() == [0] * 4 and slots.tolist() == [-1] * 4
    paged_release(pool, none.view(0, 3), none, none)
    full = PagePool.full(5, 16)
    one = ints([[-1] * 4])
    paged_reserve(full, one, ints([0]), ints([40]), 40)
    assert one.tolist() == [[0, 1, 2, -1]] and full.free_count.tolist() == [2]


def test_graph_and_streams():
    """A captured step goes on from what the replays before have left; another pool at the same time on another stream."""
    from moba_amd import paged_release, paged_reserve
    free, count, table, lengths, _, _ = case(30, 40, 16, 2000, 3)
    pool, t, n, wanted, kept = pool_of(free, count, 16), ints(table), ints(lengths), ints([3] * 30), ints([0] * 30)
    state = (free, count, table, lengths)
    paged_reserve(pool_of(free, count, 16), t.clone(), n.clone(), wanted, 100)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged_reserve(pool, t, n, wanted, 100)
        kept.copy_(n - wanted.clamp(max=2))
        paged_release(pool, t, n, kept)
    side, rng = torch.cuda.Stream(), random.Random(8)
    for i in range(6):
        new = [rng.randint(0, 6) for _ in range(30)]
        wanted.copy_(torch.tensor(new))
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            check_reserve(*case(12, 9, 32, 90, i)[:5], 60, 32)
        torch.cuda.synchronize()
        free, count, table, lengths = state
        count, table, lengths, *want = reserved(free, count, table, lengths, new, 100, 16)
        state = released(free, count, table, lengths, [a - min(b, 2) for a, b in zip(lengths, new)], 16)
        assert all(x.tolist() == w for x, w in zip(out, want)), i
        assert pool.free_pages.tolist() == state[0] and pool.free_count.tolist() == [state[1]]
        assert t.tolist() == state[2] and n.tolist() == state[3], i
