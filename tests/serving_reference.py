"""The operators of serving in 64 bits or whole numbers on the CPU, written as plainly as they read, for the tests."""

import torch

from paged_reference import attended


# ---- tables
def pages_of(tokens, page):
    return -(-tokens // page)


def reserved(free, count, table, lengths, new, rows, page):
    """What paged_reserve leaves and returns, from lists: (count, table, lengths, cu_new, owners, positions, slots)."""
    table, lengths, cu, owners, positions, slots = [list(r) for r in table], list(lengths), [0], [], [], []
    pool, top = len(free), min(max(count, 0), len(free))
    count, tokens, pages = top, 0, 0
    for b, n in enumerate(new):
        old, n = max(lengths[b], 0), max(n, 0)
        if old + n > min(len(table[b]) * page, 2 ** 31 - 1):
            n = 0
        need = pages_of(old + n, page) - pages_of(old, page)
        tokens, pages = tokens + n, pages + need
        if tokens > rows or (need and pages > top):
            n = need = 0
        for i in range(need):
            count -= 1
            table[b][pages_of(old, page) + i] = free[count]
        if n:
            lengths[b] = old + n
        for at in range(old, old + n):
            id = table[b][at // page]
            owners.append(b)
            positions.append(at)
            slots.append(id * page + at % page if 0 <= id < pool else -1)
        cu.append(cu[-1] + n)
    behind = rows - len(owners)
    return count, table, lengths, cu, owners + [-1] * behind, positions + [0] * behind, slots + [-1] * behind


def released(free, count, table, lengths, keep, page):
    """What paged_release leaves: (free, count, table, lengths)."""
    free, table, lengths, back = list(free), [list(r) for r in table], list(lengths), []
    for b, k in enumerate(keep):
        old = max(lengths[b], 0)
        kept = min(max(k, 0), old)
        for i in range(min(pages_of(kept, page), len(table[b])), min(pages_of(old, page), len(table[b]))):
            if 0 <= table[b][i] < len(free):
                back.append(table[b][i])
            table[b][i] = -1
        if kept < old:
            lengths[b] = kept
    count = min(max(count, 0), len(free))
    for id in reversed(back):
        if count < len(free):
            free[count] = id
            count += 1
    return free, count, table, lengths


# ---- attention
def check_against(got, want, slack, dtype):
    """got within half a step of its type and `slack` of want; where want is not finite, the same."""
    got = got.cpu()
    assert got.dtype == dtype and got.shape == want.shape
    assert torch.equal(got.isnan(), want.isnan()), (got.isnan().sum(), want.isnan().sum())
    fine = want.isfinite()
    assert torch.equal(got[~fine & ~want.isnan()].double(), want[~fine & ~want.isnan()])
    bound = torch.finfo(dtype).eps / 2 * 1.001 * want.abs() + slack + 2.0 ** -25
    off = (got.double() - want).abs()
    bad = fine & ~(off <= bound)
    assert not bad.any(), (bad.nonzero()[:5].tolist(), (off / bound)[fine].max().item())


def check_prefix(batch, groups, got, query, scaling=None):
    """paged_prefix_attention against the attention of the sequences one by one.  Half a step of a probability (of values with odd
    scales too: 2^-8) times the largest value more where a group has so many rows that the shared keys are attended in the precision
    of many rows; see paged_reference.attended."""
    want, slack = attended(batch, query, scaling)
    rep = query.shape[1] // batch.pages[0].shape[1]
    starts = [sum(batch.new[:b]) for b in range(len(batch.new) + 1)]
    largest = 0.0
    for half in [batch.pages[1]]:
        x = half.double() if batch.scales[1] is None else half.double() * batch.scales[1][:, :, None, None].double()
        largest = x.where(x.isfinite(), 0).abs().max()
    for first, end in groups:
        rows = starts[end] - starts[first]
        if rows * rep > (64 if batch.quantized else 32):
            part = 0.0 if batch.quantized and query.dtype == torch.float16 else torch.finfo(query.dtype).eps / 2
            if batch.quantized and not bool((torch.frexp(batch.scales[1])[0] == 0.5).all()):
                part += 2.0 ** -8
            slack[starts[first]:starts[end]] += part * largest
    check_against(got, want, slack, query.dtype)


def held(batch, b, length):
    """(there [length], k, v [length, kv heads, d] in 64 bits) of sequence b's tokens, whose pages the table may name wrongly."""
    table = batch.table[b]
    pages = [int(table[i]) if i < table.shape[0] else -1 for i in range(-(-length // batch.page))]
    good = [0 <= p < batch.pages[0].shape[0] for p in pages]
    there = torch.tensor(good, dtype=torch.bool).repeat_interleave(batch.page)[:length]
    ids = torch.tensor([p if g else 0 for p, g in zip(pages, good)], dtype=torch.long)
    kv = []
    for half in range(2):
        x = batch.pages[half][ids].double()
        if batch.quantized:
            x = x * batch.scales[half][ids][:, :, None, None].double()
        kv.append(x.transpose(1, 2).reshape(-1, x.shape[1], x.shape[3])[:length])
    return there, *kv


def chosen_attended(batch, query, blocks, block_size, scaling=None):
    """[rows, heads, d] in 64 bits: every new token and head against its blocks up to itself; and how far a result may be off, as in
    paged_reference.attended for few rows."""
    d, hkv = query.shape[2], batch.pages[0].shape[1]
    rep = query.shape[1] // hkv
    scale = d ** -0.5 if scaling is None else scaling
    out, slack, row = torch.zeros(query.shape, dtype=torch.float64), torch.zeros((*query.shape[:2], 1), dtype=torch.float64), 0
    for b, (o, c) in enumerate(zip(batch.old, batch.new)):
        if c:
            there, k, v = held(batch, b, o + c)
            own = torch.arange(o + c) // block_size
        for j in range(c):
            for h in range(query.shape[1]):
                mine = torch.zeros(o + c, dtype=torch.bool)
                for x in set(blocks[row + j, h].tolist()):
                    mine |= own == x
                seen = mine & there & (torch.arange(o + c) <= o + j)
                if not seen.any():
                    continue
                kk, vv, q = k[seen, h // rep], v[seen, h // rep], query[row + j, h].double()
                out[row + j, h] = torch.softmax((kk * q).sum(-1) * scale, 0) @ vv
                size = abs(scale) * q.norm() * kk.norm(dim=-1).amax()
                slack[row + j, h] = (2 * (d + 12) * 2.0 ** -24 * size + 2.0 ** -15) * vv.where(vv.isfinite(), 0).abs().amax()
        row += c
    return out, slack


def check_chosen(batch, got, query, blocks, block_size, scaling=None):
    check_against(got, *chosen_attended(batch, query, blocks, block_size, scaling), query.dtype)


# ---- sums and selection
def key_sums(batch):
    """{page: (sum, bound) of [kv heads, d]} in 64 bits of the pages that have received new tokens; bound: 2^-24 for each of the
    additions that one number passes through, of the sum of magnitudes."""
    out = {}
    for b, (o, c) in enumerate(zip(batch.old, batch.new)):
        for i in range(o // batch.page, pages_of(o + c, batch.page) if c else 0):
            id = int(batch.table[b, i]) if i < batch.table.shape[1] else -1
            if not 0 <= id < batch.pages[0].shape[0]:
                continue
            x = batch.pages[0][id, :, :o + c - i * batch.page].double()
            if batch.quantized:
                x = x * batch.scales[0][id][:, None, None].double()
            out[id] = (x.sum(1), (batch.page + 2) * 2.0 ** -24 * x.abs().sum(1))
    return out


def selected(query, sums, table, lengths, cu, page, block_size, topk):
    """[rows, heads, topk]: Python's exact fractions decide where two blocks' products are near."""
    from fractions import Fraction
    out = torch.full((*query.shape[:2], topk), -1, dtype=torch.int32)
    each, rep, wide = block_size // page, query.shape[1] // sums.shape[1], table.shape[1]
    count = -(-wide // each)
    rows = query.shape[0]
    clamp = lambda x, lo, hi: min(max(x, lo), hi)  # noqa: E731
    for b in range(len(lengths)):
        lo = clamp(int(cu[b]), 0, rows)
        hi = clamp(int(cu[b + 1]), lo, rows)
        total = None
        for t in range(lo, hi):
            at = max(int(lengths[b]), 0) - hi + t
            if at < 0:
                continue
            own = at // block_size
            history = min(own, count)
            if total is None:
                grid = torch.zeros((count, sums.shape[1], sums.shape[2]), dtype=torch.float64)
                for j in range(count):
                    for i in range(j * each, min((j + 1) * each, wide)):
                        id = int(table[b, i])
                        if 0 <= id < sums.shape[0]:
                            grid[j] += sums[id].double()
                total = grid
            for h in range(query.shape[1]):
                s = (total[:history, h // rep] * query[t, h].double()).sum(-1)
                s = torch.where(s.isnan(), float("-inf"), s)
                order = sorted(range(history), key=lambda j: (-s[j].item(), j))
                k = min(topk - 1, history)
                if 0 < k < history and s[order[k - 1]].isfinite() and s[order[k]].isfinite():
                    gap = (s[order[k - 1]] - s[order[k]]).item()
                    size = (total[order[k - 1], h // rep].abs() * query[t, h].double().abs()).sum().item()
                    if gap < 2.0 ** -40 * size:     # (the order of the sums could decide)
                        exact = {j: sum(Fraction(x) * Fraction(y) for x, y in zip(total[j, h // rep].tolist(), query[t, h].double().tolist()))
                                 for j in order}
                        order = sorted(range(history), key=lambda j: (-exact[j], j))
                picks = sorted(order[:k]) + ([own] if own < count else [])
                out[t, h, :len(picks)] = torch.tensor(picks, dtype=torch.int32)
    return out
