"""The operators of serving from the paged cache, as cases whose time and results can be compared with a plain form.

Five operators, each through the package's public entry points:

  reserve  ``paged_reserve`` and ``paged_release``: pages for new tokens, and where each of these belongs, from the sequences' lengths;
           and the way back (drafted tokens that were rejected, requests that end)
  prefix   ``paged_prefix_attention``: new tokens of sequences that begin with the same pages, which are read once for all of them
  sums     ``paged_key_sums``: the sum of the keys of every page that has received tokens
  select   ``paged_select_blocks``: of every new token and head the blocks with the largest products with the sum of their keys,
           and the token's own
  blocks   ``paged_block_attention``: every new token and head against the keys of its blocks only

With ``own`` false everything is computed from elementary torch operations in 32 bits (the selection's scores in 64: a block
next to the border is in or out) and rounded once.
"""

import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_E4M3 = torch.float8_e4m3fn
_PLAIN_BYTES = 16e9    # that a plain form may lay out


def _reserve(name, **kw):
    base = dict(name=name, op="reserve", page=64, wide=2048, spare=1024, old="0", new="1", pad=0)
    base.update(kw)
    return base


def _cached(name, op, **kw):
    base = dict(name=name, op=op, heads=32, kv_heads=8, head_dim=128, dtype="bf16", cache="e4m3", page=64, old="0", new="1")
    base.update(kw)
    return base


def _prefix(name, **kw):
    """groups: sequences of each; shared: tokens that a group's sequences begin with, in front of `old`."""
    return _cached(name, "prefix", **{"groups": "1", "shared": "0", **kw})


def _sums(name, **kw):
    return _cached(name, "sums", **kw)


def _select(name, **kw):
    return _cached(name, "select", **{"block": 4096, "topk": 12, **kw})


def _blocks(name, **kw):
    return _cached(name, "blocks", **{"block": 4096, "topk": 12, **kw})


_USERS = "8191,1,4095,700,63,64,2000,5003,127,1024,0,3579,900,31,6001,400"
_LONG_USERS = "65000,131,16000,7000,630,64000,2000,5003,127,10240,0,35790,900,31,24001,400"


def listed():
    return [
        # a step of 64 users with five drafted tokens each, all of which are rejected: latency counts
        _reserve("reserve_drafts", old=",".join([_USERS] * 4), new=",".join(["5"] * 64), pad=16),
        # eight long documents come in, one of them too many for the pool, and go again; small pages
        _reserve("reserve_documents", page=16, wide=8192, spare=30000, old="0,0,77,0,0,4090,0,0",
                 new="131072,29343,53769,62439,31658,66749,120000,7602"),
        # sixteen users of one assistant, whose instructions and examples are 32K tokens; one token each
        _prefix("prefix_tokens", groups="16", shared="32768", old=_USERS, new=",".join(["1"] * 16)),
        # five drafted tokens of four users behind a prompt that is no whole number of tiles, fp16, 16-bit pages of 16 tokens
        _prefix("prefix_few", groups="4", shared="8208", old="700,0,63,2000", new="5,5,3,5", dtype="fp16", cache="same", page=16,
                head_dim=64),
        # two applications in one batch: pieces of prompts behind 12K tokens, single tokens behind 4K and, of one user, alone
        _prefix("prefix_groups", groups="4,8,1", shared="12288,4096,0", old="0,0,512,0,0,97,1067,31,500,820,64,1,4000",
                new="200,300,301,97,1,1,1,1,1,1,1,1,60"),
        # a decoding step of sixteen users
        _sums("sums_tokens", old=_USERS, new=",".join(["1"] * 16)),
        # the headline prompt has just gone into the cache
        _sums("sums_prompt_128k", new="131072"),
        # the headline configuration's blocks of 4096 tokens, 12 of them, for the next token behind 128K ...
        _select("select_token_128k", old="131071"),
        # ... and small blocks for five drafted tokens of sixteen users, fp16
        _select("select_drafts", old=_LONG_USERS, new=",".join(["5"] * 16), block=512, topk=16, dtype="fp16"),
        # the attention that goes with it: the headline configuration, ...
        _blocks("blocks_token_128k", old="131071"),
        # ... a batch of sixteen users, fp16, small blocks ...
        _blocks("blocks_tokens", old=_LONG_USERS, new=",".join(["1"] * 16), block=512, topk=16, dtype="fp16"),
        # ... and drafted tokens, 16-bit pages
        _blocks("blocks_few", old="20000,19000,20480,12345", new="5,5,5,5", block=256, topk=8, cache="same"),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def _join(values):
    return ",".join(str(v) for v in values)


def _ints(text):
    return [int(v) for v in text.split(",")]


def _draw_once(rng):
    op = rng.choice(("reserve", "prefix", "prefix", "sums", "select", "blocks", "blocks"))
    page = rng.choice((16, 32, 64, 64, 128))
    if op == "reserve":
        batch, most = _log_int(rng, 1, 512), _log_int(rng, 1, 32768)
        old = [rng.randint(0, _log_int(rng, 10, 32768)) for _ in range(batch)]
        new = [rng.randint(0, most) for _ in range(batch)]
        need = sum(-(-(o + n) // page) + -o // page for o, n in zip(old, new))
        wide = -(-max(o + n for o, n in zip(old, new)) // page)
        return _reserve("", page=page, wide=max(1, wide + rng.choice((5, 5, -wide // 8))), spare=max(1, int(need * rng.choice((1, 1.5, 0.6)))),
                        old=_join(old), new=_join(new), pad=rng.choice((0, 7)))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    kv = rng.choice((1, 2, 4, 8))
    head_dim = rng.choice((64, 128, 128, 128))
    common = dict(kv_heads=kv, heads=kv * rng.choice((1, 2, 4, 5, 8)), head_dim=head_dim, dtype=dtype, page=page,
                  cache=rng.choice(("e4m3", "e4m3", "same")))
    kind = rng.choice(("token", "token", "few", "many"))
    batch = _log_int(rng, 1, 64) if kind == "token" else _log_int(rng, 1, 16) if kind == "few" else rng.randint(1, 4)
    most = _log_int(rng, 50, 4000 if op == "prefix" else 131072)
    old = [int(most * (1 - 0.9 * rng.random() ** 2)) if rng.random() < 0.9 else 0 for _ in range(batch)]
    piece = _log_int(rng, 10, 131072 if op == "sums" else 700 if op == "prefix" else 64)
    new = [1 if kind == "token" else rng.randint(0, 9 if kind == "few" else piece) for _ in range(batch)]
    new[rng.randrange(batch)] = 1 if kind == "token" else rng.randint(2, 9) if kind == "few" else piece
    common.update(old=_join(old), new=_join(new))
    if op == "sums":
        return _sums("", **common)
    if op == "prefix":
        groups = []
        while sum(groups) < batch:
            groups.append(min(rng.choice((1, 3, 16, 64)), batch - sum(groups)))
        return _prefix("", groups=_join(groups), shared=_join(_log_int(rng, 30, 65536) // page * page for _ in groups), **common)
    block = page * rng.choice((1, 2, 3, 4, 8, 32))
    return (_select if op == "select" else _blocks)("", block=block, topk=rng.randint(1, 24), **common)


def _totals(case):
    """Tokens of every sequence after the call, and those of them that its group shares."""
    front = [s for n, s in zip(_ints(case["groups"]), _ints(case["shared"])) for _ in range(n)] if case["op"] == "prefix" else [0] * 10000
    return [f + o + n for f, o, n in zip(front, _ints(case["old"]), _ints(case["new"]))], front


def _plain_bytes(case):
    if case["op"] == "reserve":
        return 40.0 * len(_ints(case["old"])) * case["wide"]
    total, new = _totals(case)[0], _ints(case["new"])
    if case["op"] in ("prefix", "select"):
        keys = len(total) * (max(total) if case["op"] == "prefix" else 2 * max(total) / case["page"])
        return keys * (8.0 * case["kv_heads"] * case["head_dim"] + 8.0 * case["heads"] * max(new))
    return 8.0 * sum(new) * case["heads"] * case["head_dim"] * case["topk"] * case["block"] if case["op"] == "blocks" else 0.0


def draw(rng):
    """One more case of the same ranges: no dearer than the dearest listed one of its kind, in operations and in bytes, and no
    larger than a plain form can lay out."""
    most = {}
    for c in listed():
        w, m = work(c), most.setdefault(c["op"], {"bytes": 0.0, "flops": 0.0})
        most[c["op"]] = {x: max(m[x], w[x]) for x in m}
    while True:
        case = _draw_once(rng)
        need = work(case)
        if all(need[x] <= most[case["op"]][x] for x in need) and _plain_bytes(case) <= _PLAIN_BYTES and sum(_ints(case["new"])):
            del case["name"]
            return case


def _history(case):
    """Of every new token: the number of whole blocks in front of its own."""
    return [(o + i) // case["block"] for o, n in zip(_ints(case["old"]), _ints(case["new"])) for i in range(n)]


def work(case):
    """What a pass cannot do without: inputs read once, outputs written once."""
    old, new, page = _ints(case["old"]), _ints(case["new"]), case["page"]
    if case["op"] == "reserve":
        need = sum(-(-(o + n) // page) + -o // page for o, n in zip(old, new))
        return {"bytes": 16.0 * min(need, case["spare"]) + 16.0 * (sum(new) + case["pad"]) + 24.0 * len(old), "flops": 0.0}
    d, hq, hkv, width, tokens = case["head_dim"], case["heads"], case["kv_heads"], 1 if case["cache"] == "e4m3" else 2, sum(new)
    if case["op"] == "sums":
        pages = sum((o + n - 1) // page + 1 - o // page for o, n in zip(old, new) if n)
        held = sum(o + n - o // page * page for o, n in zip(old, new) if n)
        return {"bytes": held * hkv * d * width + 4.0 * pages * hkv * d, "flops": 1.0 * held * hkv * d}
    if case["op"] == "select":
        pages = sum((o + n - 1) // case["block"] * (case["block"] // page) for o, n in zip(old, new) if n)
        return {"bytes": 4.0 * pages * hkv * d + 2.0 * tokens * hq * d + 4.0 * tokens * hq * case["topk"],
                "flops": pages * hkv * d + 2.0 * d * hq * sum(_history(case))}
    if case["op"] == "blocks":
        keys = pairs = at = 0
        history = _history(case)
        for o, n in zip(old, new):
            for h in history[at:at + n][-1:]:     # every row takes its blocks from a pool of twice as many
                picks = min(case["topk"] - 1, h)
                pool = min(2 * picks, h)
                once = pool * (1 - (1 - picks / pool) ** (n * hq // hkv)) if pool else 0
                keys += once * case["block"] + o + n - h * case["block"]
            pairs += sum(min(case["topk"] - 1, h) * case["block"] + o + i + 1 - h * case["block"] for i, h in enumerate(history[at:at + n]))
            at += n
        return {"bytes": 2.0 * width * keys * hkv * d + 4.0 * tokens * hq * d + 4.0 * tokens * hq * case["topk"], "flops": 4.0 * d * hq * pairs}
    total, front = _totals(case)
    groups, at, keys = _ints(case["groups"]), 0, sum(t - f for t, f, n in zip(total, front, new) if n)
    for n, s in zip(groups, _ints(case["shared"])):
        keys += s if any(new[at:at + n]) else 0
        at += n
    pairs = sum(n * (t - n) + n * (n + 1) // 2 for t, n in zip(total, new))
    return {"bytes": 2.0 * width * keys * hkv * d + 4.0 * tokens * hq * d, "flops": 4.0 * d * hq * pairs}


# ------------------------------------------------------------------------------------------------------------ inputs
def _normal(g, shape, dtype):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _sums_upto(values):
    return [sum(values[:i]) for i in range(len(values) + 1)]


def _pages(g, case, count):
    """Pages of one of the cache's halves: (elements, scales or None), N(0, 1)."""
    shape = (count, case["kv_heads"], case["page"], case["head_dim"])
    x = torch.randn(shape, generator=g, device="cuda")
    if case["cache"] == "same":
        return x.to(_DTYPES[case["dtype"]]), None
    scales = torch.exp2(torch.ceil(torch.log2(x.abs().amax((2, 3)) / 448)))
    return (x / scales[:, :, None, None]).to(_E4M3), scales


def _prepare_reserve(case, seed):
    old, new, page, wide = _ints(case["old"]), _ints(case["new"]), case["page"], case["wide"]
    held = [min(-(-o // page), wide) for o in old]
    ids = list(range(sum(held) + case["spare"]))
    random.Random(seed).shuffle(ids)
    table = torch.full((len(old), wide), -1, dtype=torch.int32)
    for b, n in enumerate(held):
        table[b, :n] = torch.tensor(ids[len(ids) - n:], dtype=torch.int32)
        del ids[len(ids) - n:]
    free = torch.zeros(sum(held) + case["spare"], dtype=torch.int32)
    free[:len(ids)] = torch.tensor(ids, dtype=torch.int32)
    s = {"case": case, "page_table": table.cuda(), "lengths": _int32(old), "new": _int32(new), "keep": _int32(old),
         "free_pages": free.cuda(), "free_count": _int32([len(ids)]), "rows": sum(new) + case["pad"]}
    if own:
        from moba_amd import PagePool
        s["pool"] = PagePool(s["free_pages"], s["free_count"], page)
    return s


def prepare(case, seed):
    if case["op"] == "reserve":
        return _prepare_reserve(case, seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    dtype, d, hq, hkv, page = _DTYPES[case["dtype"]], case["head_dim"], case["heads"], case["kv_heads"], case["page"]
    old, new = _ints(case["old"]), _ints(case["new"])
    total, front = _totals(case)
    need = [-(-t // page) for t in total]
    ids = list(range(sum(need) + 3))
    rng.shuffle(ids)
    table = torch.full((len(need), max(1, max(need))), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(ids[at:at + n], dtype=torch.int32)
        at += n
    s = {"case": case, "lengths": _int32(total), "cu_new": _int32(_sums_upto(new)), "query": _normal(g, (sum(new), hq, d), dtype)}
    if case["op"] == "prefix":
        groups = _ints(case["groups"])
        s["cu_groups"], s["shared"] = _int32(_sums_upto(groups)), _int32(_ints(case["shared"]))
        for first, n in zip(_sums_upto(groups), groups):
            whole = front[first] // page
            table[first:first + n, :whole] = table[first, :whole].clone()
    s["page_table"] = table.cuda()
    if case["op"] == "select":
        s["sums"] = torch.randn((len(ids), hkv, d), generator=g, device="cuda") * page ** 0.5
        return s
    for half in ("k", "v"):
        s[half + "_pages"], s[half + "_scales"] = _pages(g, case, len(ids))
    if case["op"] == "sums":
        s["sums"] = torch.zeros((len(ids), hkv, d), device="cuda")
        # the pages that receive tokens, which whoever hands out pages knows, and how many tokens each of them holds
        hit = [(int(table[b, i]), min(page, total[b] - i * page)) for b in range(len(new)) if new[b]
               for i in range(old[b] // page, (total[b] - 1) // page + 1)]
        s["touched"], s["filled"] = (torch.tensor(x, device="cuda") for x in zip(*hit))
    if case["op"] == "blocks":
        s["blocks"] = _some_blocks(g, case, s)
    if own:
        from moba_amd import PagedKVCache
        s["cache"] = PagedKVCache(s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"])
    return s


def _some_blocks(g, case, s):
    """Of every token and head its own block and topk - 1 in front of it, ascending, -1 behind the last: from a pool of twice as
    many that its sequence and key/value head has."""
    hkv, rep, k = case["kv_heads"], case["heads"] // case["kv_heads"], case["topk"]
    b, at = _new_tokens(s)[1:]
    history = at // case["block"]
    wide = max(int(history.max()), k - 1, 1)
    order = torch.rand((s["lengths"].numel(), hkv, wide), generator=g, device="cuda")
    mark = torch.rand((at.numel(), hkv, rep, wide), generator=g, device="cuda")
    blk = torch.arange(wide, device="cuda")
    there = blk < history[:, None, None]
    rank = torch.where(there, order[b], 2.0).argsort(-1).argsort(-1)                     # (a token's history: by its own length)
    pool = there & (rank < 2 * torch.clamp(history, max=k - 1)[:, None, None])
    mark = torch.where(pool[:, :, None], mark, 2.0)
    chosen = (mark.argsort(-1).argsort(-1) < min(k - 1, wide)) & pool[:, :, None]
    picks = torch.where(chosen, blk, 1 << 30).sort(-1).values[..., :max(k - 1, 0)]
    picks = torch.cat((picks, history[:, None, None, None].expand(-1, hkv, rep, 1)), -1).sort(-1).values
    return torch.where(picks < 1 << 30, picks, -1).view(at.numel(), hkv * rep, k).int()


def _new_tokens(s):
    """Of every new token: its number, its sequence and its position there."""
    t = torch.arange(s["query"].shape[0], device="cuda")
    b = torch.searchsorted(s["cu_new"], t, right=True) - 1
    return t, b, s["lengths"][b].long() - s["cu_new"][b + 1] + t


# ------------------------------------------------------------------------------------------------------------ passes
def run(s):
    return {"reserve": _run_reserve, "prefix": _run_prefix, "sums": _run_sums, "select": _run_select, "blocks": _run_blocks}[s["case"]["op"]](s, s["case"])


def _run_reserve(s, case):
    held = [s["page_table"], s["lengths"], s["free_pages"], s["free_count"]]
    if own:
        from moba_amd import paged_release, paged_reserve
        step = paged_reserve(s["pool"], s["page_table"], s["lengths"], s["new"], s["rows"])
        paged_release(s["pool"], s["page_table"], s["lengths"], s["keep"])
        return [*step, *held]
    page, rows, table, free, count = case["page"], s["rows"], s["page_table"], s["free_pages"], s["free_count"]
    old, n, column = s["lengths"].long(), s["new"].long(), torch.arange(table.shape[1], device="cuda")
    # a sequence gets its pages if all of it fits: into its row of the table, with those before it into the rows, and the pool
    n = torch.where(old + n <= table.shape[1] * page, n, 0)
    have = (old + page - 1) // page
    need = (old + n + page - 1) // page - have
    served = (n.cumsum(0) <= rows) & ((need == 0) | (need.cumsum(0) <= count))
    n, need = n * served, need * served
    cu_new = torch.nn.functional.pad(n.cumsum(0), (1, 0)).int()
    number = column - have[:, None]
    fresh = (number >= 0) & (number < need[:, None])
    place = count - 1 - ((need.cumsum(0) - need)[:, None] + number)
    table.copy_(torch.where(fresh, free[place.clamp(0, free.numel() - 1)], table))
    count -= need.sum().int()
    s["lengths"] += n.int()
    t = torch.arange(rows, device="cuda")
    b = torch.searchsorted(cu_new, t, right=True) - 1
    live = t < cu_new[-1]
    b = torch.where(live, b, 0)
    at = torch.where(live, old[b] + t - cu_new[b], 0)
    slots = torch.where(live, table[b, at // page].long() * page + at % page, -1)
    step = [cu_new, torch.where(live, b, -1).int(), at.int(), slots]
    # ... and back: the last sequence's last page first, so that the first one's first is on top again
    kept = torch.minimum(s["keep"], s["lengths"])
    gone = (column >= ((kept + page - 1) // page)[:, None]) & (column < ((s["lengths"] + page - 1) // page)[:, None])
    total = gone.sum()
    place = torch.where(gone, count + total - gone.flatten().cumsum(0).view_as(gone), free.numel())
    wide = torch.cat((free, free[:1]))
    wide[place] = table
    free.copy_(wide[:-1])
    count += total.int()
    table.masked_fill_(gone, -1)
    s["lengths"].copy_(kept)
    return [*step, *held]


def _laid_out(s, half, ids, *rest):
    """Pages [ids] of a half of the cache in 32 bits; `rest`: heads that go with the ids, or all."""
    x = s[half + "_pages"][(ids, *rest)].float()
    return x if s[half + "_scales"] is None else x * s[half + "_scales"][(ids, *rest)][..., None, None]


def _padded_rows(s, case):
    """The query's rows by sequence, [batch, heads of a kv head's, longest, ...], and the rows' last visible key."""
    d, hq, hkv, longest = case["head_dim"], case["heads"], case["kv_heads"], max(_ints(case["new"]))
    begin, count = s["cu_new"][:-1, None], s["cu_new"].diff()[:, None]
    i = torch.arange(longest, device="cuda")
    q = s["query"][(begin + torch.minimum(i, count - 1).clamp(min=0)).clamp(max=s["query"].shape[0] - 1)]
    return q.reshape(-1, longest, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).flatten(2, 3), s["lengths"][:, None] - count + i


def _packed_rows(s, x):
    """[batch, kv heads, heads, longest, ...] as packed rows."""
    _, b, at = _new_tokens(s)
    return x.permute(0, 3, 1, 2, *range(4, x.dim()))[b, at - (s["lengths"] - s["cu_new"].diff())[b]].flatten(1, 2)


def _run_prefix(s, case):
    if own:
        from moba_amd import paged_prefix_attention
        return paged_prefix_attention(s["query"], s["cache"], s["page_table"], s["lengths"], s["cu_new"], s["cu_groups"], s["shared"])
    d, hkv, page, rep = case["head_dim"], case["kv_heads"], case["page"], case["heads"] // case["kv_heads"]
    table = s["page_table"].clamp(min=0).long()
    batch, keys = table.shape[0], table.shape[1] * page
    q, last = _padded_rows(s, case)
    longest = last.shape[1]
    k = _laid_out(s, "k", table).transpose(1, 2).reshape(batch, hkv, keys, d)
    scores = torch.matmul(q.float(), k.transpose(-1, -2).contiguous()).mul_(d ** -0.5).view(batch, hkv, rep, longest, keys)
    key = torch.arange(keys, device="cuda")
    scores.masked_fill_((key > last[:, :, None])[:, None, None], float("-inf"))
    scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    total = scores.sum(-1, keepdim=True)
    v = _laid_out(s, "v", table).transpose(1, 2).reshape(batch, hkv, keys, d)
    # (keys that nobody sees hold whatever the page held)
    v = torch.where((key < s["lengths"][:, None])[:, None, :, None], v, 0)
    out = torch.matmul(scores.view(batch, hkv, -1, keys), v).view(batch, hkv, rep, longest, d) / total
    return _packed_rows(s, out).to(s["query"].dtype)


def _run_sums(s, case):
    if own:
        from moba_amd import paged_key_sums
        paged_key_sums(s["cache"], s["sums"], s["page_table"], s["lengths"], s["cu_new"], s["query"].shape[0])
        return s["sums"]
    held = torch.arange(case["page"], device="cuda") < s["filled"][:, None]
    s["sums"][s["touched"]] = torch.where(held[:, None, :, None], _laid_out(s, "k", s["touched"]), 0).sum(2)
    return s["sums"]


def _run_select(s, case):
    block, topk = case["block"], case["topk"]
    if own:
        from moba_amd import paged_select_blocks
        return paged_select_blocks(s["query"], s["sums"], s["page_table"], s["lengths"], s["cu_new"], case["page"], block, topk)
    d, hkv, rep, each = case["head_dim"], case["kv_heads"], case["heads"] // case["kv_heads"], block // case["page"]
    table = s["page_table"].clamp(min=0).long()
    whole = max(table.shape[1] // each, 1)
    table = torch.nn.functional.pad(table, (0, max(0, each - table.shape[1])))[:, :whole * each]
    sums = s["sums"][table].double().unflatten(1, (whole, each)).sum(2)
    q, last = _padded_rows(s, case)
    scores = torch.matmul(q.double(), sums.permute(0, 2, 3, 1).contiguous()).view(-1, hkv, rep, last.shape[1], whole)
    own_block = last // block
    blk = torch.arange(whole, device="cuda")
    scores.masked_fill_((blk >= own_block[:, :, None])[:, None, None], float("-inf"))
    # (stable: of equal scores the lowest block comes first)
    order = scores.sort(dim=-1, descending=True, stable=True).indices[..., :topk - 1]
    own_block = own_block[:, None, None, :, None].expand(*scores.shape[:-1], 1).long()
    order = torch.where(torch.arange(order.shape[-1], device="cuda") < own_block, order, 1 << 30)
    order = torch.nn.functional.pad(order, (0, topk - 1 - order.shape[-1]), value=1 << 30)
    picks = torch.cat((order, own_block), -1).sort(-1).values
    return _packed_rows(s, torch.where(picks < 1 << 30, picks, -1)).int()


def _run_blocks(s, case):
    block, page, topk = case["block"], case["page"], case["topk"]
    if own:
        from moba_amd import paged_block_attention
        return paged_block_attention(s["query"], s["cache"], s["blocks"], s["page_table"], s["lengths"], s["cu_new"], block)
    d, hq, each = case["head_dim"], case["heads"], block // page
    _, b, at = _new_tokens(s)
    head = (torch.arange(hq, device="cuda") // (hq // case["kv_heads"]))[:, None]
    blocks = s["blocks"].clamp(min=0).long()
    number = (blocks[..., None] * each + torch.arange(each, device="cuda")).flatten(2)                   # pages of the blocks
    ids = s["page_table"][b[:, None, None], number.clamp(max=s["page_table"].shape[1] - 1)].clamp(min=0).long()
    key = (blocks[..., None] * block + torch.arange(block, device="cuda")).flatten(2)
    seen = (key <= at[:, None, None]) & (s["blocks"] >= 0).repeat_interleave(block, -1)
    scores = torch.matmul(_laid_out(s, "k", ids, head).flatten(2, 3), s["query"].float()[..., None])[..., 0].mul_(d ** -0.5)
    scores.masked_fill_(~seen, float("-inf"))
    scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    v = torch.where(seen[..., None], _laid_out(s, "v", ids, head).flatten(2, 3), 0)
    return (torch.matmul(scores[:, :, None], v)[:, :, 0] / scores.sum(-1, keepdim=True)).to(s["query"].dtype)


# ------------------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    if case["op"] in ("reserve", "select"):     # (whole numbers)
        return None
    s = prepare(case, seed)
    return {"prefix": _exact_attention, "sums": _exact_sums, "blocks": _exact_attention}[case["op"]](s, case)


def _exact_pages(s, half, ids, head):
    x = s[half + "_pages"][ids, head].double()
    return x if s[half + "_scales"] is None else x * s[half + "_scales"][ids, head].double()[:, None, None]


def _exact_sums(s, case):
    out, page = s["sums"].double(), case["page"]
    for b, (o, n) in enumerate(zip(_ints(case["old"]), _ints(case["new"]))):
        if not n:
            continue
        lo = o // page
        ids = s["page_table"][b, lo:-(-(o + n) // page)].long()
        for h in range(case["kv_heads"]):
            x = _exact_pages(s, "k", ids, h)
            x[-1, o + n - (lo + ids.numel() - 1) * page:] = 0
            out[ids, h] = x.sum(1)
    return out


def _exact_attention(s, case):
    """Softmax attention of every sequence and head, a row's blocks (all of them without any) and what it sees as one mask."""
    d, rep, page = case["head_dim"], case["heads"] // case["kv_heads"], case["page"]
    out, at = torch.zeros(s["query"].shape, dtype=torch.float64, device="cuda"), 0
    for b, (t, n) in enumerate(zip(_totals(case)[0], _ints(case["new"]))):
        if not n:
            continue
        ids = s["page_table"][b, :-(-t // page)].long()
        place = torch.arange(t, device="cuda")
        causal = place <= torch.arange(t - n, t, device="cuda")[:, None]
        for h in range(case["kv_heads"]):
            k, v = (_exact_pages(s, half, ids, h).reshape(-1, d)[:t] for half in ("k", "v"))
            for head in range(h * rep, (h + 1) * rep):
                seen = causal
                if case["op"] == "blocks":
                    chosen = torch.zeros((n, -(-t // case["block"]) + 1), dtype=torch.bool, device="cuda")
                    chosen.scatter_(1, s["blocks"][at:at + n, head].long().remainder(chosen.shape[1]), True)     # (-1: the one behind the last)
                    seen = causal & chosen[:, place // case["block"]]
                scores = s["query"][at:at + n, head].double() @ k.T / math.sqrt(d)
                out[at:at + n, head] = torch.softmax(scores.masked_fill(~seen, -math.inf), -1) @ v
        at += n
    return out
