"""The operators around the attention of a decoder layer, as cases whose time and results can be compared with a plain form.

Three operators, each through the package's public entry point:

  norm    ``qk_norm_rope``: the root-mean-square norm of every query and key head and the rotation by position, for packed
          tokens; forward, or forward and backward
  append  ``paged_append``: the keys and values of new tokens into a paged cache (16-bit elements, or 8 bits with a scale for
          every page and head), keys and queries rotated by their positions on the way
  attend  ``paged_attention``: new tokens of every sequence against such a cache: one token each, a few, or a long piece

With ``own`` false everything is computed from elementary torch operations in 32 bits (angles in 64) and rounded once.

A page's scale is the power of two 2^k with the smallest k for which the page's largest magnitude is at most 448 * 2^k; a page
that already holds tokens keeps its scale if that is larger, and its elements are rounded again where the scale grows.
"""

import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_E4M3 = torch.float8_e4m3fn
_MOST = 448.0          # the largest e4m3 value
_LEAST_EXPONENT = -100  # of a page's scale
_EPS = 1e-6


def _norm(name, **kw):
    base = dict(name=name, op="norm", train=False, lens="1", heads=32, kv_heads=8, head_dim=128, rotary=128, interleaved=False,
                weights=True, dtype="bf16", far=0)
    base.update(kw)
    return base


def _append(name, **kw):
    base = dict(name=name, op="append", heads=32, kv_heads=8, head_dim=128, rotary=128, interleaved=False, dtype="bf16",
                cache="e4m3", page=64, old="0", new="1")
    base.update(kw)
    return base


def _attend(name, **kw):
    base = dict(name=name, op="attend", heads=32, kv_heads=8, head_dim=128, dtype="bf16", cache="e4m3", page=64, old="0", new="1")
    base.update(kw)
    return base


def listed():
    return [
        # generation for one user, far into a long document: launches and latency count
        _norm("norm_token", lens="1", far=131071),
        # one layer of the headline configuration: a 128K-token prompt of 32 heads on 8
        _norm("norm_prompt_128k", lens="131072"),
        # a training batch of five documents packed to 20K tokens
        _norm("norm_train_packed", train=True, lens="1023,7001,400,3579,8477", heads=8, kv_heads=2),
        # training with narrow heads, neighbouring elements rotated together, half of every head rotated, fp16
        _norm("norm_train_narrow", train=True, lens="32768,29343,5003", head_dim=64, rotary=32, interleaved=True, dtype="fp16"),
        # one decoding step of sixteen users whose caches hold from a few to thousands of tokens
        _append("append_tokens", old="8191,1,4095,700,63,64,2000,5003,127,1024,0,3579,900,31,6001,400", new=",".join(["1"] * 16)),
        # the whole headline prompt goes into an empty 8-bit cache
        _append("append_prompt_128k", new="131072"),
        # a mixed batch, fp16, 16-bit pages of 16 tokens, narrow heads: short turns, one token, a prompt's next piece
        _append("append_mixed", old="4090,17,34816,0,301", new="5,1,2048,300,77", dtype="fp16", cache="same", page=16, head_dim=64,
                rotary=64, interleaved=True),
        # generation: a short conversation, ...
        _attend("attend_token_4k", old="4096"),
        # ... a long document, ...
        _attend("attend_token_128k", old="131071"),
        # ... and a batch of sixteen users of very different lengths, fp16
        _attend("attend_tokens", old="8190,131,16000,700,63,64,2000,5003,127,1024,0,3579,900,31,24001,400",
                new=",".join(["1"] * 16), dtype="fp16"),
        # five drafted tokens of four sequences to be checked in one pass, pages of 16-bit elements
        _attend("attend_few", old="20000,19000,20480,12345", new="5,5,5,5", cache="same"),
        # a long prompt taken in pieces of 2048 tokens: the seventeenth piece, 8-bit pages
        _attend("attend_piece_2k", old="32768", new="2048"),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def _join(values):
    return ",".join(str(v) for v in values)


def _ints(text):
    return [int(v) for v in text.split(",")]


def _draw_once(rng):
    op = rng.choice(("norm", "append", "attend"))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    kv = rng.choice((1, 2, 4, 8))
    heads = kv * rng.choice((1, 2, 4, 5, 8))
    if op == "norm":
        head_dim = rng.choice((64, 96, 128, 128))
        total, parts = _log_int(rng, 1, 131072), rng.randint(1, 6)
        marks = sorted(rng.randint(0, total) for _ in range(parts - 1))
        lens = [b - a for a, b in zip([0] + marks, marks + [total])]
        return _norm("", train=rng.random() < 0.6, lens=_join(lens), heads=heads, kv_heads=kv, head_dim=head_dim,
                     rotary=rng.choice((head_dim, head_dim, head_dim // 2)), interleaved=rng.random() < 0.4,
                     weights=rng.random() < 0.75, dtype=dtype, far=rng.choice((0, 0, _log_int(rng, 1, 1000000))))
    kind = rng.choice(("token", "token", "few", "many"))
    batch = _log_int(rng, 1, 64) if kind == "token" else _log_int(rng, 1, 16) if kind == "few" else rng.randint(1, 4)
    most = _log_int(rng, 50, 131072 if op == "attend" else 8192)
    old = [int(most * (1 - 0.9 * rng.random() ** 2)) if rng.random() < 0.9 else 0 for _ in range(batch)]
    if kind == "token":
        new = [1] * batch
    elif kind == "few":
        new = [rng.randint(0, 9) for _ in range(batch)]
        new[rng.randrange(batch)] = rng.randint(2, 9)
    else:
        piece = _log_int(rng, 10, 4096 if op == "attend" else 32768)
        new = [rng.randint(0, piece) for _ in range(batch)]
        new[rng.randrange(batch)] = piece
    head_dim = rng.choice((64, 128, 128, 128))
    common = dict(heads=heads, kv_heads=kv, head_dim=head_dim, dtype=dtype, cache=rng.choice(("e4m3", "e4m3", "same")),
                  page=rng.choice((16, 32, 64, 64, 128)), old=_join(old), new=_join(new))
    if op == "append":
        return _append("", rotary=rng.choice((head_dim, head_dim, head_dim // 2)), interleaved=rng.random() < 0.4, **common)
    return _attend("", **common)


def draw(rng):
    """One more case of the same ranges: no dearer than the dearest listed one, in operations and in bytes."""
    most = [work(c) for c in listed()]
    flops, nbytes = (max(w[x] for w in most) for x in ("flops", "bytes"))
    while True:
        case = _draw_once(rng)
        need = work(case)
        if need["flops"] <= flops and need["bytes"] <= nbytes:
            del case["name"]
            return case


def work(case):
    """What a pass cannot do without: inputs read once, outputs written once."""
    d, hq, hkv = case["head_dim"], case["heads"], case["kv_heads"]
    if case["op"] == "norm":
        elements = sum(_ints(case["lens"])) * (hq + hkv) * d
        passes = 4 if case["train"] else 2        # x, y; and their gradients
        return {"bytes": 2.0 * passes * elements, "flops": (25.0 if case["train"] else 8.0) * elements}
    old, new = _ints(case["old"]), _ints(case["new"])
    tokens, width = sum(new), 1 if case["cache"] == "e4m3" else 2
    if case["op"] == "append":
        return {"bytes": 2.0 * tokens * (2 * hq + 2 * hkv) * d + 2.0 * width * tokens * hkv * d,
                "flops": 6.0 * tokens * (hq + hkv) * d}
    keys = sum(o + n for o, n in zip(old, new) if n)
    pairs = sum(n * o + n * (n + 1) // 2 for o, n in zip(old, new))
    return {"bytes": 2.0 * width * keys * hkv * d + 4.0 * tokens * hq * d, "flops": 4.0 * d * hq * pairs}


# ------------------------------------------------------------------------------------------------------------ inputs
def _inv_freq(rotary):
    return (500000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)).float().cuda()


def _normal(g, shape, dtype):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _scale_of(most):
    """The scale of pages whose largest magnitudes are `most`."""
    mantissa, exponent = torch.frexp(most)
    k = exponent - 9 + (mantissa > 0.875).int()
    return torch.exp2(torch.where(most > 0, k, _LEAST_EXPONENT).clamp(min=_LEAST_EXPONENT).float()).to(most.dtype)


def _pages(g, case, filled):
    """Pages of one of the cache's halves, `filled` [pages] tokens of each in use: (elements, scales or None)."""
    shape = (filled.numel(), case["kv_heads"], case["page"], case["head_dim"])
    if case["cache"] == "same":
        return _normal(g, shape, _DTYPES[case["dtype"]]), None
    x = torch.randn(shape, generator=g, device="cuda")
    used = torch.arange(case["page"], device="cuda") < filled[:, None]
    scales = _scale_of((x.abs() * used[:, None, :, None]).amax((2, 3)))
    return (x / scales[:, :, None, None]).clamp(-_MOST, _MOST).to(_E4M3), scales


def _layout(case, seed, held):
    """Page table of sequences of old + new tokens, and how many tokens each page of the pool holds, `held` of each sequence."""
    page, old, new = case["page"], _ints(case["old"]), _ints(case["new"])
    need = [-(-(o + n) // page) for o, n in zip(old, new)]
    pool = sum(need) + 3
    ids = list(range(pool))
    random.Random(seed).shuffle(ids)
    table, filled = [[-1] * max(1, max(need)) for _ in need], [page] * pool
    for b, count in enumerate(need):
        for i in range(count):
            table[b][i] = ids.pop()
            filled[table[b][i]] = min(max(held[b] - i * page, 0), page)
    return table, filled


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, d, hq, hkv = _DTYPES[case["dtype"]], case["head_dim"], case["heads"], case["kv_heads"]
    if case["op"] == "norm":
        lens = _ints(case["lens"])
        s = {"case": case, "q": _normal(g, (sum(lens), hq, d), dtype), "k": _normal(g, (sum(lens), hkv, d), dtype) * 2,
             "inv_freq": _inv_freq(case["rotary"]),
             "positions": torch.cat([torch.arange(n) + case["far"] for n in lens]).cuda(), "q_weight": None, "k_weight": None}
        if case["weights"]:
            for name in ("q_weight", "k_weight"):
                s[name] = (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(dtype)
        if case["train"]:
            for name in ("q", "k", "q_weight", "k_weight"):
                if s[name] is not None:
                    s[name].requires_grad_()
            s["dq"], s["dk"] = (_normal(g, s[x].shape, dtype) for x in ("q", "k"))
        return s
    old, new = _ints(case["old"]), _ints(case["new"])
    total = [o + n for o, n in zip(old, new)]
    table, filled = _layout(case, seed, old if case["op"] == "append" else total)
    filled = torch.tensor(filled, device="cuda")
    s = {"case": case, "page_table": torch.tensor(table, dtype=torch.int32, device="cuda"),
         "lengths": torch.tensor(total, dtype=torch.int32, device="cuda"),
         "cu_new": torch.tensor([0] + [sum(new[:i + 1]) for i in range(len(new))], dtype=torch.int32, device="cuda"),
         "query": _normal(g, (sum(new), hq, d), dtype)}
    for half in ("k", "v"):
        s[half + "_pages"], s[half + "_scales"] = _pages(g, case, filled)
    if case["op"] == "append":
        s["key"], s["value"] = _normal(g, (sum(new), hkv, d), dtype) * 2, _normal(g, (sum(new), hkv, d), dtype)
        s["inv_freq"] = _inv_freq(case["rotary"])
        # the pages that receive tokens, which whoever hands out pages knows: page ids, the sequences they belong to, and
        # which of a sequence's pages they are; where each sequence's begin
        hit = [(table[b][i], b, i) for b in range(len(new)) if new[b] for i in range(old[b] // case["page"], (total[b] - 1) // case["page"] + 1)]
        s["touched"] = tuple(torch.tensor(x, device="cuda") for x in zip(*hit))
        first = [0]
        for o, n, t in zip(old, new, total):
            first.append(first[-1] + ((t - 1) // case["page"] + 1 - o // case["page"] if n else 0))
        s["touched_from"] = torch.tensor(first[:-1], device="cuda")
    if own:
        from moba_amd import PagedKVCache
        s["cache"] = PagedKVCache(s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"])
    return s


# ------------------------------------------------------------------------------------------------------------ passes
def run(s):
    case = s["case"]
    if case["op"] == "norm":
        return _run_norm(s, case)
    return _run_append(s, case) if case["op"] == "append" else _run_attend(s, case)


def _rotated(x, positions, inv_freq, interleaved):
    """x [tokens, heads, head_dim] in 32 bits, its first 2 * len(inv_freq) elements rotated."""
    angles = positions.double()[:, None] * inv_freq.double()
    cos, sin = angles.cos().float()[:, None], angles.sin().float()[:, None]
    half = inv_freq.numel()
    part, rest = x[..., :2 * half], x[..., 2 * half:]
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
        part = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = part[..., :half], part[..., half:]
        part = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((part, rest), -1)


def _plain_norm(x, weight, s, case):
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS) * weight
    return _rotated(x, s["positions"], s["inv_freq"], case["interleaved"])


def _run_norm(s, case):
    inputs = [s[n] for n in ("q", "k", "q_weight", "k_weight")]
    if own:
        from moba_amd import qk_norm_rope
        q, k, qw, kw = inputs
        yq, yk = qk_norm_rope(q, k, s["positions"], s["inv_freq"], qw, kw, eps=_EPS, interleaved=case["interleaved"])
        if not case["train"]:
            return [yq, yk]
        return [yq, yk, *torch.autograd.grad((yq, yk), [x for x in inputs if x is not None], (s["dq"], s["dk"]))]
    wide = [None if x is None else x.detach().float().requires_grad_(case["train"]) for x in inputs]
    yq, yk = (_plain_norm(wide[i], wide[i + 2], s, case) for i in (0, 1))
    y = [v.detach().to(x.dtype) for v, x in ((yq, s["q"]), (yk, s["k"]))]
    if not case["train"]:
        return y
    grads = torch.autograd.grad((yq, yk), [x for x in wide if x is not None], (s["dq"].float(), s["dk"].float()))
    return [*y, *(g.to(s["q"].dtype) for g in grads)]


def _new_tokens(s, tokens):
    """Of every new token: its sequence and its position there."""
    t = torch.arange(tokens, device="cuda")
    b = torch.searchsorted(s["cu_new"], t, right=True) - 1
    return t, b, s["lengths"][b] - s["cu_new"][b + 1] + t


def _run_append(s, case):
    outputs = {n: s[n] for n in ("k_pages", "v_pages", "k_scales", "v_scales") if s[n] is not None}
    if own:
        from moba_amd import paged_append
        outputs["query"] = paged_append(s["cache"], s["key"], s["value"], s["page_table"], s["lengths"], s["cu_new"],
                                        inv_freq=s["inv_freq"], query=s["query"], interleaved=case["interleaved"])
        return outputs
    page, tokens = case["page"], s["query"].shape[0]
    t, b, at = _new_tokens(s, tokens)
    turn = lambda x: _rotated(x.float(), at, s["inv_freq"], case["interleaved"])  # noqa: E731
    outputs["query"] = turn(s["query"]).to(s["query"].dtype)
    began = s["lengths"] - s["cu_new"].diff()
    item, row = s["touched_from"][b] + at // page - began[b] // page, at % page
    for half, x in (("k", turn(s["key"])), ("v", s["value"].float())):
        pages, scales = s[half + "_pages"], s[half + "_scales"]
        if scales is None:
            pages[s["touched"][0][item], :, row] = x.to(pages.dtype)
            continue
        ids, seq, number = s["touched"]
        grid = torch.zeros((ids.numel(), page, *x.shape[1:]), device="cuda")
        grid[item, row] = x
        grid = grid.transpose(1, 2)
        place = number[:, None] * page + torch.arange(page, device="cuda")
        held = place < began[seq][:, None]
        fresh = (~held & (place < s["lengths"][seq][:, None]))[:, None, :, None]
        former, codes = scales[ids], pages[ids]
        scale = torch.where(held[:, :1], former, 0).maximum(_scale_of(grid.abs().amax((2, 3))))
        again = held[:, None, :, None] & (scale > former)[:, :, None, None]
        grid = torch.where(fresh, grid, codes.float() * former[:, :, None, None]) / scale[:, :, None, None]
        changed = torch.where(fresh | again, grid.clamp(-_MOST, _MOST), codes.float())
        pages[ids] = changed.to(_E4M3)
        scales[ids] = scale
    return outputs


def _run_attend(s, case):
    longest = max(_ints(case["new"]))
    if own:
        from moba_amd import paged_attention
        return paged_attention(s["query"], s["cache"], s["page_table"], s["lengths"], s["cu_new"], max_new=longest)
    d, hq, hkv, page = case["head_dim"], case["heads"], case["kv_heads"], case["page"]
    table = s["page_table"].clamp(min=0).long()
    batch, keys = table.shape[0], table.shape[1] * page

    def laid_out(half):
        x = s[half + "_pages"][table].float()
        if s[half + "_scales"] is not None:
            x = x * s[half + "_scales"][table][..., None, None]
        return x.transpose(1, 2).reshape(batch, hkv, keys, d)

    begin, count = s["cu_new"][:-1, None], s["cu_new"].diff()[:, None]
    i = torch.arange(longest, device="cuda")
    q = s["query"].float()[(begin + torch.minimum(i, count - 1).clamp(min=0)).clamp(max=s["query"].shape[0] - 1)]
    q = q.reshape(batch, longest, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(batch, hkv, -1, d)
    scores = torch.matmul(q, laid_out("k").transpose(-1, -2).contiguous()).mul_(d ** -0.5)
    scores = scores.view(batch, hkv, hq // hkv, longest, keys)
    last = s["lengths"][:, None] - count + i
    hidden = torch.arange(keys, device="cuda") > last[:, :, None]
    scores.masked_fill_(hidden[:, None, None], float("-inf"))
    scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    total = scores.sum(-1, keepdim=True)
    # (keys that nobody sees hold whatever the page held)
    v = torch.where((torch.arange(keys, device="cuda") < s["lengths"][:, None])[:, None, :, None], laid_out("v"), 0)
    out = torch.matmul(scores.view(batch, hkv, -1, keys), v).view_as(scores[..., :1].expand(*scores.shape[:-1], d)) / total
    _, b, at = _new_tokens(s, s["query"].shape[0])
    out = out.permute(0, 3, 1, 2, 4)[b, at - (s["lengths"] - count[:, 0])[b]]
    return out.reshape(-1, hq, d).to(s["query"].dtype)


# ------------------------------------------------------------------------------------------------------------ in 64 bits
def _turned(x, positions, inv_freq, interleaved, back=False):
    """x in 64 bits, the rotated pairs as complex numbers."""
    angles = positions.double()[:, None] * inv_freq.double()
    turn = torch.polar(torch.ones_like(angles), -angles if back else angles)[:, None]
    n = inv_freq.numel()
    out = x.clone()
    if interleaved:
        pairs = torch.view_as_complex(x[..., :2 * n].reshape(*x.shape[:-1], n, 2).contiguous()) * turn
        out[..., :2 * n] = torch.view_as_real(pairs).flatten(-2)
    else:
        pairs = torch.complex(x[..., :n].contiguous(), x[..., n:2 * n].contiguous()) * turn
        out[..., :n], out[..., n:2 * n] = pairs.real, pairs.imag
    return out


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "norm":
            return _exact_norm(s, case)
        return _exact_append(s, case) if case["op"] == "append" else _exact_attend(s, case)


def _exact_norm(s, case):
    tokens = s["q"].shape[0]
    y, dx, dw = [], [], []
    for name in ("q", "k"):
        x, weight = s[name], s[name + "_weight"]
        ys, ds, sums = [], [], 0
        for lo in range(0, tokens, 16384):
            part = slice(lo, lo + 16384)
            xx, at = x[part].double(), s["positions"][part]
            w = None if weight is None else weight.double()
            r = 1 if w is None else 1 / torch.sqrt((xx * xx).sum(-1, keepdim=True) / xx.shape[-1] + _EPS)
            unit = xx * r
            ys.append(_turned(unit if w is None else unit * w, at, s["inv_freq"], case["interleaved"]))
            if case["train"]:
                up = _turned(s["d" + name][part].double(), at, s["inv_freq"], case["interleaved"], back=True)
                if w is None:
                    ds.append(up)
                else:
                    sums = sums + (up * unit).sum((0, 1))
                    up = up * w
                    ds.append(r * (up - unit * (up * unit).sum(-1, keepdim=True) / xx.shape[-1]))
        y.append(torch.cat(ys))
        if case["train"]:
            dx.append(torch.cat(ds))
            if weight is not None:
                dw.append(sums)
    return y + dx + dw


def _exact_append(s, case):
    page, old, new = case["page"], _ints(case["old"]), _ints(case["new"])
    out = {n: s[n].double() for n in ("k_pages", "v_pages", "k_scales", "v_scales") if s[n] is not None}
    place = torch.cat([torch.arange(o, o + n) for o, n in zip(old, new)]).cuda()
    out["query"] = _turned(s["query"].double(), place, s["inv_freq"], case["interleaved"])
    halves = {"k": _turned(s["key"].double(), place, s["inv_freq"], case["interleaved"]), "v": s["value"].double()}
    at = 0
    for b, (o, n) in enumerate(zip(old, new)):
        if not n:
            continue
        lo, hi = o // page, (o + n - 1) // page + 1
        ids, skip = s["page_table"][b, lo:hi].long(), o - lo * page
        for half, x in halves.items():
            rows = out[half + "_pages"][ids].transpose(1, 2).flatten(0, 1)
            fresh = torch.zeros_like(rows)
            fresh[skip:skip + n] = x[at:at + n]
            if case["cache"] == "e4m3":
                most = fresh.view(-1, page, *rows.shape[1:]).abs().amax((1, 3))
                want = torch.exp2(torch.ceil(torch.log2(most / _MOST)))
                want = torch.where(most <= want / 2 * _MOST, want / 2, torch.where(most > want * _MOST, want * 2, want))
                want = torch.where(most > 0, want.clamp(min=2.0 ** _LEAST_EXPONENT), 2.0 ** _LEAST_EXPONENT)
                if skip:
                    before = out[half + "_scales"][ids[0]]
                    want[0] = torch.maximum(want[0], before)
                    rows[:skip] *= (before / want[0])[:, None]
                out[half + "_scales"][ids] = want
                fresh = (fresh.view(-1, page, *rows.shape[1:]) / want[:, None, :, None]).flatten(0, 1)
            rows[skip:skip + n] = fresh[skip:skip + n]
            out[half + "_pages"][ids] = rows.view(-1, page, *rows.shape[1:]).transpose(1, 2)
        at += n
    return out


def _exact_attend(s, case):
    d, rep, page = case["head_dim"], case["heads"] // case["kv_heads"], case["page"]
    out, at = torch.zeros(s["query"].shape, dtype=torch.float64, device="cuda"), 0
    for b, (o, n) in enumerate(zip(_ints(case["old"]), _ints(case["new"]))):
        if not n:
            continue
        ids = s["page_table"][b, :-(-(o + n) // page)].long()
        hidden = torch.arange(o + n, device="cuda") > torch.arange(o, o + n, device="cuda")[:, None]
        for h in range(case["kv_heads"]):
            kv = []
            for half in ("k", "v"):
                x = s[half + "_pages"][ids][:, h].double()
                if s[half + "_scales"] is not None:
                    x = x * s[half + "_scales"][ids][:, h, None, None].double()
                kv.append(x.reshape(-1, d)[:o + n])
            for head in range(h * rep, (h + 1) * rep):
                p = s["query"][at:at + n, head].double() @ kv[0].T / math.sqrt(d)
                out[at:at + n, head] = torch.softmax(p.masked_fill(hidden, -math.inf), -1) @ kv[1]
        at += n
    return out
