"""The paged cache's operators in 64 bits on the CPU, written as plainly as they read, for the tests."""

import random

import torch

from rotary_reference import pair_size, turned

E4M3 = torch.float8_e4m3fn


def scale_of(most):
    """Smallest 2^k, k >= -100, with most <= 448 * 2^k."""
    k = -100
    while most > 448.0 * 2.0 ** k:
        k += 1
    return 2.0 ** k


class Batch:
    """Sequences of old + new tokens on shuffled pages, and a cache in which the old tokens lie (the rest is noise)."""

    def __init__(self, old, new, page, kv_heads, d, dtype, quantized, seed=0, spare=2, pad_rows=0, noise=1.0, device="cuda"):
        g = torch.Generator().manual_seed(seed)
        rng = random.Random(seed)
        self.old, self.new, self.page, self.dtype, self.quantized = old, new, page, dtype, quantized
        need = [-(-(o + n) // page) for o, n in zip(old, new)]
        pool = sum(need) + spare
        ids = list(range(pool))
        rng.shuffle(ids)
        wide = max(need + [1]) + 1
        self.table = torch.full((len(old), wide), -1, dtype=torch.int32)
        for b, n in enumerate(need):
            for i in range(n):
                self.table[b, i] = ids.pop()
        self.lengths = torch.tensor([o + n for o, n in zip(old, new)], dtype=torch.int32)
        self.cu = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32)
        self.rows = sum(new) + pad_rows
        shape = (pool, kv_heads, page, d)
        if quantized:
            self.pages = [(noise * 100 * torch.randn(shape, generator=g)).clamp(-448, 448).to(E4M3) for _ in range(2)]
            self.scales = [2.0 ** torch.randint(-9, -4, shape[:2], generator=g).float() for _ in range(2)]
        else:
            self.pages = [(noise * torch.randn(shape, generator=g)).to(dtype) for _ in range(2)]
            self.scales = [None, None]
        self.g = g

    def tensors(self, *heads):
        d = self.pages[0].shape[3]
        return [torch.randn((self.rows, h, d), generator=self.g).to(self.dtype) for h in heads]

    def cache(self, device="cuda"):
        from moba_amd import PagedKVCache
        return PagedKVCache(*(x.clone().to(device) for x in self.pages),
                            *(None if s is None else s.clone().to(device) for s in self.scales))

    def index(self, device="cuda"):
        return self.table.to(device), self.lengths.to(device), self.cu.to(device)

    def positions(self):
        """Of every row: its position, or None."""
        at = [o + i for o, n in zip(self.old, self.new) for i in range(n)]
        return at + [None] * (self.rows - len(at))


def appended(batch, k, v, inv_freq, interleaved):
    """Per half: what the cache has to hold after the call: (values [pool, heads, page, d] in 64 bits, error allowed, scales or None,
    where the scale may be the next one as well)."""
    at = [p if p is not None else 0 for p in batch.positions()]
    positions = torch.tensor(at, dtype=torch.int64)
    n = 0 if inv_freq is None else inv_freq.numel()
    kd = k.double()
    sides = [(kd if not n else turned(kd, positions, inv_freq, interleaved),
              30 * 2.0 ** -24 * pair_size(kd, n, interleaved) if n else torch.zeros_like(kd)), (v.double(), torch.zeros_like(v.double()))]
    result = []
    for half, (x, slack) in enumerate(sides):
        pages, scales = batch.pages[half], batch.scales[half]
        want = pages.double() if scales is None else pages.double() * scales[:, :, None, None].double()
        bound = torch.zeros_like(want)
        new_scales = None if scales is None else scales.clone()
        doubtful = None if scales is None else torch.zeros(scales.shape, dtype=torch.bool)
        fresh = {}
        row = 0
        for b, (o, c) in enumerate(zip(batch.old, batch.new)):
            for i in range(o, o + c):
                page = int(batch.table[b, i // batch.page]) if i // batch.page < batch.table.shape[1] else -1
                if 0 <= page < pages.shape[0]:
                    fresh.setdefault(page, []).append((i % batch.page, row))
                row += 1
        for page, tokens in fresh.items():
            slots, rows = [s for s, _ in tokens], [r for _, r in tokens]
            held = min(slots)
            for h in range(pages.shape[1]):
                new = x[rows, h]
                if scales is None:
                    want[page, h, slots] = new
                    half_step = torch.finfo(batch.dtype).eps / 2
                    bound[page, h, slots] = half_step * 1.001 * new.abs() + slack[rows, h] + (2.0 ** -25 if batch.dtype == torch.float16 else 0)
                    continue
                most = new.abs()[new.isfinite()].max().item() if new.isfinite().any() else 0.0
                s = scale_of(most)
                doubtful[page, h] = half == 0 and abs(most / (448 * s) - 0.75) >= 0.25 - 2.0 ** -18   # (at either end of a power of two)
                former = scales[page, h].item() if held else 0.0
                s = max(s, former)
                new_scales[page, h] = s
                want[page, h, slots] = torch.where(new.isinf(), new.sign() * 448 * s, new)
                bound[page, h, slots] = torch.maximum(2.0 ** -4 * new.abs(), torch.tensor(2.0 ** -10 * s, dtype=torch.float64)) * 1.001 + slack[rows, h]
                bound[page, h, slots] = torch.where(new.isfinite(), bound[page, h, slots], torch.zeros((), dtype=torch.float64))
                if s > former:
                    old = want[page, h, :held]
                    bound[page, h, :held] = torch.maximum(2.0 ** -4 * old.abs(), torch.tensor(2.0 ** -10 * s, dtype=torch.float64))
        result.append((want, bound, new_scales, doubtful, fresh))
    return result


def check_append(batch, cache, k, v, inv_freq, interleaved):
    """cache after paged_append(cache, k, v, ...) against `appended`."""
    got = [(cache.k_pages.cpu(), cache.k_scales), (cache.v_pages.cpu(), cache.v_scales)]
    for half, (want, bound, scales, doubtful, fresh) in enumerate(appended(batch, k, v, inv_freq, interleaved)):
        pages, new_scales = got[half]
        touched = torch.zeros(pages.shape[:3], dtype=torch.bool)
        for page, tokens in fresh.items():
            touched[page, :, [s for s, _ in tokens]] = True
        value = pages.double()
        if scales is not None:
            new_scales = new_scales.cpu()
            same = new_scales == scales
            near = doubtful & ((new_scales == 2 * scales) | (new_scales == scales / 2))
            assert bool((same | near).all()), (half, new_scales[~(same | near)], scales[~(same | near)])
            assert bool((torch.frexp(new_scales)[0] == 0.5).all())
            grown = new_scales > batch.scales[half]
            for page, tokens in fresh.items():
                held = min(s for s, _ in tokens)
                for h in range(pages.shape[1]):
                    if grown[page, h]:
                        touched[page, h, :held] = True
            value = value * new_scales[:, :, None, None].double()
        bits = torch.uint8 if scales is not None else torch.int16
        assert torch.equal(pages.view(bits)[~touched], batch.pages[half].view(bits)[~touched]), half   # the rest is as it was
        value, want, bound = value[touched], want[touched], bound[touched]
        assert torch.equal(value.isnan(), want.isnan())
        fine = ~want.isnan()
        off = (value - want).abs()[fine]
        assert bool((off <= bound[fine]).all()), (half, (off - bound[fine]).max().item())


def check_query(batch, got, query, inv_freq, interleaved):
    at = torch.tensor([p if p is not None else 0 for p in batch.positions()], dtype=torch.int64)
    x = query.double()
    n = 0 if inv_freq is None else inv_freq.numel()
    want = turned(x, at, inv_freq, interleaved) if n else x
    live = sum(batch.new)
    bound = torch.finfo(query.dtype).eps / 2 * 1.001 * want.abs() + (30 * 2.0 ** -24 * pair_size(x, n, interleaved) if n else 0) + 2.0 ** -25
    got = got.cpu()
    assert bool(((got[:live].double() - want[:live]).abs() <= bound[:live]).all())
    assert not got[live:].any()


def attended(batch, query, scaling=None):
    """[rows, heads, d] in 64 bits: every new token against its sequence's tokens up to itself; rows that see nothing: zeros.
    Returns also how far a result in 32 bits may be off, [rows, heads, 1]: with e the error of a score, a probability is off by
    2e of itself (its own and the sum's), and by 2^-15 for the exponential, the two elements it is split into and the sums, or by half a step of its type
    where a sequence has more than 32 rows, or 64 with 8-bit pages, and it is one element (all but fp16 queries on 8-bit pages); all of it times the largest finite value that the row sees.  e: D roundings of a sum of products, and 2^-22 of the score in the base-2 domain."""
    d, hkv = query.shape[2], batch.pages[0].shape[1]
    rep = query.shape[1] // hkv
    scale = d ** -0.5 if scaling is None else scaling
    out, slack, row = torch.zeros(query.shape, dtype=torch.float64), torch.zeros((*query.shape[:2], 1), dtype=torch.float64), 0
    for b, (o, c) in enumerate(zip(batch.old, batch.new)):
        if not c:
            continue
        length, table = o + c, batch.table[b]
        many = c * rep > (64 if batch.quantized else 32)
        rounded = many and not (batch.quantized and query.dtype == torch.float16)
        part = torch.finfo(query.dtype).eps / 2 if rounded else 0.0
        if batch.quantized and many and not all(bool((torch.frexp(s)[0] == 0.5).all()) for s in batch.scales):
            part += 2.0 ** -8       # (values times a scale that is no power of two are rounded to bf16)
        pages = [int(table[i]) if i < table.shape[0] else -1 for i in range(-(-length // batch.page))]
        good = [0 <= p < batch.pages[0].shape[0] for p in pages]
        there = torch.tensor(good).repeat_interleave(batch.page)[:length]
        ids = torch.tensor([p if g else 0 for p, g in zip(pages, good)])
        kv = []
        for half in range(2):
            x = batch.pages[half][ids].double()
            if batch.quantized:
                x = x * batch.scales[half][ids][:, :, None, None].double()
            kv.append(x.transpose(1, 2).reshape(-1, hkv, d)[:length])
        for j in range(c):
            seen = there & (torch.arange(length) <= o + j)
            if not seen.any():
                continue
            k, v = (x[seen].transpose(0, 1).repeat_interleave(rep, 0) for x in kv)      # [heads, keys, d]
            q = query[row + j].double()
            p = torch.softmax(torch.bmm(k, q[:, :, None])[..., 0] * scale, -1)
            out[row + j] = torch.bmm(p[:, None], v)[:, 0]
            size = abs(scale) * q.norm(dim=-1) * k.norm(dim=-1).amax(-1)
            slack[row + j] = ((2 * (d + 12) * 2.0 ** -24 * size + 2.0 ** -15 + part) * v.where(v.isfinite(), 0).abs().amax((1, 2)))[:, None]
        row += c
    return out, slack


def check_attention(batch, got, query, scaling=None):
    want, slack = attended(batch, query, scaling)
    got = got.cpu()
    assert got.dtype == query.dtype and got.shape == query.shape
    assert torch.equal(got.isnan(), want.isnan()), (got.isnan().sum(), want.isnan().sum())
    fine = want.isfinite()
    assert torch.equal(got[~fine & ~want.isnan()].double(), want[~fine & ~want.isnan()])
    bound = torch.finfo(query.dtype).eps / 2 * 1.001 * want.abs() + slack + 2.0 ** -25
    off = (got.double() - want).abs()
    bad = fine & ~(off <= bound)
    assert not bad.any(), (bad.nonzero()[:5].tolist(), (off / bound)[fine].max().item())
