"""The precision that paged_prefix_attention promises for few rows, on inputs whose scores are exact in 32 bits, for the tests.

Queries are whole numbers up to 2, keys multiples of 1/4 up to 3 (8-bit pages: whole numbers up to 4, times a power of two as the scale), so
that a score's products and sums are exact in 32 bits whatever their order, and what is left is
  a score in the base-2 domain: its products with the softmax scale and log2(e), the subtraction of the reference, and a run's log-sum-exp
     where runs meet, each half a step (2^-24) of numbers up to `top` + 10: at most 2^-21 * (top + 10) together, once for the row and once for
     the sum
  a probability: the sum of two elements, 2^-18 of it off (bf16: 2^-9 * 2^-9; 2^-24 in fp16), its exponential 2^-21, times the value's
     scale 2^-24
  sums: one 2^-24 for each key, of the products and of the probabilities, and some for the runs
times sum p |v|, and of the quotient's two sides.  Then half a step of the result's type."""

import torch

from paged_reference import Batch


def limit(d, quantized):
    """Rows (tokens times heads on a key/value head) of a group or a sequence that have that precision."""
    return 128 if d == 128 and not quantized else 256


def exact_batch(old, new, page, kv_heads, d, dtype, quantized, seed):
    batch = Batch(old, new, page, kv_heads, d, dtype, quantized, seed=seed)
    g, shape = batch.g, batch.pages[0].shape
    k = torch.randint(-12, 13, shape, generator=g).float() / 4
    if quantized:       # (odd scales for the values, whose products are rounded where there are many rows)
        k = torch.randint(-4, 5, shape, generator=g).float()
        batch.pages = [k.to(batch.pages[0].dtype), torch.randn(shape, generator=g).to(batch.pages[1].dtype)]
        batch.scales = [2.0 ** torch.randint(-2, 1, shape[:2], generator=g).float(), torch.rand(shape[:2], generator=g) + 0.5]
    else:
        batch.pages = [k.to(dtype), torch.randn(shape, generator=g).to(dtype)]
    return batch


def exact_queries(batch, heads):
    d = batch.pages[0].shape[3]
    return torch.randint(-2, 3, (batch.rows, heads, d), generator=batch.g).to(batch.dtype)


def wanted(batch, query, one_element=False):
    """(result, bound of its error) in 64 bits; one_element: with probabilities and values rounded as where there are many rows."""
    d, hkv = query.shape[2], batch.pages[0].shape[1]
    rep, scale, row = query.shape[1] // hkv, d ** -0.5, 0
    out, bound = torch.zeros(query.shape, dtype=torch.float64), torch.zeros(query.shape, dtype=torch.float64)
    kind = torch.bfloat16 if batch.quantized else query.dtype
    for b, (o, c) in enumerate(zip(batch.old, batch.new)):
        ids = batch.table[b, :-(-(o + c) // batch.page)].long()
        k, v = (x[ids].double() if s is None else x[ids].double() * s[ids][:, :, None, None].double() for x, s in zip(batch.pages, batch.scales))
        k, v = (x.transpose(1, 2).reshape(-1, hkv, d)[:o + c].transpose(0, 1).repeat_interleave(rep, 0) for x in (k, v))   # [heads, keys, d]
        for j in range(c):
            n = o + j + 1
            s = torch.bmm(k[:, :n], query[row + j].double()[:, :, None])[..., 0] * scale
            p, vv = torch.softmax(s, -1), v[:, :n]
            if one_element:
                p = torch.exp(s - s.amax(-1, keepdim=True))
                total, p = p.sum(-1, keepdim=True), p.to(kind).double()
                out[row + j] = torch.bmm(p[:, None], vv.to(kind).double())[:, 0] / total
                continue
            out[row + j] = torch.bmm(p[:, None], vv)[:, 0]
            top = s.abs().amax(-1, keepdim=True) * 1.4427
            step = 2 * 2.0 ** -21 * (top + 10) + (2.0 ** -18 if kind == torch.bfloat16 else 2.0 ** -24) + 2 * 2.0 ** -21 + (2 * n + 64) * 2.0 ** -24
            bound[row + j] = step * torch.bmm(p[:, None], vv.abs())[:, 0]
        row += c
    half = torch.finfo(query.dtype).eps / 2 * 1.001
    return out, half * (out.abs() + bound) + bound + 2.0 ** -25


def is_within(got, want, bound):
    return (got.cpu().double() - want).abs() <= bound


# groups' first and last sequences, their shared tokens; of every sequence: tokens before, new ones; heads, key/value heads.  The last group is
# there to have more rows than are few, where `beside`.
def cases(d, quantized):
    most = limit(d, quantized)
    for rows in (33, 48, 65, 100, 128, 129, 200, most):          # single tokens, four heads or one to a key/value head
        if rows > most:
            continue
        rep = 4 if rows % 4 == 0 else 1
        yield [96] * (rows // rep), [1] * (rows // rep), rep
    yield [96, 100, 130], [most // 8, 1, most // 16], 4             # pieces of prompts, few rows each and together
    yield [96, 120], [most // 4, 0], 4                              # one of as many rows as are few
    yield [96] * 7, [3, 0, 5, 1, 2, 9, 1], 5
