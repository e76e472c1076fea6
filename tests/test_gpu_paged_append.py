"""paged_append on the GPU against its definition in 64 bits, token by token."""

import pytest
import torch

from paged_reference import E4M3, Batch, check_append, check_query
from rotary_reference import frequencies

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16

CASES = [  # old, new, page, heads, kv heads, head_dim, rotated pairs, interleaved, dtype, quantized, rows behind
    ([0], [1], 64, 4, 1, 128, 64, False, BF16, True, 0),
    ([131071], [1], 64, 8, 2, 128, 64, False, BF16, True, 0),
    ([0, 63, 64, 65, 10, 127], [1, 1, 1, 1, 0, 1], 64, 4, 2, 128, 64, False, FP16, True, 0),
    ([0, 63, 64, 65, 10, 127], [1, 1, 1, 1, 0, 1], 64, 4, 2, 128, 64, True, BF16, False, 2),
    ([5, 0, 31, 100], [70, 16, 0, 3], 16, 3, 3, 128, 32, False, BF16, True, 5),
    ([5, 0, 31, 100], [70, 17, 1, 300], 32, 5, 5, 64, 32, True, FP16, True, 1),
    ([5, 0, 31], [70, 17, 1], 16, 2, 1, 64, 16, False, FP16, False, 0),
    ([200, 3], [600, 300], 256, 4, 4, 128, 64, False, BF16, True, 0),       # pages of more tokens than have angles at a time
    ([200, 3], [130, 257], 128, 9, 9, 64, 32, False, BF16, False, 0),
    ([7] * 70, [1, 0, 2, 5, 1] * 14, 16, 2, 2, 64, 32, False, BF16, True, 3),   # more sequences than a wave has lanes
    ([1, 40], [33, 5], 32, 1, 17, 64, 0, False, BF16, True, 0),             # no rotation
    ([(1 << 17) - 5], [9], 256, 1, 1, 64, 32, False, BF16, True, 0),
]


@pytest.mark.parametrize("old,new,page,heads,kv_heads,d,pairs,interleaved,dtype,quantized,behind", CASES)
def test_append(old, new, page, heads, kv_heads, d, pairs, interleaved, dtype, quantized, behind):
    from moba_amd import paged_append
    print("append", old[:6], new[:6], page, heads, kv_heads, d, pairs, interleaved, dtype, quantized, behind, flush=True)
    batch = Batch(old, new, page, kv_heads, d, dtype, quantized, seed=page + d + len(old), pad_rows=behind)
    k, v, q = batch.tensors(kv_heads, kv_heads, heads)
    k[:, ::2] *= 5     # (scales that grow, and scales that do not)
    cache, inv_freq = batch.cache(), frequencies(pairs) if pairs else None
    got = paged_append(cache, k.cuda(), v.cuda(), *batch.index(), inv_freq=None if inv_freq is None else inv_freq.cuda(),
                       query=q.cuda(), interleaved=interleaved)
    check_query(batch, got, q, inv_freq, interleaved)
    check_append(batch, cache, k, v, inv_freq, interleaved)
    again = batch.cache()
    assert paged_append(again, k.cuda(), v.cuda(), *batch.index(), inv_freq=None if inv_freq is None else inv_freq.cuda(),
                        interleaved=interleaved) is None
    for name in ("k_pages", "v_pages", "k_scales", "v_scales"):
        a, b = getattr(again, name), getattr(cache, name)
        assert a is None or torch.equal(a.view(torch.uint8), b.view(torch.uint8)), name


def test_token_by_token():
    """Tokens one at a time: every step against the definition from the state before it, scales growing on the way."""
    from moba_amd import paged_append
    batch = Batch([0, 30], [1, 1], 16, 2, 64, BF16, True, seed=4, spare=6)
    batch.table = torch.arange(2 * 5, dtype=torch.int32).view(2, 5)
    batch.pages, batch.scales = [x[:1].expand(10, 2, 16, 64).clone() for x in batch.pages], [s[:1].expand(10, 2).clone() for s in batch.scales]
    inv_freq = frequencies(32)
    for step in range(40):
        batch.lengths = torch.tensor([o + 1 for o in batch.old], dtype=torch.int32)
        k, v = (x * (1 + 0.3 * step) for x in batch.tensors(2, 2))
        cache = batch.cache()
        paged_append(cache, k.cuda(), v.cuda(), *batch.index(), inv_freq=inv_freq.cuda())
        check_append(batch, cache, k, v, inv_freq, False)
        batch.pages, batch.scales = [cache.k_pages.cpu(), cache.v_pages.cpu()], [cache.k_scales.cpu(), cache.v_scales.cpu()]
        batch.old = [o + 1 for o in batch.old]


def test_values_at_the_ends():
    """Zeros, the type's smallest and largest numbers, infinities and NaN, in new pages and in pages that hold tokens."""
    from moba_amd import paged_append
    for dtype in (BF16, FP16):
        batch = Batch([0, 20], [20, 5], 16, 3, 64, dtype, True, seed=9)
        k, v = batch.tensors(3, 3)
        tiny, huge = torch.finfo(dtype).smallest_normal, torch.finfo(dtype).max
        v[:16, 0] = 0
        v[:16, 1] = v[:16, 1].sign() * tiny
        v[3, 2, 7], v[20, 1, 0] = huge, -huge
        v[17, 0, 5], v[18, 1, 6], v[21, 2, 1] = float("inf"), float("-inf"), float("nan")
        v[5, 2, 9], v[6, 2, 9], v[7, 2] = float("inf"), float("-inf"), float("nan")   # beside the largest number
        k[2, 0] = 0
        k[:16, 1] = 0
        k[19, 2, 40] = float("nan")
        cache = batch.cache()
        paged_append(cache, k.cuda(), v.cuda(), *batch.index())
        check_append(batch, cache, k, v, None, False)
        # a page's largest magnitude at 448 * 2^k takes 2^k, the next number of the type the next scale
        edge = Batch([0], [2], 16, 2, 64, dtype, True, seed=1)
        k, v = torch.zeros((2, 2, 64), dtype=dtype), torch.zeros((2, 2, 64), dtype=dtype)
        v[0, 0, 0], v[0, 1, 0] = 3.5, 3.5 * (1 + 2 * torch.finfo(dtype).eps)
        cache = edge.cache()
        paged_append(cache, k.cuda(), v.cuda(), *edge.index())
        page = int(edge.table[0, 0])
        assert cache.v_scales[page].tolist() == [2.0 ** -7, 2.0 ** -6] and cache.k_scales[page].tolist() == [2.0 ** -100] * 2
        check_append(edge, cache, k, v, None, False)


def test_pages_that_are_none():
    """Table entries out of range, positions behind the table's row, lengths that do not fit: nothing outside is touched."""
    from moba_amd import paged_append
    for quantized in (True, False):
        batch = Batch([30, 0, 14], [40, 20, 4], 16, 2, 128, BF16, quantized, seed=2, spare=5)
        batch.table[0, 2], batch.table[0, 3], batch.table[1, 0] = -5, batch.pages[0].shape[0], 2 ** 31 - 1
        batch.table = batch.table[:, :4].contiguous()                      # (sequence 0's tokens from 64 on have no entry)
        k, v, q = batch.tensors(2, 2, 4)
        cache, inv_freq = batch.cache(), frequencies(64)
        got = paged_append(cache, k.cuda(), v.cuda(), *batch.index(), inv_freq=inv_freq.cuda(), query=q.cuda())
        check_append(batch, cache, k, v, inv_freq, False)
        check_query(batch, got, q, inv_freq, False)
        # fewer tokens than new ones: those before position 0 are nobody's
        short = Batch([0], [40], 16, 2, 128, BF16, quantized, seed=3)
        k, v = short.tensors(2, 2)
        table, _, cu = short.index()
        cache = short.cache()
        paged_append(cache, k.cuda(), v.cuda(), table, torch.tensor([10], dtype=torch.int32, device="cuda"), cu, inv_freq=inv_freq.cuda())
        short.new, short.cu, short.rows = [10], torch.tensor([0, 10]), 10
        check_append(short, cache, k[30:], v[30:], inv_freq, False)
        # row ranges that are none: the call ends, and the cache's neighbours are as they were
        for cu in ([5, 3], [-9, 60], [50, 50], [2 ** 31 - 1, -2 ** 31]):
            cache = short.cache()
            paged_append(cache, k.cuda(), v.cuda(), table, torch.tensor([10], dtype=torch.int32, device="cuda"),
                         torch.tensor(cu, dtype=torch.int32, device="cuda"), query=k.cuda())
            free = torch.ones(short.pages[0].shape[0], dtype=torch.bool)
            free[short.table[0, :1].long()] = False
            assert torch.equal(cache.v_pages.cpu().view(torch.uint8)[free], short.pages[1].view(torch.uint8)[free]), cu


def test_views():
    from moba_amd import paged_append
    batch = Batch([10, 3], [20, 9], 32, 2, 64, BF16, True, seed=6)
    g = torch.Generator().manual_seed(1)
    fused = torch.randn((29, 10, 64), generator=g).to(BF16).cuda()
    inv_freq = frequencies(32, "cuda")
    table, lengths, cu = batch.index()
    want = batch.cache()
    q, k, v = fused[:, :6], fused[:, 6:8], fused[:, 8:]
    turned = paged_append(want, k.contiguous(), v.contiguous(), table, lengths, cu, inv_freq=inv_freq, query=q.contiguous())
    wide = torch.full((2, 2 * table.shape[1]), -1, dtype=torch.int32, device="cuda")
    wide[:, ::2] = table
    big = torch.full((2, table.shape[1] + 7), -1, dtype=torch.int32, device="cuda")
    big[:, :table.shape[1]] = table
    for kk, vv, qq, tt in ((k, v, q, table), (k.transpose(0, 1).contiguous().transpose(0, 1), v, q, big[:, :table.shape[1]]),
                           (k, torch.cat([v, v], -1)[..., :64], q, wide[:, ::2]),
                           (k, torch.stack([v, v], -1)[..., 0], torch.stack([q, q], -1)[..., 1], table)):
        cache = batch.cache()
        got = paged_append(cache, kk, vv, tt, lengths, cu, inv_freq=inv_freq, query=qq)
        assert torch.equal(got, turned)
        assert torch.equal(cache.k_pages.view(torch.uint8), want.k_pages.view(torch.uint8)) and torch.equal(cache.v_scales, want.v_scales)
        assert torch.equal(cache.v_pages.view(torch.uint8), want.v_pages.view(torch.uint8)) and torch.equal(cache.k_scales, want.k_scales)


def test_nothing_to_append():
    from moba_amd import PagedKVCache, paged_append
    cache = PagedKVCache.empty(3, 2, head_dim=64, page_size=16)
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    none = torch.empty((0, 2, 64), dtype=BF16, device="cuda")
    some = torch.ones((4, 2, 64), dtype=BF16, device="cuda")
    assert paged_append(cache, none, none, ints(0, 1).view(1, 2), ints(5), ints(0, 0)) is None
    assert paged_append(cache, none, none, ints(0, 1).view(1, 2), ints(5), ints(0, 0), query=none).shape == (0, 2, 64)
    got = paged_append(cache, some, some, torch.empty((0, 2), dtype=torch.int32, device="cuda"), ints(), ints(0), query=some)
    assert not got.any()
    got = paged_append(cache, some, some, ints(0, 1, 2, 0).view(2, 2), ints(5, 0), ints(0, 0, 0), query=some)
    assert not got.any() and not cache.k_pages.float().any()
    assert cache.k_pages.dtype == E4M3


def test_a_cache_of_more_than_2_31_elements():
    from moba_amd import PagedKVCache, paged_append
    pages = 2 ** 31 // (8 * 256 * 128) + 3
    cache = PagedKVCache(torch.zeros((pages, 8, 256, 128), dtype=E4M3, device="cuda"), torch.zeros((pages, 8, 256, 128), dtype=E4M3, device="cuda"),
                         *(torch.ones((pages, 8), device="cuda") for _ in range(2)))
    k = torch.ones((300, 8, 128), dtype=BF16, device="cuda") * 3.5
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    paged_append(cache, k, k, ints(pages - 1, pages - 2).view(1, 2), ints(300), ints(0, 300))
    assert (cache.v_scales[-2:] == 2.0 ** -7).all()
    assert (cache.k_pages[-1].float() == 448).all() and (cache.v_pages[-2, :, :44].float() == 448).all()
    assert not cache.v_pages[-2, :, 44:].float().any() and not cache.k_pages[:2].float().any()


def test_graph_and_streams():
    """A captured step follows the lengths, the table and the new rows, and two streams work on two caches at once."""
    from moba_amd import paged_append
    batch = Batch([0, 50, 63], [1, 1, 1], 64, 2, 128, BF16, True, seed=8)
    inv_freq = frequencies(64, "cuda")
    table, lengths, cu = batch.index()
    k, v, q = (x.cuda() for x in batch.tensors(2, 2, 4))
    static, eager = batch.cache(), batch.cache()
    paged_append(batch.cache(), k, v, table, lengths, cu, inv_freq=inv_freq, query=q)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged_append(static, k, v, table, lengths, cu, inv_freq=inv_freq, query=q)
        lengths += 1
    lengths.copy_(batch.lengths)
    steps = lengths.clone()
    side = torch.cuda.Stream()
    for i in range(4):
        for x in (k, v, q):
            x.mul_(1.5)
        graph.replay()
        torch.cuda.synchronize()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = paged_append(eager, k, v, table, steps, cu, inv_freq=inv_freq, query=q)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(static.k_scales, eager.k_scales), i
        for name in ("k_pages", "v_pages"):
            assert torch.equal(getattr(static, name).view(torch.uint8), getattr(eager, name).view(torch.uint8)), (i, name)
        steps += 1
        if i == 1:   # a sequence leaves, another takes its place
            for t in (lengths, steps):
                t[1] = 1
    assert lengths.tolist() == steps.tolist()


@pytest.mark.parametrize("page", [16, 128])
def test_scales_that_held_tokens_may_have(page):
    """Far smaller than the new tokens need, so that their ratio is no 32-bit number; and others than paged_append's own: zero,
    negative, no power of two, smaller and larger than the new tokens'.  What the page holds stands for the same values as before."""
    from moba_amd import paged_append
    held = page - 5
    batch = Batch([held], [3], page, 8, 64, BF16, True, seed=17)
    page_id = int(batch.table[0, 0])
    # head:                       0          1          2       3    4       5      6       7
    scales = torch.tensor([2.0 ** -100, 2.0 ** -60, 2.0 ** -7, 0.0, -0.01, -300.0, 0.013, 77.7])
    grown = [True, True, False, True, True, False, True, False]
    for s in batch.scales:
        s[page_id] = scales
    for codes in batch.pages:                             # (all of magnitude 1 to 448, so that none is lost without reason)
        codes[page_id] = (codes[page_id].float().sign() * codes[page_id].float().abs().clamp(min=1)).to(E4M3)
    k, v = (x.clamp(-4, 4) for x in batch.tensors(8, 8))
    for x in (k, v):
        x[:, 0], x[:, 1] = x[:, 0] * 2.0 ** 70, x[:, 1] * 2.0 ** 120
        x[:, 2] = x[:, 2] * 0.1
        x[:, 3:7] = x[:, 3:7] * 20
    cache = batch.cache()
    paged_append(cache, k.cuda(), v.cuda(), *batch.index())
    for half, (pages, new, x) in enumerate(((cache.k_pages, cache.k_scales, k), (cache.v_pages, cache.v_scales, v))):
        codes, new = pages[page_id].cpu(), new[page_id].cpu()
        before, after = (c.double() * s[:, None, None].double() for c, s in ((batch.pages[half][page_id], scales), (codes, new)))
        for h in range(8):
            if not grown[h]:
                assert new[h] == scales[h] and torch.equal(codes[h, :held].view(torch.uint8), batch.pages[half][page_id, h, :held].view(torch.uint8)), h
            assert new[h].abs() * 448 * (1 + 2.0 ** -22) >= x[:, h].abs().max() and new[h].abs() >= scales[h].abs(), (h, new[h])
            # half a step of e4m3 of a normal number or of the smallest, and of the factors' 32 bits
            for got, want in ((after[h, :held], before[h, :held]), (after[h, held:held + 3], x[:, h].double())):
                bound = torch.maximum(2.0 ** -4 * want.abs(), 2.0 ** -10 * new[h].double().abs()) * 1.001
                assert ((got - want).abs() <= bound).all(), (half, h, new[h], ((got - want).abs() / bound).max())


@pytest.mark.parametrize("quantized", [True, False])
def test_derivatives_that_there_are_none_of(quantized):
    import torch.autograd.forward_ad as fwd
    from moba_amd import PagedKVCache, paged_append, paged_attention
    batch = Batch([10], [2], 16, 2, 64, BF16, quantized)
    k, v, q = (x.cuda() for x in batch.tensors(2, 2, 4))
    index, f = batch.index(), frequencies(32, "cuda")
    names = ("k_scales", "v_scales") if quantized else ("k_pages", "v_pages")
    changed = lambda name, change: PagedKVCache(**{  # noqa: E731
        n: change(x) if n == name else x for n, x in vars(batch.cache()).items()})
    for name in names:
        cache = changed(name, lambda x: x.requires_grad_())
        for call in (lambda: paged_append(cache, k, v, *index), lambda: paged_attention(q, cache, *index)):
            with pytest.raises(RuntimeError, match="no gradients"):
                call()
            with torch.no_grad():
                call()
    with pytest.raises(RuntimeError, match="no gradients"):
        paged_append(batch.cache(), k, v, *index, inv_freq=f.clone().requires_grad_())
    with fwd.dual_level():
        dual = lambda x: fwd.make_dual(x, torch.ones_like(x))  # noqa: E731
        for name in names:
            cache = changed(name, dual)
            for call in (lambda: paged_append(cache, k, v, *index), lambda: paged_attention(q, cache, *index)):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call()
        for args in ((dual(k), v, q, f), (k, dual(v), q, f), (k, v, dual(q), f), (k, v, q, dual(f))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                paged_append(batch.cache(), *args[:2], *index, query=args[2], inv_freq=args[3])
        with pytest.raises(RuntimeError, match="forward-mode"):
            paged_attention(dual(q), batch.cache(), *index)


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("quantized", [True, False])
def test_autograd_learns_what_was_written(quantized, native, monkeypatch):
    """A graph that kept the cache's tensors for its backward pass says that they have changed."""
    from moba_amd import _lib, paged_append, paged_attention
    if not native:
        monkeypatch.setattr(_lib.host(), "paged_append", lambda *a: NotImplemented)
    batch = Batch([10], [2], 16, 2, 64, BF16, quantized)
    k, v, q = (x.cuda() for x in batch.tensors(2, 2, 4))
    index, cache = batch.index(), batch.cache()
    fields = [x for x in vars(cache).values() if x is not None]
    kept = cache.v_scales if quantized else cache.v_pages
    leaf = torch.ones_like(kept, requires_grad=True)
    loss = (leaf * kept).sum()
    before = [x._version for x in fields]
    paged_attention(q, cache, *index)
    assert [x._version for x in fields] == before
    paged_append(cache, k, v, *index)
    assert [x._version for x in fields] == [n + 1 for n in before]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        cache = batch.cache()
        paged_append(cache, k, v, *index)
    paged_append(cache, k, v, *index)
    check_append(batch, cache, k.cpu(), v.cpu(), None, False)
