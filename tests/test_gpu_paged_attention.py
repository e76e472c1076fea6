"""paged_attention on the GPU against softmax attention in 64 bits on what the pages hold."""

import pytest
import torch

from paged_reference import Batch, attended, check_append, check_attention
from rotary_reference import frequencies

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16

CASES = [  # old, new, page, heads, kv heads, head_dim, dtype, quantized, rows behind
    ([0], [1], 64, 4, 1, 128, BF16, True, 0),
    ([0], [1], 16, 1, 1, 64, FP16, False, 0),
    ([4096], [1], 64, 32, 8, 128, BF16, True, 0),
    ([4095], [1], 64, 32, 8, 128, BF16, False, 0),
    ([127, 128, 129, 31, 32, 0, 15, 16], [1] * 8, 16, 6, 2, 128, FP16, True, 0),
    ([127, 128, 129, 31, 32, 0, 15, 16], [1] * 8, 32, 6, 2, 64, BF16, True, 3),
    ([127, 128, 129, 31, 32, 0, 15, 16], [1] * 8, 128, 5, 1, 64, FP16, False, 0),
    ([300, 5, 2000, 77], [1, 0, 3, 8], 256, 12, 4, 128, BF16, True, 2),
    ([300, 5, 2000, 77], [1, 0, 3, 8], 64, 12, 4, 128, FP16, False, 2),
    ([50, 0, 1000], [20, 33, 5], 64, 7, 1, 128, FP16, True, 0),             # more rows than a group has
    ([50, 0, 1000], [20, 33, 5], 16, 40, 1, 64, BF16, False, 0),            # more heads on one than a group has rows
    ([10 * i for i in range(70)], [1, 2, 0, 1, 1] * 14, 16, 4, 2, 64, BF16, True, 0),   # more sequences than a wave has lanes
    ([70000, 100], [1, 1], 64, 8, 2, 128, BF16, True, 0),                   # runs of more keys than pages are looked up at a time
    ([70000], [2], 16, 4, 4, 64, FP16, False, 0),
    ([0], [130], 32, 4, 2, 128, BF16, False, 0),
    ([100, 3, 0, 500], [200, 1, 129, 9], 64, 8, 2, 128, BF16, True, 1),     # many rows and few in one batch
    ([100, 3, 0, 500], [200, 1, 129, 9], 16, 8, 2, 64, FP16, True, 0),
    ([100, 3, 0, 500], [200, 1, 129, 9], 256, 6, 2, 128, FP16, False, 0),
    ([100, 3, 0, 500], [200, 1, 129, 9], 32, 9, 3, 64, BF16, False, 0),
    ([3000], [40], 16, 4, 1, 128, FP16, True, 0),                           # many rows, few groups: several runs each
    ([3001, 2222], [33, 70], 128, 5, 5, 128, BF16, False, 0),
    ([63], [65], 16, 1, 1, 128, BF16, True, 0),
    ([40, 10], [560, 45], 64, 30, 2, 64, BF16, True, 1),                    # more rows than the merge has waves for, an odd share of heads
]


@pytest.mark.parametrize("old,new,page,heads,kv_heads,d,dtype,quantized,behind", CASES)
def test_attention(old, new, page, heads, kv_heads, d, dtype, quantized, behind):
    from moba_amd import paged_attention
    print("attend", old[:6], new[:6], page, heads, kv_heads, d, dtype, quantized, behind, flush=True)
    batch = Batch(old, new, page, kv_heads, d, dtype, quantized, seed=page + d + len(old), pad_rows=behind)
    q, = batch.tensors(heads)
    cache, index = batch.cache(), batch.index()
    got = paged_attention(q.cuda(), cache, *index)
    check_attention(batch, got, q)
    assert torch.equal(got, paged_attention(q.cuda(), cache, *index))          # the same bits every time
    check_attention(batch, paged_attention(q.cuda(), cache, *index, scaling=0.31, max_new=max(new)), q, 0.31)
    check_attention(batch, paged_attention(q.cuda(), cache, *index, max_new=0), q)   # (a hint, whatever it says)


def test_either_type_on_8_bit_pages():
    from moba_amd import paged_attention
    batch = Batch([500, 3], [1, 2], 32, 2, 64, BF16, True, seed=1)
    for dtype in (BF16, FP16):
        q = batch.tensors(6)[0].to(dtype)
        check_attention(batch, paged_attention(q.cuda(), batch.cache(), *batch.index()), q)


@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("d", [64, 128])
def test_large_scores_and_scales(quantized, d):
    """Scores of hundreds, scales of every size beside each other, negative and zero softmax scales."""
    from moba_amd import paged_attention
    batch = Batch([700, 40, 200], [1, 3, 35], 16, 2, d, BF16, quantized, seed=2)
    if quantized:
        batch.scales[1] *= 2.0 ** torch.randint(-60, 60, batch.scales[1].shape, generator=batch.g).float()
    else:
        batch.pages[1][::2] *= 2.0 ** 40
    q = batch.tensors(4)[0] * 30
    for scaling in (None, -0.1, 0.0, 1.0):
        check_attention(batch, paged_attention(q.cuda(), batch.cache(), *batch.index(), scaling=scaling), q, scaling)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_any_scales(dtype):
    """Scales that paged_append does not make: no powers of two, negative ones, zero."""
    from moba_amd import paged_attention
    batch = Batch([300, 40, 90], [1, 3, 70], 16, 2, 128, dtype, True, seed=7)
    for s in batch.scales:
        s *= torch.rand(s.shape, generator=batch.g) + 0.5
        s[::5] *= -1
        s[3::7] = 0
    q, = batch.tensors(8)
    for scaling in (None, -0.05):
        check_attention(batch, paged_attention(q.cuda(), batch.cache(), *batch.index(), scaling=scaling), q, scaling)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("d", [64, 128])
def test_first_keys_that_say_nothing_of_the_others(d, quantized, dtype):
    """Many rows whose first keys have no page, or scores far above or below those that follow."""
    from moba_amd import paged_attention
    for change in ("none", "above", "below"):
        batch = Batch([150, 0, 300], [40, 90, 17], 16, 2, d, dtype, quantized, seed=9)
        q, = batch.tensors(8)
        q, keys = q.abs() * 40, batch.pages[0]
        if change == "none":
            batch.table[0, :3], batch.table[1, :2], batch.table[2, 0] = -1, -1, -1
        else:
            first = [int(batch.table[b, i]) for b in range(3) for i in range(2)]
            for page in range(keys.shape[0]):     # scores of some hundreds of either sign, or small
                sign = 1 if change == "above" else -1
                keys[page] = (keys[page].float().abs() * (sign if page in first else 0.05)).to(keys.dtype)
        check_attention(batch, paged_attention(q.cuda(), batch.cache(), *batch.index()), q)


@pytest.mark.parametrize("quantized", [True, False])
def test_values_that_are_not_finite(quantized):
    """They reach the rows that see them; what lies behind a sequence's end, or in other sequences' pages, reaches nobody."""
    from moba_amd import paged_attention
    for d, dtype in ((128, BF16), (64, FP16)):
        batch = Batch([200, 70, 9, 33], [1, 6, 1, 40], 32, 2, d, dtype, quantized, seed=3)
        nan, pages = float("nan"), batch.pages
        for b, (o, c) in enumerate(zip(batch.old, batch.new)):                     # behind the end, all sequences
            last = int(batch.table[b, (o + c) // 32])
            if last >= 0:
                for x in pages:
                    x[last, :, (o + c) % 32:] = nan
        used = set(batch.table.flatten().tolist())
        for page in set(range(pages[0].shape[0])) - used:
            pages[0][page], pages[1][page] = nan, nan
        q, = batch.tensors(6)
        check_attention(batch, paged_attention(q.cuda(), batch.cache(), *batch.index()), q)
        # a value of sequence 1's fourth new token (position 73): rows 4, 5 and 6 of the batch see it, 1 to 3 do not
        page, slot = int(batch.table[1, 73 // 32]), 73 % 32
        pages[1][page, 1, slot, 5] = nan if quantized else float("inf")
        check_attention(batch, paged_attention(q.cuda(), batch.cache(), *batch.index()), q)
        # and one of its keys, other head
        pages[0][page, 0, slot, 7] = nan
        # the same among many rows: sequence 3's eleventh new token
        page, slot = int(batch.table[3, 43 // 32]), 43 % 32
        pages[1][page, 0, slot, 9], pages[0][page, 1, slot, 60] = nan, nan
        got = paged_attention(q.cuda(), batch.cache(), *batch.index())
        check_attention(batch, got, q)
        assert got[4:7, :3].isnan().all() and got[:4, :3].isfinite().all() and got[7:18].isfinite().all() and got[18:, 3:].isnan().all()


@pytest.mark.parametrize("d,dtype", [(128, BF16), (64, BF16), (128, FP16), (64, FP16)])
def test_scores_that_are_not_finite(d, dtype):
    """Infinite keys and queries, NaN among the queries: NaN in the rows whose softmax is none, and in no others; a key with the
    score minus infinity counts for nothing."""
    from moba_amd import paged_attention
    batch = Batch([300, 50, 7], [6, 60, 1], 16, 2, d, dtype, False, seed=14)
    q, = batch.tensors(6)
    for b, position, head, sign in ((0, 303, 0, 1), (1, 80, 1, -1), (0, 17, 1, 1), (2, 3, 0, -1)):
        batch.pages[0][int(batch.table[b, position // 16]), head, position % 16, 9] = sign * float("inf")
    q[2, 1, 4], q[20, 5, 0], q[40, 2, 3], q[41, 0, 8] = float("nan"), float("inf"), float("nan"), -float("inf")
    got = paged_attention(q.cuda(), batch.cache(), *batch.index())
    want = attended(batch, q)[0]
    assert want.isnan().any() and not want.isnan().all((1, 2)).any()
    got, fine = got.cpu().double(), want.isfinite()
    assert torch.equal(got.isnan(), want.isnan())
    # half a step of the result and of a probability, of many rows one element; 2^-10: 2 * (d + 12) * 2^-24 of a score's size, at
    # most 11 or so, and 2^-15, of the largest value
    tolerance = torch.finfo(dtype).eps / 2 * 1.001 * (want[fine].abs().max() + batch.pages[1].abs().max().double()) + 2.0 ** -10
    assert ((got - want).abs()[fine] <= tolerance).all()


@pytest.mark.parametrize("quantized", [True, False])
def test_tables_that_do_not_fit(quantized):
    """Entries that are no page, lengths beyond the table or below the number of new tokens, row ranges that are none."""
    from moba_amd import paged_attention
    batch = Batch([100, 0, 300, 40, 200], [2, 20, 1, 3, 50], 16, 2, 64, BF16, quantized, seed=4)
    batch.table[4, 3], batch.table[4, 9] = -7, 2 ** 30
    batch.table[0, 1], batch.table[0, 4], batch.table[1], batch.table[2, 5:] = -1, batch.pages[0].shape[0], 2 ** 31 - 1, -2 ** 31
    q, = batch.tensors(4)
    got = paged_attention(q.cuda(), batch.cache(), *batch.index())
    check_attention(batch, got, q)
    assert not got[2:22].any()
    cut = Batch([100], [2], 16, 2, 64, BF16, quantized, seed=5)
    cut.table = cut.table[:, :3].contiguous()                   # 48 of 102 tokens
    q, = cut.tensors(4)
    check_attention(cut, paged_attention(q.cuda(), cut.cache(), *cut.index()), q)
    table, _, cu = cut.index()
    lengths = lambda n: torch.tensor([n], dtype=torch.int32, device="cuda")  # noqa: E731
    got = paged_attention(q.cuda(), cut.cache(), table, lengths(1), cu)       # its first new token lies before position 0
    cut.old, cut.new = [0], [1]
    check_attention(cut, got[1:], q[1:])
    assert not got[0].any()
    for n in (0, -5):
        assert not paged_attention(q.cuda(), cut.cache(), table, lengths(n), cu).any()
    assert paged_attention(q.cuda(), cut.cache(), table, lengths(2 ** 31 - 1), cu).isfinite().all()
    for bad in ([1, 0], [-7, 900], [2 ** 31 - 1, -2 ** 31]):
        paged_attention(q.cuda(), cut.cache(), table, lengths(30), torch.tensor(bad, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()


def test_views_and_nothing():
    from moba_amd import PagedKVCache, paged_attention
    batch = Batch([100, 30], [1, 4], 16, 2, 128, BF16, True, seed=6)
    q = batch.tensors(6)[0].cuda()
    cache, (table, lengths, cu) = batch.cache(), batch.index()
    want = paged_attention(q, cache, table, lengths, cu)
    fused = torch.cat([q, q[:, :2]], 1)
    odd = torch.empty(q.numel() + 1, dtype=BF16, device="cuda")[1:].view_as(q).copy_(q)
    for view in (fused[:, :6], q.transpose(0, 1).contiguous().transpose(0, 1), torch.stack([q, q], -1)[..., 0], odd):
        assert torch.equal(paged_attention(view, cache, table, lengths, cu), want)
    wide = torch.full((2, 2 * table.shape[1]), -1, dtype=torch.int32, device="cuda")
    wide[:, ::2] = table
    assert torch.equal(paged_attention(q, cache, wide[:, ::2], lengths, cu), want)
    assert paged_attention(q[:0], cache, table, lengths, cu).shape == (0, 6, 128)
    empty = torch.empty((0, 2), dtype=torch.int32, device="cuda")
    assert not paged_attention(q, cache, empty, lengths[:0], cu[:1]).any()
    shared = table[:1].expand(2, -1)                                        # one table under two sequences
    got = paged_attention(q[:2], cache, shared, lengths[:1].expand(2), torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda"))
    same = paged_attention(q[:2], cache, shared.contiguous(), lengths[:1].repeat(2), torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda"))
    assert torch.equal(got, same) and torch.equal(got[0], want[0])
    assert not paged_attention(q, PagedKVCache.empty(2, 2, page_size=16), table, torch.zeros_like(lengths), cu).any()


def test_a_cache_of_more_than_2_31_elements():
    from moba_amd import PagedKVCache, paged_attention
    E4M3 = torch.float8_e4m3fn
    pages = 2 ** 31 // (8 * 256 * 128) + 2
    zeros = lambda: torch.zeros((pages, 8, 256, 128), dtype=E4M3, device="cuda")  # noqa: E731
    cache = PagedKVCache(zeros(), zeros(), *(torch.ones((pages, 8), device="cuda") for _ in range(2)))
    for i, page in enumerate((pages - 1, 0)):
        cache.v_pages[page] = torch.full((8, 256, 128), 2.0 + 2 * i, device="cuda").to(E4M3)
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    got = paged_attention(torch.ones((1, 8, 128), dtype=BF16, device="cuda"), cache, ints(pages - 1, 0).view(1, 2), ints(512), ints(0, 1))
    assert (got == 3).all()


def test_graph_and_streams():
    """A captured call follows lengths, table and row ranges; two calls at once have workspaces of their own."""
    from moba_amd import paged_attention
    batch = Batch([1000, 50, 63, 400], [1, 1, 1, 1], 64, 2, 128, BF16, True, seed=8)
    other = Batch([3000, 5], [2, 2], 64, 2, 128, BF16, True, seed=9)
    q, oq = batch.tensors(8)[0].cuda(), other.tensors(8)[0].cuda()
    cache, (table, lengths, cu) = batch.cache(), batch.index()
    o_cache, o_index = other.cache(), other.index()
    want_other = paged_attention(oq, o_cache, *o_index)
    torch.cuda.synchronize()
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged_attention(q, cache, table, lengths, cu)
    with torch.cuda.graph(second):
        out_other = paged_attention(oq, o_cache, *o_index)
    side = torch.cuda.Stream()
    for i, (lens, rows) in enumerate((([1001, 51, 64, 401], [0, 1, 2, 3, 4]), ([1, 51, 1000, 2], [0, 1, 2, 3, 4]),
                                      ([900, 51, 0, 401], [0, 2, 3, 3, 4]), ([300, 300, 300, 300], [0, 0, 0, 4, 4]))):
        table.copy_(batch.table[[i % 4, 0, 0, 3]] if i else batch.table)
        lengths.copy_(torch.tensor(lens))
        cu.copy_(torch.tensor(rows))
        torch.cuda.synchronize()
        side.wait_stream(torch.cuda.current_stream())
        graph.replay()
        with torch.cuda.stream(side):
            second.replay()
            eager_other = paged_attention(oq, o_cache, *o_index)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        assert torch.equal(out, paged_attention(q, cache, table, lengths, cu)), i
        assert torch.equal(out_other, want_other) and torch.equal(eager_other, want_other), i


@pytest.mark.parametrize("quantized", [False, True])
def test_graph_of_many_rows(quantized):
    """Pieces of prompts and single tokens change places between replays."""
    from moba_amd import paged_attention
    batch = Batch([900, 300, 0], [150, 40, 1], 16, 2, 128, BF16, quantized, seed=13, pad_rows=9)
    q = batch.tensors(8)[0]
    cache, (table, lengths, cu) = batch.cache(), batch.index()
    given = q.cuda()
    paged_attention(given, cache, table, lengths, cu)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged_attention(given, cache, table, lengths, cu)
    for old, new in (([900, 300, 0], [150, 40, 1]), ([1049, 0, 0], [1, 190, 1]), ([0, 339, 0], [0, 1, 0]), ([849, 100, 1], [200, 0, 0])):
        batch.old, batch.new = old, new
        rows = [0, new[0], new[0] + new[1], sum(new)]
        lengths.copy_(torch.tensor([o + n for o, n in zip(old, new)]))
        cu.copy_(torch.tensor(rows))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, paged_attention(given, cache, table, lengths, cu))
        check_attention(batch, out, q)


@pytest.mark.parametrize("quantized", [False, True])
def test_serving(quantized):
    """As they are used together: a prompt normed, rotated, attended by the packed operator and appended to the cache, a second
    prompt in two pieces, then tokens one at a time; every step's cache and attention against the definitions."""
    from moba_amd import moba_attn_varlen_gqa, paged_append, paged_attention, qk_norm_rope
    heads, kv_heads, d, page = 4, 2, 128, 32
    batch = Batch([0, 0], [150, 40], page, kv_heads, d, BF16, quantized, seed=12, spare=12, noise=0.0)
    batch.table = torch.randperm(batch.pages[0].shape[0] // 2 * 2, generator=batch.g).to(torch.int32).view(2, -1)
    inv_freq = frequencies(64)
    w = [(1 + 0.2 * torch.randn(d, generator=batch.g)).to(BF16).cuda() for _ in range(2)]
    cache = batch.cache()
    for step in range(6):
        batch.new = [[150, 40], [0, 30], [1, 1], [1, 1], [1, 1], [0, 1]][step]
        batch.rows = sum(batch.new)
        batch.lengths = torch.tensor([o + n for o, n in zip(batch.old, batch.new)], dtype=torch.int32)
        batch.cu = torch.tensor([0, batch.new[0], batch.rows], dtype=torch.int32)
        q, k, v = (x.cuda() for x in batch.tensors(heads, kv_heads, kv_heads))
        at = torch.tensor(batch.positions()).cuda()
        q, k = qk_norm_rope(q, k, at, inv_freq.cuda(), *w)
        paged_append(cache, k, v, *batch.index())
        check_append(batch, cache, k.cpu(), v.cpu(), None, False)
        batch.pages = [cache.k_pages.cpu(), cache.v_pages.cpu()]
        if quantized:
            batch.scales = [cache.k_scales.cpu(), cache.v_scales.cpu()]
        out = paged_attention(q, cache, *batch.index(), max_new=max(batch.new))
        check_attention(batch, out, q.cpu())
        if step == 0 and not quantized:
            # the packed operator, one chunk a sequence: the same attention (tolerance of the operator's own tests)
            packed = moba_attn_varlen_gqa(q, k, v, batch.cu.cuda(), 150, 1024, 3)
            assert (packed.float() - out.float()).abs().max() < 2e-2
        batch.old = [o + n for o, n in zip(batch.old, batch.new)]


def test_the_general_path_gives_the_same(monkeypatch):
    """What the native calls leave to the Python path -- tensors to be copied first -- is computed the same."""
    from moba_amd import _lib, paged_append, paged_attention
    host = _lib.host()
    native = {name: getattr(host, name) for name in ("paged_append", "paged_attention")}
    for quantized, d in ((True, 128), (False, 64)):
        batch = Batch([100, 3, 70], [1, 50, 4], 32, 2, d, BF16, quantized, seed=3)
        q, k, v = (x.cuda() for x in batch.tensors(6, 2, 2))
        index, inv_freq, got = batch.index(), frequencies(16, "cuda"), []
        for general in (False, True):
            for name, f in native.items():
                monkeypatch.setattr(host, name, (lambda *a: NotImplemented) if general else f)
            cache = batch.cache()
            turned = paged_append(cache, k, v, *index, inv_freq=inv_freq, query=q, interleaved=True)
            got.append([turned, cache.k_pages.view(torch.uint8), cache.v_pages.view(torch.uint8), paged_attention(turned, cache, *index),
                        paged_attention(turned, cache, *index, scaling=0.2, max_new=50)])
        assert all(torch.equal(a, b) for a, b in zip(*got))
        fields = (cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales)
        append = lambda k=k, v=v, i=index, f=inv_freq, q=q: native["paged_append"](*fields, k, v, *i, f, q, False)  # noqa: E731
        attend = lambda q=q, i=index, hint=None: native["paged_attention"](*fields, q, *i, None, hint)  # noqa: E731
        short, flat = (index[0], index[1][:2], index[2]), (index[0][0], *index[1:])
        for args in (dict(k=k[:5]), dict(k=k.cpu()), dict(v=v.float()), dict(q=q[:, :0]), dict(q=q[:4]), dict(f=inv_freq[:3]),
                     dict(i=short), dict(i=flat), dict(k=k[..., ::2]), dict(k=k[:0], v=v[:0], q=q[:0])):
            assert append(**args) is NotImplemented, args.keys()
        for args in (dict(q=q[:0]), dict(q=q[:, :5]), dict(q=q.cpu()), dict(q=q[..., ::2]), dict(i=short), dict(i=flat), dict(hint=-1)):
            assert attend(**args) is NotImplemented, args.keys()


def test_the_native_calls_let_other_threads_run():
    """In the entry points' places stands CPython's own PyGILState_Check, whose answer -- 1 with the lock -- would be an error code."""
    import ctypes
    from moba_amd import _lib, paged_append, paged_attention
    batch = Batch([10], [1], 16, 2, 64, BF16, True)
    q, k = (x.cuda() for x in batch.tensors(4, 2))
    check = ctypes.pythonapi.PyGILState_Check
    try:
        _lib.bind_layer(_lib.host(), moba_paged_append=check, moba_paged_attention=check)
        assert paged_append(batch.cache(), k, k, *batch.index(), query=q).shape == q.shape
        assert paged_attention(q, batch.cache(), *batch.index()).shape == q.shape
    finally:
        _lib.bind_layer(_lib.host())
    check_attention(batch, paged_attention(q, batch.cache(), *batch.index()), q.cpu())
