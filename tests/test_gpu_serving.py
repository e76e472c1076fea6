"""What the operators of serving have in common: their native calls and the general path beside these, padded batches, refusals of tensors
on the GPU."""

import ctypes

import pytest
import torch

from paged_reference import Batch

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16
NAMES = ("paged_reserve", "paged_release", "paged_prefix_attention", "paged_key_sums", "paged_select_blocks", "paged_block_attention")


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prefixed(quantized, d, dtype):
    """Three sequences, the first two of which share six pages of 32 tokens."""
    batch = Batch([200, 195, 70], [1, 9, 4], 32, 2, d, dtype, quantized, seed=3)
    batch.table[1, :6] = batch.table[0, :6]
    return batch


def everything(batch, q, index=None, groups=None, pool=None):
    """Every operator once: all that they return or write."""
    import moba_amd as m
    cache, index = batch.cache(), index or batch.index()
    cu_groups, shared = groups or (ints(0, 2), ints(192))
    sums = cache.key_sums()
    m.paged_key_sums(cache, sums, *index, batch.rows)
    blocks = m.paged_select_blocks(q, sums, *index, batch.page, 64, 3)
    out = [sums, blocks, m.paged_block_attention(q, cache, blocks, *index, 64), m.paged_block_attention(q, cache, blocks, *index, 64, scaling=0.2),
           m.paged_prefix_attention(q, cache, *index, cu_groups, shared), m.paged_prefix_attention(q, cache, *index, cu_groups, shared, scaling=-0.2)]
    pool = pool or m.PagePool.full(20, 16)
    table, lengths = torch.full((3, 6), -1, dtype=torch.int32, device="cuda"), ints(0, 0, 0)
    out += m.paged_reserve(pool, table, lengths, ints(5, 40, 16), 64)
    out += [table.clone(), lengths.clone(), pool.free_count.clone()]
    m.paged_release(pool, table, lengths, ints(5, 3, 0))
    return out + [table, lengths, pool.free_count, pool.free_pages]


@pytest.mark.parametrize("quantized,d,dtype", [(True, 128, BF16), (False, 64, FP16)])
def test_the_general_path_gives_the_same(monkeypatch, quantized, d, dtype):
    """What the native calls leave to the Python path -- tensors to be copied first -- is computed the same."""
    from moba_amd import _lib
    host, batch = _lib.host(), prefixed(quantized, d, dtype)
    q = batch.tensors(4)[0].cuda()
    want = everything(batch, q)
    assert all(torch.isfinite(x).all() for x in want[2:6])
    native = {name: getattr(host, name) for name in NAMES}
    # (each wrapper asks once, checks, and asks again)
    for name, f in native.items():
        calls = [0]

        def second(*a, f=f, calls=calls):
            calls[0] += 1
            return NotImplemented if calls[0] % 2 else f(*a)
        monkeypatch.setattr(host, name, second)
    assert all(torch.equal(a, b) for a, b in zip(want, everything(batch, q)))


def test_parameters_and_subclasses():
    class Mine(torch.Tensor):
        pass
    batch = prefixed(True, 128, BF16)
    q = batch.tensors(4)[0].cuda()
    want = everything(batch, q)
    for x in (torch.nn.Parameter(q, requires_grad=False), q.as_subclass(Mine)):
        got = everything(batch, x, tuple(t.as_subclass(Mine) for t in batch.index()), tuple(t.as_subclass(Mine) for t in (ints(0, 2), ints(192))))
        assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("quantized,d,dtype", [(True, 64, FP16), (False, 128, BF16)])
def test_a_padded_batch(quantized, d, dtype):
    """Sequences without tokens behind the last, rows and groups that belong to none, index tensors anywhere in memory: the rows of the
    others are the same."""
    import moba_amd as m
    batch = prefixed(quantized, d, dtype)
    q = batch.tensors(4)[0].cuda()
    want = everything(batch, q)
    place = lambda t: torch.cat([t.new_full((1,), 99), t.flatten()])[1:].view_as(t)  # noqa: E731  (4 bytes off)
    table, lengths, cu = batch.index()
    index = (place(torch.cat([table, torch.full((70, table.shape[1]), -1, dtype=torch.int32, device="cuda")])),
             place(torch.cat([lengths, lengths.new_zeros(70)])), place(torch.cat([cu, cu[-1:].expand(70)])))
    groups, shared = place(ints(0, 2, 73, 73)), place(ints(192, 0, 64))
    wide, rows = torch.cat([q, q[:5]]), batch.rows
    cache, sums = batch.cache(), batch.cache().key_sums()
    m.paged_key_sums(cache, sums, *index, rows + 5)
    assert torch.equal(sums, want[0])
    blocks = m.paged_select_blocks(wide, sums, *index, batch.page, 64, 3)
    assert torch.equal(blocks[:rows], want[1]) and (blocks[rows:] == -1).all()
    for got, w in ((m.paged_block_attention(wide, cache, blocks, *index, 64), want[2]),
                   (m.paged_prefix_attention(wide, cache, *index, groups, shared), want[4])):
        # (other runs of the keys: other sums of 32 bits, rounded once)
        assert ((got[:rows].double() - w.double()).abs() <= torch.finfo(dtype).eps * w.double().abs() + 2.0 ** -14 * w.double().abs().amax()).all()
        assert not got[rows:].any()


def test_gradients_are_refused():
    import moba_amd as m
    from torch.autograd import forward_ad
    batch = prefixed(False, 64, BF16)
    q, cache, index = batch.tensors(4)[0].cuda(), batch.cache(), batch.index()
    sums = cache.key_sums()
    blocks = m.paged_select_blocks(q, sums, *index, 32, 64, 3)
    calls = (lambda x: m.paged_select_blocks(x, sums, *index, 32, 64, 3), lambda x: m.paged_block_attention(x, cache, blocks, *index, 64),
             lambda x: m.paged_prefix_attention(x, cache, *index, ints(0, 2), ints(192)))
    for call in calls:
        with pytest.raises(RuntimeError, match="gradients"):
            call(q.clone().requires_grad_())
        with forward_ad.dual_level(), pytest.raises(RuntimeError, match="tangent"):
            call(forward_ad.make_dual(q, q))
        with torch.no_grad():
            assert torch.equal(call(q.clone().requires_grad_()), call(q))
        with torch.inference_mode():
            assert torch.equal(call(q.clone()), call(q))
    with pytest.raises(RuntimeError):
        m.paged_key_sums(cache, sums.clone().requires_grad_(), *index, batch.rows)


def test_the_native_calls_let_other_threads_run():
    """In the entry points' places stands CPython's own PyGILState_Check, whose answer -- 1 with the lock -- would be an error code."""
    from moba_amd import _lib
    batch = prefixed(True, 128, BF16)
    q, check = batch.tensors(4)[0].cuda(), ctypes.pythonapi.PyGILState_Check
    want = everything(batch, q)
    try:
        _lib.bind_serving(_lib.host(), **{"moba_" + name: check for name in NAMES})
        assert len(everything(batch, q)) == len(want)
    finally:
        _lib.bind_serving(_lib.host())
    assert all(torch.equal(a, b) for a, b in zip(want, everything(batch, q)))


def test_wrong_tensors_are_told_apart():
    """Tensors on the GPU that do not fit are refused with a word of what is wrong, by every call."""
    import moba_amd as m
    batch = prefixed(True, 128, BF16)
    q, cache, (table, lengths, cu) = batch.tensors(4)[0].cuda(), batch.cache(), batch.index()
    sums, blocks, pool = cache.key_sums(), torch.zeros((batch.rows, 4, 2), dtype=torch.int32, device="cuda"), m.PagePool.full(9, 16)
    wrong = [((table.long(), lengths, cu), TypeError), ((table, lengths[:2], cu), ValueError), ((table, lengths, cu[:2]), ValueError),
             ((table[0], lengths, cu), ValueError), ((table.cpu(), lengths, cu), ValueError), ((table[:, :0], lengths, cu), ValueError)]
    for index, error in wrong:
        for call in (lambda: m.paged_prefix_attention(q, cache, *index, ints(0, 2), ints(192)), lambda: m.paged_key_sums(cache, sums, *index, 9),
                     lambda: m.paged_select_blocks(q, sums, *index, 32, 64, 3), lambda: m.paged_block_attention(q, cache, blocks, *index, 64)):
            with pytest.raises(error):
                call()
    good = (table, lengths, cu)
    for call, error in ((lambda: m.paged_prefix_attention(q[:, :3], cache, *good, ints(0, 2), ints(192)), ValueError),
                        (lambda: m.paged_prefix_attention(q.float(), cache, *good, ints(0, 2), ints(192)), TypeError),
                        (lambda: m.paged_prefix_attention(q, cache, *good, ints(0, 2, 3), ints(192)), ValueError),
                        (lambda: m.paged_prefix_attention(q, cache, *good, ints(0, 2).cpu(), ints(192)), ValueError),
                        (lambda: m.paged_key_sums(cache, sums[1:], *good, 9), ValueError),
                        (lambda: m.paged_key_sums(cache, sums, *good, -1), ValueError),
                        (lambda: m.paged_key_sums(cache, sums.double(), *good, 9), TypeError),
                        (lambda: m.paged_select_blocks(q, sums, *good, 32, 48, 3), ValueError),
                        (lambda: m.paged_select_blocks(q, sums, *good, 32, 64, 65), ValueError),
                        (lambda: m.paged_select_blocks(q, sums, *good, 8, 64, 3), ValueError),
                        (lambda: m.paged_select_blocks(q, sums, *good, 32, 64, 0), ValueError),
                        (lambda: m.paged_block_attention(q, cache, blocks[1:], *good, 64), ValueError),
                        (lambda: m.paged_block_attention(q, cache, blocks.long(), *good, 64), TypeError),
                        (lambda: m.paged_block_attention(q, cache, blocks, *good, 0), ValueError),
                        (lambda: m.paged_reserve(pool, table, lengths, lengths.long(), 9), TypeError),
                        (lambda: m.paged_reserve(pool, table, lengths, lengths[:1], 9), ValueError),
                        (lambda: m.paged_reserve(pool, table, lengths, lengths, -1), ValueError),
                        (lambda: m.paged_reserve(pool, table.cpu(), lengths, lengths, 9), ValueError),
                        (lambda: m.paged_release(pool, table, lengths[::2], lengths[::2]), ValueError)):
        with pytest.raises(error):
            call()
