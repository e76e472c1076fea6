"""What the operators of serving and their entry points refuse, before anything is launched (no GPU)."""

import ctypes

import pytest
import torch

from test_paged_host import make

BF16, I32 = torch.bfloat16, torch.int32


def test_the_pool_refuses():
    from moba_amd import PagePool
    pool = PagePool.full(5, 16, device="cpu")
    assert pool.free_pages.tolist() == [4, 3, 2, 1, 0] and pool.free_count.tolist() == [5] and pool.page_size == 16
    some, one = torch.zeros(4, dtype=I32), torch.zeros(1, dtype=I32)
    for error, args in [(TypeError, (some.long(), one, 16)), (TypeError, (some, one.float(), 16)), (ValueError, (some.view(2, 2), one, 16)),
                        (ValueError, (some[::2], one, 16)), (ValueError, (some[:0], one, 16)), (ValueError, (some, some, 16)),
                        (ValueError, (some, one, 48)), (ValueError, (some, one, 8))]:
        with pytest.raises(error):
            PagePool(*args)
    with pytest.raises(ValueError):
        PagePool.full(0)


def test_tables_refuse():
    from moba_amd import PagePool, paged_release, paged_reserve
    pool, table, two = PagePool.full(5, 16, device="cpu"), torch.zeros((2, 3), dtype=I32), torch.zeros(2, dtype=I32)
    with pytest.raises(RuntimeError, match="AMD GPU"):
        paged_reserve(pool, table, two, two, 4)
    with pytest.raises(RuntimeError, match="AMD GPU"):
        paged_release(pool, table, two, two)
    many = torch.zeros(8193, dtype=I32)
    for error, args in [(TypeError, (table.long(), two, two)), (TypeError, (table, two.long(), two)), (TypeError, (table, two, two.float())),
                        (ValueError, (table[0], two, two)), (ValueError, (table, two[:1], two)), (ValueError, (table, two, two[:1])),
                        (ValueError, (table, table, two)), (ValueError, (table[:, :0], two, two)), (ValueError, (table[:1].expand(2, -1), two, two)),
                        (ValueError, (table.T.contiguous().T, two, two)), (ValueError, (table, torch.zeros(4, dtype=I32)[::2], two)),
                        (ValueError, (torch.zeros((8193, 1), dtype=I32), many, many))]:
        with pytest.raises(error):
            paged_reserve(pool, *args, 4)
        with pytest.raises(error):
            paged_release(pool, *args)
    for rows in (-1, 1 << 30):
        with pytest.raises(ValueError):
            paged_reserve(pool, table, two, two, rows)


def test_tables_entry_points_refuse():
    from moba_amd import _lib
    lib = _lib.load()
    some = 256   # (never read)

    def reserve(free=some, count=some, table=some, lengths=some, new=some, cu=some, owners=some, positions=some, slots=some, space=some, B=2, rows=4,
                page=16, pool=3, wide=1, stride=1):
        return lib.moba_paged_reserve(free, count, table, lengths, new, cu, owners, positions, slots, space, B, rows, page, pool, wide, stride, None)

    def release(free=some, count=some, table=some, lengths=some, new=some, B=2, page=16, pool=3, wide=1, stride=1):
        return lib.moba_paged_release(free, count, table, lengths, new, B, page, pool, wide, stride, None)

    common = [dict(free=None), dict(count=None), dict(table=None), dict(lengths=None), dict(new=None), dict(B=0), dict(pool=0), dict(wide=0),
              dict(stride=-1)]
    for wrong in common + [dict(cu=None), dict(owners=None), dict(positions=None), dict(slots=None), dict(space=None, rows=9000),
                           dict(space=some + 2), dict(slots=some + 4), dict(rows=-1)]:
        assert reserve(**wrong) == -1, wrong
    for wrong in common:
        assert release(**wrong) == -1, wrong
    for call in (reserve, release):
        assert call(page=48) == -2 and call(page=512) == -2
        for wrong in (dict(B=8193), dict(pool=1 << 31), dict(wide=1 << 31), dict(wide=1 << 30)):
            assert call(**wrong) == -4, wrong
    assert reserve(rows=1 << 30) == -4
    size = lib.moba_paged_reserve_workspace_bytes
    assert size(0, 9000) == size(7, 8192) == 0 and size(7, 8193) == 32


def attention_args(**changes):
    args = dict(query=torch.zeros((5, 4, 64), dtype=BF16), cache=make(), page_table=torch.zeros((2, 1), dtype=I32),
                lengths=torch.ones(2, dtype=I32), cu_new=torch.zeros(3, dtype=I32))
    args.update(changes)
    return args


q, t = torch.zeros((5, 4, 64), dtype=BF16), torch.zeros((2, 1), dtype=I32)
WRONG = [(TypeError, dict(query=q.float())), (TypeError, dict(cache=make(torch.float16))), (TypeError, dict(lengths=torch.ones(2))),
         (TypeError, dict(page_table=t.long())), (ValueError, dict(query=q[:, :3])), (ValueError, dict(query=q[:, :0])),
         (ValueError, dict(query=q[0])), (ValueError, dict(query=q[..., :32])), (ValueError, dict(page_table=t[0])),
         (ValueError, dict(page_table=t[:, :0])), (ValueError, dict(cu_new=t[:, 0])),
         (RuntimeError, dict(query=q.clone().requires_grad_()))]


def test_prefix_refuses():
    from moba_amd import paged_prefix_attention
    groups = dict(cu_groups=torch.zeros(3, dtype=I32), shared=torch.zeros(2, dtype=I32))
    call = lambda **c: paged_prefix_attention(**attention_args(**{**groups, **c}))  # noqa: E731
    with pytest.raises(RuntimeError, match="AMD GPU"):
        call()
    for error, changes in WRONG + [(TypeError, dict(shared=torch.zeros(2))), (TypeError, dict(cu_groups=torch.zeros(3).long())),
                                   (ValueError, dict(shared=torch.zeros(3, dtype=I32))), (ValueError, dict(cu_groups=t)),
                                   (ValueError, dict(cu_groups=torch.zeros(0, dtype=I32), shared=torch.zeros(0, dtype=I32)))]:
        with pytest.raises(error):
            call(**changes)


def test_sums_refuse():
    from moba_amd import paged_key_sums
    sums = make().key_sums()
    assert sums.shape == (3, 2, 64) and sums.dtype == torch.float32 and not sums.any()

    def call(**changes):
        args = {k: v for k, v in attention_args().items() if k != "query"}
        args.update(sums=sums, rows=5)
        args.update(changes)
        return paged_key_sums(**args)

    with pytest.raises(RuntimeError, match="AMD GPU"):
        call()
    for error, changes in [(TypeError, dict(sums=sums.double())), (TypeError, dict(lengths=torch.ones(2))), (ValueError, dict(sums=sums[:2])),
                           (ValueError, dict(sums=sums[..., :32])), (ValueError, dict(sums=sums.transpose(1, 2).contiguous().transpose(1, 2))),
                           (ValueError, dict(rows=-1)), (ValueError, dict(rows=1 << 30)), (ValueError, dict(page_table=t[0])),
                           (RuntimeError, dict(sums=sums.clone().requires_grad_()))]:
        with pytest.raises(error):
            call(**changes)


def test_select_refuses():
    from moba_amd import paged_select_blocks
    sums = torch.zeros((3, 2, 64))

    def call(**changes):
        args = {k: v for k, v in attention_args().items() if k != "cache"}
        args.update(sums=sums, page_size=16, block_size=32, topk=3)
        args.update(changes)
        return paged_select_blocks(**args)

    with pytest.raises(RuntimeError, match="AMD GPU"):
        call()
    wide = torch.zeros((2, 16385), dtype=I32)
    for error, changes in [w for w in WRONG if "cache" not in w[1]] + [
            (TypeError, dict(sums=sums.half())), (ValueError, dict(sums=sums[0])), (ValueError, dict(sums=sums[:0])),
            (ValueError, dict(sums=sums[:, :0])), (ValueError, dict(sums=torch.zeros(3, 2, 128))), (ValueError, dict(page_size=48)),
            (ValueError, dict(block_size=24)), (ValueError, dict(block_size=0)), (ValueError, dict(block_size=1 << 25)), (ValueError, dict(topk=0)),
            (ValueError, dict(topk=65)), (ValueError, dict(page_table=wide, block_size=16)), (RuntimeError, dict(sums=sums.clone().requires_grad_()))]:
        with pytest.raises(error):
            call(**changes)


def test_blocks_refuse():
    from moba_amd import paged_block_attention
    blocks = torch.zeros((5, 4, 3), dtype=I32)
    call = lambda **c: paged_block_attention(**attention_args(**{"blocks": blocks, "block_size": 32, **c}))  # noqa: E731
    with pytest.raises(RuntimeError, match="AMD GPU"):
        call()
    for error, changes in WRONG + [(TypeError, dict(blocks=blocks.long())), (ValueError, dict(blocks=blocks[0])), (ValueError, dict(blocks=blocks[:4])),
                                   (ValueError, dict(blocks=blocks[:, :2])), (ValueError, dict(blocks=blocks[..., :0])),
                                   (ValueError, dict(blocks=torch.zeros((5, 4, 65), dtype=I32))), (ValueError, dict(block_size=24)),
                                   (ValueError, dict(block_size=0)), (ValueError, dict(block_size=-16)), (ValueError, dict(block_size=1 << 25))]:
        with pytest.raises(error):
            call(**changes)


def test_attention_entry_points_refuse():
    from moba_amd import _lib
    lib = _lib.load()
    some = 256   # (never read)

    def common(first, second, more, q=some, out=some, kp=some, vp=some, ks=some, vs=some, table=some, lengths=some, cu=some, space=some, T=5,
               B=2, H=4, Hkv=2, D=64, page=16, pool=3, wide=1, strides=(256, 64, 1), cache8=1, dtype=0):
        s = None if strides is None else (ctypes.c_int64 * 3)(*strides)
        return first, second, more, q, out, kp, vp, ks, vs, table, lengths, cu, space, T, B, H, Hkv, D, page, pool, wide, s, cache8, dtype

    def prefix(groups=some, shared=some, G=1, **kw):
        g, f, G, q, out, kp, vp, ks, vs, table, lengths, cu, space, T, B, H, Hkv, D, page, pool, wide, s, c8, dtype = common(groups, shared, G, **kw)
        return lib.moba_paged_prefix_attention(q, out, kp, vp, ks, vs, table, lengths, cu, g, f, space, T, B, G, H, Hkv, D, page, pool, wide, s, c8,
                                               0.125, dtype, None)

    def blocks(blocks=some, block=32, topk=3, **kw):
        x, block, k, q, out, kp, vp, ks, vs, table, lengths, cu, space, T, B, H, Hkv, D, page, pool, wide, s, c8, dtype = common(blocks, block, topk, **kw)
        return lib.moba_paged_block_attention(q, out, kp, vp, ks, vs, x, table, lengths, cu, space, T, B, H, Hkv, D, page, pool, wide, block, k, s,
                                              c8, 0.125, dtype, None)

    for call in (prefix, blocks):
        for wrong in (dict(q=None), dict(out=None), dict(kp=None), dict(vp=None), dict(ks=None), dict(vs=None), dict(table=None),
                      dict(lengths=None), dict(cu=None), dict(space=None), dict(strides=None), dict(T=0), dict(B=0), dict(H=0), dict(Hkv=0),
                      dict(H=5), dict(pool=0), dict(wide=0), dict(q=some + 8), dict(kp=some + 8), dict(space=some + 4), dict(out=some + 4),
                      dict(strides=(256, 60, 1))):
            assert call(**wrong) == -1, wrong
        for wrong in (dict(D=96), dict(page=48), dict(page=512), dict(dtype=2)):
            assert call(**wrong) == -2, wrong
        for wrong in (dict(T=1 << 24), dict(T=1 << 23, H=1 << 10), dict(pool=1 << 31), dict(wide=1 << 31), dict(B=1 << 23, T=1 << 23)):
            assert call(**wrong) == -4, wrong
    assert prefix(groups=None) == prefix(shared=None) == prefix(G=0) == blocks(blocks=None) == blocks(topk=0) == -1
    assert blocks(block=24) == blocks(block=0) == blocks(block=-16) == -2
    assert blocks(topk=65) == blocks(block=1 << 25) == -4
    size = lib.moba_paged_prefix_attention_workspace_bytes
    assert size(5, 2, 0, 4, 2, 64, 1) == size(5, 2, 1, 5, 2, 64, 1) == size(5, 2, 1, 4, 2, 96, 1) == 0 < size(5, 2, 1, 4, 2, 64, 1) < 1 << 28
    size = lib.moba_paged_block_attention_workspace_bytes
    assert size(5, 2, 4, 2, 64, 16, 9, 24, 3, 1) == size(5, 2, 4, 2, 64, 16, 9, 32, 65, 1) == 0 < size(5, 2, 4, 2, 64, 16, 9, 32, 3, 1) < 1 << 28


def test_select_entry_points_refuse():
    from moba_amd import _lib
    lib = _lib.load()
    some = 256   # (never read)

    def sums(kp=some, ks=some, to=some, table=some, lengths=some, cu=some, T=5, B=2, Hkv=2, D=64, page=16, pool=3, wide=1, cache8=1, dtype=0):
        return lib.moba_paged_key_sums(kp, ks, to, table, lengths, cu, T, B, Hkv, D, page, pool, wide, 1, cache8, dtype, None)

    def select(q=some, sums=some, to=some, table=some, lengths=some, cu=some, space=some, T=5, B=2, H=4, Hkv=2, D=64, page=16, pool=3, wide=1,
               block=32, topk=3, strides=(256, 64, 1), dtype=0):
        s = None if strides is None else (ctypes.c_int64 * 3)(*strides)
        return lib.moba_paged_select_blocks(q, sums, to, table, lengths, cu, space, T, B, H, Hkv, D, page, pool, wide, block, topk, s, dtype, None)

    for wrong in (dict(kp=None), dict(ks=None), dict(to=None), dict(table=None), dict(lengths=None), dict(cu=None), dict(T=0), dict(B=0),
                  dict(Hkv=0), dict(pool=0), dict(wide=0), dict(kp=some + 8), dict(to=some + 2)):
        assert sums(**wrong) == -1, wrong
    for wrong in (dict(T=1 << 30), dict(pool=1 << 31), dict(wide=1 << 31), dict(B=1 << 24)):
        assert sums(**wrong) == -4, wrong
    for wrong in (dict(q=None), dict(sums=None), dict(to=None), dict(table=None), dict(lengths=None), dict(cu=None), dict(space=None),
                  dict(strides=None), dict(T=0), dict(B=0), dict(H=0), dict(Hkv=0), dict(H=5), dict(pool=0), dict(wide=0), dict(topk=0),
                  dict(q=some + 8), dict(sums=some + 4), dict(space=some + 4), dict(strides=(256, 60, 1))):
        assert select(**wrong) == -1, wrong
    for call in (sums, select):
        for wrong in (dict(D=96), dict(page=48), dict(page=512), dict(dtype=2)):
            assert call(**wrong) == -2, wrong
    assert select(block=24) == select(block=0) == -2
    for wrong in (dict(T=1 << 24), dict(T=1 << 23, H=1 << 10), dict(pool=1 << 31), dict(wide=1 << 31), dict(topk=65), dict(wide=1 << 16, block=16),
                  dict(B=1 << 24)):
        assert select(**wrong) == -4, wrong
    size = lib.moba_paged_select_blocks_workspace_bytes
    assert size(5, 2, 4, 2, 16, 1 << 16, 16) == size(5, 2, 4, 2, 16, 9, 24) == 0 and size(5, 2, 4, 2, 16, 9, 32) == 5 * 4 * 5 * 8
    assert size(1 << 20, 2, 64, 2, 16, 16384, 16) <= 1 << 29
