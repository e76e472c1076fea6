"""What the paged cache's operators and entry points refuse, before anything is launched (no GPU)."""

import ctypes

import pytest
import torch

from rotary_reference import frequencies

E4M3, BF16 = torch.float8_e4m3fn, torch.bfloat16


def make(dtype=E4M3, pages=3, heads=2, page=16, d=64):
    from moba_amd import PagedKVCache
    return PagedKVCache.empty(pages, heads, head_dim=d, page_size=page, dtype=dtype, device="cpu")


def test_the_cache_refuses():
    from moba_amd import PagedKVCache
    k = torch.zeros((3, 2, 16, 64), dtype=E4M3)
    s, k16 = torch.ones((3, 2)), torch.zeros((3, 2, 16, 64), dtype=BF16)
    assert make().quantized and not make(BF16).quantized and make(torch.float16).k_pages.shape == (3, 2, 16, 64)
    wrong = [
        (TypeError, (k.float(), k.float())), (TypeError, (k, k16, s, s)), (TypeError, (k, k, s.double(), s)),
        (TypeError, (k.to(torch.float8_e5m2), k.to(torch.float8_e5m2), s, s)),
        (ValueError, (k, k)), (ValueError, (k, k, s)), (ValueError, (k16, k16, s, s)), (ValueError, (k, k, s[:2], s)),
        (ValueError, (k[0], k[0], s, s)), (ValueError, (k, k[:2], s, s)), (ValueError, (k[:, :, :8], k[:, :, :8], s, s)),
        (ValueError, (k[:0], k[:0], s[:0], s[:0])), (ValueError, (k[:, :0], k[:, :0], s[:, :0], s[:, :0])),
        (ValueError, (k[..., :32], k[..., :32], s, s)), (ValueError, (k.transpose(0, 1), k.transpose(0, 1), s.T, s.T)),
        (ValueError, (k, k, s, s.T.contiguous().T)),
        (ValueError, (torch.zeros(3 * 2 * 16 * 64 + 1, dtype=BF16)[1:].view(3, 2, 16, 64), k16)),
    ]
    for error, args in wrong:
        with pytest.raises(error):
            PagedKVCache(*args)
    with pytest.raises(ValueError):
        make(heads=257)


def append_args(**changes):
    args = dict(cache=make(), key=torch.zeros((5, 2, 64), dtype=BF16), value=torch.zeros((5, 2, 64), dtype=BF16),
                page_table=torch.zeros((2, 1), dtype=torch.int32), lengths=torch.ones(2, dtype=torch.int32),
                cu_new=torch.zeros(3, dtype=torch.int32), inv_freq=frequencies(32), query=torch.zeros((5, 4, 64), dtype=BF16))
    args.update(changes)
    return args


def test_append_refuses():
    from moba_amd import paged_append
    with pytest.raises(RuntimeError, match="AMD GPU"):
        paged_append(**append_args())
    x, t = torch.zeros((5, 2, 64)), torch.zeros((2, 1), dtype=torch.int32)
    wrong = [
        (TypeError, dict(key=x)), (TypeError, dict(value=x)), (TypeError, dict(query=x)), (TypeError, dict(cache=make(torch.float16))),
        (TypeError, dict(page_table=t.long())), (TypeError, dict(lengths=torch.ones(2))), (TypeError, dict(cu_new=torch.zeros(3).long())),
        (TypeError, dict(inv_freq=frequencies(32).double())),
        (ValueError, dict(key=x.to(BF16)[:4])), (ValueError, dict(value=x.half())), (ValueError, dict(query=x.half())),
        (ValueError, dict(query=x.to(BF16)[:4])), (ValueError, dict(query=x.to(BF16)[:, :0])), (ValueError, dict(key=x.to(BF16)[0])),
        (ValueError, dict(key=x.to(BF16)[..., :32], value=x.to(BF16)[..., :32])), (ValueError, dict(query=x.to(BF16)[..., :32])),
        (ValueError, dict(cache=make(heads=3))), (ValueError, dict(cache=make(d=128))),
        (ValueError, dict(page_table=t[0])), (ValueError, dict(page_table=t[:1])), (ValueError, dict(page_table=t[:, :0])),
        (ValueError, dict(lengths=t)), (ValueError, dict(lengths=t[:1, 0])), (ValueError, dict(cu_new=torch.zeros(2, dtype=torch.int32))),
        (ValueError, dict(inv_freq=frequencies(36))), (ValueError, dict(inv_freq=frequencies(30))),
    ]
    for error, changes in wrong:
        with pytest.raises(error):
            paged_append(**append_args(**changes))


def test_append_entry_point_refuses():
    from moba_amd import _lib
    lib = _lib.load()
    some = 256   # (never read)

    def call(k=some, v=some, q=some, yq=some, kp=some, vp=some, ks=some, vs=some, table=some, lengths=some, cu=some, f=some, T=5,
             B=2, H=4, Hkv=2, D=64, rotary=64, page=16, pool=3, wide=1, strides=(256, 64, 128, 64, 128, 64, 1), cache8=1, dtype=0):
        s = None if strides is None else (ctypes.c_int64 * 7)(*strides)
        return lib.moba_paged_append(k, v, q, yq, kp, vp, ks, vs, table, lengths, cu, f, T, B, H, Hkv, D, rotary, page, pool, wide,
                                     s, cache8, 0, dtype, None)

    for wrong in (dict(k=None), dict(v=None), dict(yq=None), dict(kp=None), dict(vp=None), dict(ks=None), dict(vs=None), dict(table=None),
                  dict(lengths=None), dict(cu=None), dict(f=None), dict(strides=None), dict(T=0), dict(B=0), dict(H=0), dict(Hkv=0),
                  dict(rotary=12), dict(rotary=72), dict(rotary=-8), dict(pool=0), dict(wide=0), dict(k=some + 4), dict(q=some + 2),
                  dict(kp=some + 4), dict(strides=(256, 64, 128, 62, 128, 64, 1))):
        assert call(**wrong) == -1, wrong
    for wrong in (dict(D=96), dict(page=48), dict(page=8), dict(page=512), dict(dtype=2)):
        assert call(**wrong) == -2, wrong
    for wrong in (dict(T=1 << 30), dict(pool=1 << 31), dict(wide=1 << 31), dict(Hkv=257), dict(H=(1 << 16) + 1), dict(B=1 << 22),
                  dict(T=(1 << 30) - 1)):
        assert call(**wrong) == -4, wrong


def test_attention_refuses():
    from moba_amd import paged_attention

    def call(**changes):
        args = {k: v for k, v in append_args().items() if k in ("query", "cache", "page_table", "lengths", "cu_new")}
        args.update(changes)
        return paged_attention(**args)

    with pytest.raises(RuntimeError, match="AMD GPU"):
        call()
    q, t = torch.zeros((5, 4, 64), dtype=BF16), torch.zeros((2, 1), dtype=torch.int32)
    for error, changes in [
            (TypeError, dict(query=q.float())), (TypeError, dict(cache=make(torch.float16))), (TypeError, dict(lengths=torch.ones(2))),
            (TypeError, dict(page_table=t.long())), (ValueError, dict(query=q[:, :3])), (ValueError, dict(query=q[:, :0])),
            (ValueError, dict(query=q[0])), (ValueError, dict(query=q[..., :32])), (ValueError, dict(page_table=t[0])),
            (ValueError, dict(page_table=t[:, :0])), (ValueError, dict(cu_new=t[:, 0])), (ValueError, dict(max_new=-1))]:
        with pytest.raises(error):
            call(**changes)


def test_attention_entry_point_refuses():
    from moba_amd import _lib
    lib = _lib.load()
    some = 256   # (never read)

    def call(q=some, out=some, kp=some, vp=some, ks=some, vs=some, table=some, lengths=some, cu=some, space=some, T=5, B=2, H=4,
             Hkv=2, D=64, page=16, pool=3, wide=1, hint=-1, strides=(256, 64, 1), cache8=1, dtype=0):
        s = None if strides is None else (ctypes.c_int64 * 3)(*strides)
        return lib.moba_paged_attention(q, out, kp, vp, ks, vs, table, lengths, cu, space, T, B, H, Hkv, D, page, pool, wide, hint,
                                        s, cache8, 0.125, dtype, None)

    for wrong in (dict(q=None), dict(out=None), dict(kp=None), dict(vp=None), dict(ks=None), dict(vs=None), dict(table=None),
                  dict(lengths=None), dict(cu=None), dict(space=None), dict(strides=None), dict(T=0), dict(B=0), dict(H=0), dict(Hkv=0),
                  dict(H=5), dict(pool=0), dict(wide=0), dict(q=some + 8), dict(kp=some + 8), dict(space=some + 4), dict(out=some + 4),
                  dict(strides=(256, 60, 1))):
        assert call(**wrong) == -1, wrong
    for wrong in (dict(D=96), dict(page=48), dict(page=512), dict(dtype=2)):
        assert call(**wrong) == -2, wrong
    for wrong in (dict(T=1 << 30), dict(T=1 << 29), dict(T=1 << 24), dict(pool=1 << 31), dict(wide=1 << 31), dict(B=1 << 25, T=1 << 25)):
        assert call(**wrong) == -4, wrong
    sizes = lib.moba_paged_attention_workspace_bytes
    assert sizes(0, 2, 4, 2, 64, 1, -1) == 0 and sizes(5, 2, 5, 2, 64, 1, -1) == 0 and sizes(5, 2, 4, 2, 96, 1, -1) == 0
    # rows (a head's output and its log-sum-exp) for every unit that several runs can make, and these are no more than a few
    # rounds of workgroups; a hint that there are few new tokens leaves out those of the other kernel
    for args in ((1, 1, 32, 8, 128, 1), (64, 64, 32, 8, 128, 0), (1 << 20, 3, 8, 8, 64, 1), (1 << 20, 1 << 20, 8, 1, 64, 1)):
        need, less = sizes(*args, -1), sizes(*args, 1)
        runs = (args[1] * 12 + 15) // 16 * 16
        assert (need - runs) % (32 * (args[4] + 1) * 4) == 0 and 0 < less <= need < 2 << 30, args


def test_rows_that_want_a_gradient():
    """There are none: refused, but for calls that record no graph (which go on to the next check)."""
    from moba_amd import paged_append, paged_attention
    rest = {k: v for k, v in append_args().items() if k in ("query", "cache", "page_table", "lengths", "cu_new")}
    for name in ("key", "value", "query"):
        args = append_args(**{name: append_args()[name].requires_grad_()})
        with pytest.raises(RuntimeError, match="no gradients"):
            paged_append(**args)
        with torch.no_grad(), pytest.raises(RuntimeError, match="AMD GPU"):
            paged_append(**args)
    rest["query"] = rest["query"].requires_grad_()
    with pytest.raises(RuntimeError, match="no gradients"):
        paged_attention(**rest)
    with torch.inference_mode(), pytest.raises(RuntimeError, match="AMD GPU"):
        paged_attention(**rest)


def test_caches_compare_by_identity():
    a, b = make(), make()
    assert a == a and a != b and len({a, b}) == 2


def attention_code(T, B, H, Hkv, D, cache8=1, hint=-1):
    """What the entry point answers for sizes that it takes: here, where there is no GPU, that nothing could be launched."""
    from moba_amd import _lib
    some = 256   # (never read)
    return _lib.load().moba_paged_attention(*[some] * 10, T, B, H, Hkv, D, 16, 3, 1, hint, (ctypes.c_int64 * 3)(H * D, D, 1), cache8,
                                            0.125, 0, None)


@pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are none")
def test_long_pieces_on_8_bit_pages():
    """Up to 64 rows of a sequence are few with 8-bit pages, two groups of 32: a long piece asks for no more of them than that, neither
    workgroups nor workspace."""
    from moba_amd import _lib
    sizes = _lib.load().moba_paged_attention_workspace_bytes
    for T, B in ((2048, 1), (131072, 1), (131072, 20), (1 << 22, 1)):
        # units of 256 compute units, two workgroups to each (many rows: one), 8 key/value heads: few rows and many
        few = max(64, 33 + 2 * B)
        many = 17 + min(128, B + T * 4 // 256)
        assert sizes(T, B, 32, 8, 128, 1, -1) <= (few * 32 + many * 256) * 8 * 129 * 4 + 16 * B, (T, B)
    for args in ((1 << 22, 1, 128, 8, 128), (1 << 22, 1, 128, 8, 64), (1 << 23, 4, 128, 16, 128)):
        assert attention_code(*args) == attention_code(*args, cache8=0) == -3, args


@pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are none")
def test_launches_of_too_many_threads():
    """Refused as a limit before anything is launched, by the threads of each kernel's own workgroups: 512 of the many-row one
    for 128-element heads on 8-bit pages."""
    T = 1 << 21
    assert attention_code(T, T // 65, 256, 256, 128) == -4          # 40448 units of many rows a head: 5.3e9 threads
    assert attention_code(T, T // 65, 256, 256, 64) == -3           # 256 threads each, 48640 units: 3.2e9
    assert attention_code(1 << 22, 1 << 12, 256, 256, 128, cache8=0, hint=0) == -4   # few rows, says the hint: 8.9e9
    assert attention_code(1 << 22, 1 << 12, 256, 256, 128, cache8=0) == -3           # 2.4e9


def test_derivatives_that_there_are_none_of():
    """Refused, rather than lost: gradients of the cache and of inv_freq, and forward-mode tangents of anything."""
    import torch.autograd.forward_ad as fwd
    from moba_amd import PagedKVCache, paged_append, paged_attention
    attend = lambda cache, **changes: paged_attention(**{  # noqa: E731
        n: x for n, x in append_args(cache=cache, **changes).items() if n in ("query", "cache", "page_table", "lengths", "cu_new")})

    def caches(change):
        """The 16-bit and the 8-bit cache with one tensor changed."""
        for dtype in (BF16, E4M3):
            fields = {n: getattr(make(dtype), n) for n in ("k_pages", "v_pages", "k_scales", "v_scales")}
            for name, x in fields.items():
                if x is not None and x.dtype != E4M3:
                    yield PagedKVCache(**{**fields, name: change(x)})

    for cache in caches(lambda x: x.requires_grad_()):
        for call in (lambda: paged_append(**append_args(cache=cache)), lambda: attend(cache)):
            with pytest.raises(RuntimeError, match="no gradients"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="AMD GPU"):
                call()
    with pytest.raises(RuntimeError, match="no gradients"):
        paged_append(**append_args(inv_freq=frequencies(32).requires_grad_()))
    with fwd.dual_level(), torch.no_grad():
        dual = lambda x: fwd.make_dual(x, torch.ones_like(x))  # noqa: E731
        for cache in caches(dual):
            for call in (lambda: paged_append(**append_args(cache=cache)), lambda: attend(cache)):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call()
        for name in ("key", "value", "query", "inv_freq"):
            with pytest.raises(RuntimeError, match="forward-mode"):
                paged_append(**append_args(**{name: dual(append_args()[name])}))
        with pytest.raises(RuntimeError, match="forward-mode"):
            attend(make(), query=dual(append_args()["query"]))
