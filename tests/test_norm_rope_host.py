"""What qk_norm_rope and its entry points refuse, before anything is launched (no GPU)."""

import ctypes

import pytest
import torch

from rotary_reference import frequencies


def test_refusals():
    from moba_amd import qk_norm_rope
    q, k = torch.zeros((6, 4, 64), dtype=torch.bfloat16), torch.zeros((6, 2, 64), dtype=torch.bfloat16)
    at, f, w = torch.arange(6), frequencies(32), torch.ones(64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="AMD GPU"):
        qk_norm_rope(q, k, at, f, w, w)
    wrong = [
        (TypeError, (q.float(), k.float(), at, f)), (TypeError, (q, k.half(), at, f)),
        (TypeError, (q, k, at.float(), f)), (TypeError, (q, k, at, f.double())), (TypeError, (q, k, at, f, w.half())),
        (TypeError, (q, k, at, f, w, w.float())),
        (ValueError, (q[0], k, at, f)), (ValueError, (q, k[:5], at, f)), (ValueError, (q[..., :32], k, at, f)),
        (ValueError, (q[:, :0], k, at, f)), (ValueError, (q, k[:, :0], at, f)),
        (ValueError, (q[..., :60], k[..., :60], at, f[:28])), (ValueError, (torch.cat([q] * 3, -1), torch.cat([k] * 3, -1), at, f)),
        (ValueError, (q, k, at[:5], f)), (ValueError, (q, k, at[None], f)), (ValueError, (q, k, at, f[:30])),
        (ValueError, (q, k, at, frequencies(36))), (ValueError, (q, k, at, f[:0])), (ValueError, (q, k, at, f[None])),
        (ValueError, (q, k, at, f, w[:32])), (ValueError, (q, k, at, f, None, w[None])), (ValueError, (q, k, at, f, w, w, -1e-6)),
        (ValueError, (q, k, at, f, w, w, float("nan"))),
    ]
    for error, args in wrong:
        with pytest.raises(error):
            qk_norm_rope(*args)


def test_entry_points_refuse():
    from moba_amd import _lib
    lib = _lib.load()
    some = 256   # (never read)

    def forward(q=some, k=some, yq=some, yk=some, qw=some, kw=some, at=some, f=some, S=4, H=4, Hkv=2, D=64, rotary=64,
                strides=(256, 64, 128, 64), bits=64, w32=0, dtype=0):
        s = None if strides is None else (ctypes.c_int64 * 4)(*strides)
        return lib.moba_qk_norm_rope(q, k, yq, yk, qw, kw, at, f, S, H, Hkv, D, rotary, s, bits, 0, w32, 1e-6, dtype, None)

    def backward(dyq=some, dyk=some, qw=some, kw=some, dqw=some, dkw=some, space=some, S=4, w32=0):
        return lib.moba_qk_norm_rope_bwd(dyq, dyk, some, some, some, some, qw, kw, dqw, dkw, space, some, some, S, 4, 2, 64, 64,
                                         (ctypes.c_int64 * 4)(256, 64, 128, 64), 64, 0, w32, 1e-6, 0, None)

    for wrong in (dict(q=None), dict(k=None), dict(yq=None), dict(yk=None), dict(at=None), dict(f=None), dict(strides=None),
                  dict(q=some + 4), dict(yk=some + 2), dict(qw=some + 2), dict(kw=some + 2, w32=1), dict(S=0), dict(H=0),
                  dict(Hkv=-1), dict(D=60), dict(D=0), dict(rotary=72), dict(rotary=12), dict(rotary=-8), dict(bits=16),
                  dict(strides=(256, 64, 130, 64))):
        assert forward(**wrong) == -1, wrong
    assert forward(D=136, rotary=64) == -2 and forward(dtype=2) == -2
    assert forward(S=(1 << 25) + 1) == -4 and forward(H=(1 << 16) + 1) == -4
    for wrong in (dict(dyq=None), dict(dyk=some + 4), dict(space=None), dict(qw=None), dict(kw=None), dict(dqw=some + 1), dict(S=0),
                  dict(dkw=some + 2, w32=1), dict(space=some + 2)):
        assert backward(**wrong) == -1, wrong
    assert lib.moba_qk_norm_rope_bwd_workspace_bytes(0, 64) == 0
    assert lib.moba_qk_norm_rope_bwd_workspace_bytes(5, 64) == 2 * 2 * 64 * 4


def test_derivatives_that_there_are_none_of():
    """Refused, rather than lost: forward-mode tangents of any input, and the gradient of inv_freq."""
    import torch.autograd.forward_ad as fwd
    from moba_amd import qk_norm_rope
    q, k = torch.zeros((6, 4, 64), dtype=torch.bfloat16), torch.zeros((6, 2, 64), dtype=torch.bfloat16)
    at, f, w = torch.arange(6), frequencies(32), torch.ones(64, dtype=torch.bfloat16)
    args = [q, k, at, f, w, w]
    with fwd.dual_level():
        for i in (0, 1, 3, 4, 5):
            for where in (torch.enable_grad, torch.no_grad):
                with where(), pytest.raises(RuntimeError, match="forward-mode"):
                    qk_norm_rope(*[fwd.make_dual(x, torch.ones_like(x)) if i == j else x for j, x in enumerate(args)])
        with pytest.raises(RuntimeError, match="AMD GPU"):
            qk_norm_rope(*args)
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(lambda x: qk_norm_rope(x, k, at, f)[0], (q,), (torch.ones_like(q),))
    leaf = f.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="gradient of inv_freq"):
        qk_norm_rope(q, k, at, leaf)
    with torch.no_grad(), pytest.raises(RuntimeError, match="AMD GPU"):
        qk_norm_rope(q, k, at, leaf)
