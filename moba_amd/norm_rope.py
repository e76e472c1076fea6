"""Norm and rotation of query and key heads on MI355X: what precedes ``moba_attn_varlen`` in a decoder layer, in one pass over
q and k, forward and backward.  (The reference leaves both to the torch ops of the transformers model that calls its adapter,
moba/wrapper.py:29-40.)"""

from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib
from . import moba_efficient as E

MAX_TOKENS = 1 << 25   # that one call takes


def _strides_of(t: torch.Tensor):
    """(token stride, head stride) of a [tokens, heads, head_dim] tensor that the kernels can read where it lies, or None."""
    ts, hs = E._row_strides(t)
    fits = (t.stride(2) == 1 or t.shape[2] == 1) and ts % 4 == 0 and hs % 4 == 0 and t.data_ptr() % 8 == 0
    return (ts, hs) if fits else None


def _readable(t: torch.Tensor) -> torch.Tensor:
    return t if _strides_of(t) is not None else E._aligned(t)


def _has_tangent(*tensors) -> bool:
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _check(q, k, positions, inv_freq, q_weight, k_weight, eps):
    if q.dtype not in (torch.bfloat16, torch.float16) or k.dtype != q.dtype:
        raise TypeError("qk_norm_rope supports bfloat16 and float16 q and k (both of the same dtype)")
    if q.dim() != 3 or k.dim() != 3 or q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2] or not q.shape[1] or not k.shape[1]:
        raise ValueError("q must be [tokens, heads, head_dim] and k [tokens, kv_heads, head_dim]")
    tokens, _, d = q.shape
    if d % 8 or not 0 < d <= E.HEAD_DIM:
        raise ValueError(f"head_dim must be a multiple of 8 and at most {E.HEAD_DIM}")
    if tokens > MAX_TOKENS or max(q.shape[1], k.shape[1]) > 65536:
        raise ValueError(f"at most {MAX_TOKENS} tokens and 65536 heads")
    if positions.dtype not in (torch.int32, torch.int64):
        raise TypeError("positions must be int32 or int64")
    if positions.shape != (tokens,):
        raise ValueError("positions must be [tokens]")
    _check_inv_freq(inv_freq, d)
    weights = [w for w in (q_weight, k_weight) if w is not None]
    for w in weights:
        if w.dtype not in (q.dtype, torch.float32) or w.dtype != weights[0].dtype:
            raise TypeError("the weights must be of q's dtype or float32, both alike")
        if w.shape != (d,):
            raise ValueError("the weights must be [head_dim]")
    if any(t.device != q.device for t in (k, positions, inv_freq, *weights)):
        raise ValueError("all tensors must be on one device")
    if not eps >= 0:
        raise ValueError("eps must not be negative")
    if _has_tangent(q, k, inv_freq, *weights):
        raise RuntimeError("qk_norm_rope has no forward-mode derivatives: tensors with a tangent are refused")
    if inv_freq.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("qk_norm_rope has no gradient of inv_freq: call it under torch.no_grad(), or with inv_freq.detach()")
    if not q.is_cuda:
        raise RuntimeError("qk_norm_rope needs tensors on an AMD GPU (there is no CPU path)")


def _check_inv_freq(inv_freq, d):
    if inv_freq.dtype != torch.float32:
        raise TypeError("inv_freq must be float32")
    if inv_freq.dim() != 1 or inv_freq.numel() % 4 or not 0 < 2 * inv_freq.numel() <= d:
        raise ValueError("inv_freq must hold one number for each rotated pair: a multiple of 4, at most head_dim / 2")


def _args(q, k, positions, inv_freq, eps, interleaved, w32):
    """The arguments both entry points end with."""
    s, h, d = q.shape
    strides = (ctypes.c_int64 * 4)(*_strides_of(q), *_strides_of(k))
    return (E._ptr(positions), E._ptr(inv_freq), s, h, k.shape[1], d, 2 * inv_freq.numel(), strides,
            64 if positions.dtype == torch.int64 else 32, int(interleaved), int(w32), eps, E._dtype_code(q), E._stream(q.device))


def _weights_for_kernel(*weights):
    ready = [w if w is None or (w.is_contiguous() and w.data_ptr() % 8 == 0) else E._aligned(w) for w in weights]
    return ready, any(w is not None and w.dtype == torch.float32 for w in weights)


def _forward(q, k, positions, inv_freq, q_weight, k_weight, eps, interleaved):
    """(yq, yk) of tensors the kernels can read."""
    yq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    yk = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    if q.shape[0]:
        (qw, kw), w32 = _weights_for_kernel(q_weight, k_weight)
        with torch.cuda.device(q.device):
            _lib.check(_lib.load().moba_qk_norm_rope(
                E._ptr(q), E._ptr(k), E._ptr(yq), E._ptr(yk), E._ptr(qw), E._ptr(kw),
                *_args(q, k, positions, inv_freq, eps, interleaved, w32)), "moba_qk_norm_rope")
    return yq, yk


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, q_weight, k_weight, eps, interleaved):
        ctx.save_for_backward(q, k, positions, inv_freq, q_weight, k_weight)
        ctx.eps, ctx.interleaved = eps, interleaved
        return _forward(_readable(q), _readable(k), positions, inv_freq, q_weight, k_weight, eps, interleaved)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dyq, dyk):
        q, k, positions, inv_freq, q_weight, k_weight = ctx.saved_tensors
        if _has_tangent(dyq, dyk):
            raise RuntimeError("qk_norm_rope has no forward-mode derivatives: tensors with a tangent are refused")
        q, k, positions, inv_freq = _readable(q), _readable(k), positions.contiguous(), inv_freq.contiguous()
        dyq, dyk = E._aligned(dyq), E._aligned(dyk)
        dq, dk = torch.empty(q.shape, dtype=q.dtype, device=q.device), torch.empty(k.shape, dtype=k.dtype, device=k.device)
        need = [w is not None and ctx.needs_input_grad[4 + i] for i, w in enumerate((q_weight, k_weight))]
        new = torch.empty if q.shape[0] else torch.zeros
        dw = [new(w.shape, dtype=w.dtype, device=w.device) if n else None for n, w in zip(need, (q_weight, k_weight))]
        if q.shape[0]:
            lib = _lib.load()
            (qw, kw), w32 = _weights_for_kernel(q_weight, k_weight)
            with torch.cuda.device(q.device):
                space = None
                if any(need):
                    space = torch.empty(lib.moba_qk_norm_rope_bwd_workspace_bytes(q.shape[0], q.shape[2]), dtype=torch.uint8,
                                        device=q.device)
                _lib.check(lib.moba_qk_norm_rope_bwd(
                    E._ptr(dyq), E._ptr(dyk), E._ptr(q), E._ptr(k), E._ptr(dq), E._ptr(dk), E._ptr(qw), E._ptr(kw),
                    E._ptr(dw[0]), E._ptr(dw[1]), E._ptr(space),
                    *_args(q, k, positions, inv_freq, ctx.eps, ctx.interleaved, w32)), "moba_qk_norm_rope_bwd")
        return dq, dk, None, None, dw[0], dw[1], None, None


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor,
                 q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                 interleaved: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """Root-mean-square norm of every query and key head and rotation by position, in one pass.

    Args:
        q, k: [tokens, heads, head_dim] and [tokens, kv_heads, head_dim] bf16 or fp16, as ``moba_attn_varlen`` takes them;
            views of any token and head strides that are multiples of 4 elements are read in place.  head_dim a multiple of
            8, at most 128.
        positions: [tokens] int32 or int64
        inv_freq: [n] float32, the angle a pair turns by from one position to the next; the first 2n elements of a head are
            rotated: pairs (i, i + n), or (2i, 2i + 1) with ``interleaved``
        q_weight, k_weight: [head_dim], of q's dtype or float32: ``x * weight / sqrt(mean(x^2) + eps)`` over the elements of a
            head before the rotation; None: that side is rotated only
    Returns:
        the new q and k, packed.  Differentiable once in q, k and the weights, backward (tensors with forward-mode tangents
        are refused, and an inv_freq that requires a gradient outside ``torch.no_grad()``); the weights' gradients are summed in
        a fixed order (the same bits on every run).  A call that is being captured into a graph is refused while an eager graph of the
        same leaves is alive (its backward pass could not be captured).
    """
    y = _lib.host().norm_rope(q, k, positions, inv_freq, q_weight, k_weight, eps, interleaved)
    if y is not NotImplemented:
        return y
    # tensors that have to be copied first, none at all, or wrong ones
    _check(q, k, positions, inv_freq, q_weight, k_weight, eps)
    positions, inv_freq = positions.contiguous(), inv_freq.contiguous()
    tensors = (q, k, q_weight, k_weight)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        _lib.host().check_leaves(*tensors)
        return _QkNormRope.apply(q, k, positions, inv_freq, q_weight, k_weight, eps, interleaved)
    return _forward(_readable(q), _readable(k), positions, inv_freq, q_weight, k_weight, eps, interleaved)
