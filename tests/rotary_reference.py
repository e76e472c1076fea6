"""The rotation by position in 64 bits, for the tests of the operators that apply it."""

import torch


def turned(x, positions, inv_freq, interleaved=False, back=False):
    """x [tokens, heads, head_dim] float64; the first 2 * len(inv_freq) elements of every head turned."""
    angle = positions.double()[:, None] * inv_freq.double()
    cos, sin = angle.cos()[:, None], (-angle if back else angle).sin()[:, None]
    n = inv_freq.numel()
    lo, hi = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    out = x.clone()
    out[..., lo] = x[..., lo] * cos - x[..., hi] * sin
    out[..., hi] = x[..., hi] * cos + x[..., lo] * sin
    return out


def pair_size(x, n, interleaved=False):
    """Of every element, the length of the pair it is turned with (its own magnitude where it is not turned)."""
    lo, hi = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    out = x.abs()
    out[..., lo] = out[..., hi] = torch.hypot(x[..., lo], x[..., hi])
    return out


def frequencies(n, device="cpu", base=500000.0):
    return (base ** (-torch.arange(n, dtype=torch.float64) / max(n, 1))).float().to(device)
