"""References in 64 bits for the operator tests, and their error bounds.

``U`` is half a step of a 32-bit number: every 32-bit operation is off by at most
U relative to its result."""

import torch

U = 2.0 ** -24


def half_step(dtype, y):
    """Most that one rounding of ``y`` to ``dtype`` moves it (subnormals included)."""
    f = torch.finfo(dtype)
    return y.abs() * (f.eps / 2) + f.tiny * f.eps / 2


def turn(x, positions, inv_freq, layout="half", amplitude=1.0, inverse=False):
    """``(y, size)``: x (batch, tokens, heads, dim; float64) rotated, and |a| + |b| of
    the two elements that each result is made of."""
    half = inv_freq.numel()
    angle = positions.double()[..., None, None] * inv_freq
    c, s = amplitude * angle.cos(), amplitude * angle.sin() * (-1 if inverse else 1)
    y, size = x.clone(), x.abs()
    if layout == "half":
        ia, ib = slice(0, half), slice(half, 2 * half)
    else:
        ia, ib = slice(0, 2 * half, 2), slice(1, 2 * half, 2)
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    size[..., ia] = size[..., ib] = amplitude * (a.abs() + b.abs())
    return y, size


def norm(x, weight, eps):
    return x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * weight


# The sine of a reduced angle: |2t| <= 1 is rounded to 32 bits (2^-25 of a half
# turn: pi * U / 2 < 2 U), sincospi is off by 2 ulp (4 U at most), the amplitude's
# product by U; two products and a sum add 3 U.
TURN_ERROR = 10 * U
# The sum of squares adds up to 16 terms in a lane and 5 across lanes (21 U, half of
# it after the root), rsqrt is off by 2 ulp (4 U), mean and two products by 3 U.
NORM_ERROR = 18 * U


def check_turn(got, y, size, dtype, extra=0.0):
    tol = half_step(dtype, y) * 1.01 + (TURN_ERROR + extra) * size
    off = (got.double() - y).abs() - tol
    assert off.max().item() <= 0, f"{off.max().item():.3g} beyond the bound"
