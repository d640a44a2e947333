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


def attend(q, k_cache, v_cache, page_table, lengths, prefix_pages, prefix, counts, scale):
    """``(out, lse, tolerance, lse tolerance)`` of the sequences' new tokens, row after row:
    q (tokens, heads, dim), sequence b with counts[b] of them; in 64 bits."""
    kv, dim = k_cache.shape[2:]
    page, group = k_cache.shape[1], q.shape[1] // kv
    dtype = q.dtype
    results, at = [], 0
    for b, n in enumerate(counts):
        if n == 0:
            continue
        own = int(lengths[b])
        mine = page_table[b, :-(-own // page)].long()
        k, v = (torch.cat([c[prefix_pages.long()].reshape(-1, kv, dim)[:prefix],
                           c[mine].reshape(-1, kv, dim)[:own]]).double() for c in (k_cache, v_cache))
        x = q[at:at + n].double().view(n, kv, group, dim)
        at += n
        keys = prefix + own
        seen = torch.arange(keys, device=q.device) < (keys - n + 1 + torch.arange(n, device=q.device))[:, None]
        s = scale * torch.einsum("nkgd,jkd->nkgj", x, k)
        s = s.masked_fill(~seen[:, None, None], float("-inf"))
        size = abs(scale) * torch.einsum("nkgd,jkd->nkgj", x.abs(), k.abs())   # sum of a score's absolute products
        top = s.amax(-1, keepdim=True) if keys else s.new_full(s.shape[:-1] + (1,), float("-inf"))
        p = (s - top.clamp_min(-1e300)).exp()
        total = p.sum(-1, keepdim=True)
        out = torch.einsum("nkgj,jkd->nkgd", p, v) / total
        lse = (top + total.log())[..., 0]
        # a score: 2 dim U of its absolute products (sums of matrix instructions count double),
        # three roundings of its size; the exponential 2^-22; then the weight's rounding to the
        # values' type, of its own size or (subnormal float16) of its smallest step
        rel = (2 * dim + 8) * U * size + 2 ** -21
        weight = p * (rel + torch.finfo(dtype).eps / 2) + torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2 * seen[:, None, None]
        sums = (2 * keys + 64) * U                                       # the sums over keys, and the joins
        tol = torch.einsum("nkgj,jkd->nkgd", weight + p * sums, v.abs()) / total
        tol = tol + out.abs() * ((p * (rel + sums)).sum(-1, keepdim=True) / total)
        empty = total == 0
        out, tol = out.masked_fill(empty, 0.0), tol.masked_fill(empty, 0.0)
        lse_tol = ((p * (rel + sums)).sum(-1, keepdim=True) / total).masked_fill(empty, 0.0)[..., 0]
        lse_tol = lse_tol + 4 * U * lse.abs().nan_to_num(0, 0, 0) + 4 * U
        lse = lse.masked_fill(empty[..., 0], float("-inf"))
        results.append((out.reshape(n, -1, dim), lse.reshape(n, -1),
                        (tol + 1.01 * half_step(dtype, out)).reshape(n, -1, dim), lse_tol.reshape(n, -1)))
    return [torch.cat(x) for x in zip(*results)]
