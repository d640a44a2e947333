"""The decode-path operators on the GPU against their definitions in 64 bits."""

import ctypes
import math
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from tila_b200 import native, ops
from ops_support import NORM_ERROR, TURN_ERROR, U, attend, check_turn, half_step, norm, turn

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def normal(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def freqs(rotary):
    return ops.rotary_frequencies(rotary)[0]


def as_rows(x):
    return x.double() if x.dim() == 4 else x.double()[None]


def as_positions(positions, tokens):
    return positions if positions.dim() == 2 else positions[None]


# ---------------------------------------------------------------------------
# rotate
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("batch,tokens,heads,dim,rotary", [
    (1, 1, 1, 2, 2), (1, 1, 32, 128, 128), (2, 37, 5, 64, 64), (3, 9, 3, 80, 40), (1, 130, 2, 96, 24),
    (2, 5, 7, 128, 32), (1, 17, 4, 33, 10), (1, 3, 1, 512, 512), (1, 4, 2, 511, 6), (2, 3, 2, 40, 0), (1, 600, 1, 20, 20),
    (2, 65, 5, 80, 20), (1, 40, 3, 504, 250), (1, 33, 2, 8, 2), (1, 700, 3, 24, 22),
])
def test_rotate(layout, dtype, batch, tokens, heads, dim, rotary):
    g = gen(dim + tokens)
    x = normal(g, batch, tokens, heads, dim, dtype=dtype)
    positions = torch.randint(-5, 1 << 21, (batch, tokens), generator=g, device="cuda")
    inv = freqs(rotary)
    for call, inverse in ((ops.rotate, False), (ops.rotate_backward, True)):
        y, size = turn(x.double(), positions, inv, layout, 1.25, inverse)
        got = call(x, positions, inv, layout=layout, amplitude=1.25)
        assert got.dtype is dtype and got.shape == x.shape
        check_turn(got, y, size, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rotate_strided_in_place_and_int32_positions(dtype):
    """Heads before tokens, a part of a wider projection, an odd offset (narrow
    accesses), positions shared by the batch: all into the source's own place."""
    g = gen(3)
    inv = freqs(64)
    base = normal(g, 2, 6, 11, 64, dtype=dtype)                      # (batch, heads, tokens, dim)
    wide = normal(g, 2, 11, 3 * 6 * 64, dtype=dtype)
    flat = normal(g, 2 * 11 * 6 * 64 + 1, dtype=dtype)
    positions = torch.arange(11, device="cuda", dtype=torch.int32) * 1000
    for x in (base.transpose(1, 2), wide.view(2, 11, 18, 64)[:, :, 6:12], flat[1:].view(2, 11, 6, 64)):
        y, size = turn(x.double(), positions.expand(2, 11), inv)
        kept = wide.clone()
        got = ops.rotate(x, positions, inv, out=x)
        assert got is x
        check_turn(x, y, size, dtype)
        kept.view(2, 11, 18, 64)[:, :, 6:12] = wide.view(2, 11, 18, 64)[:, :, 6:12]
        assert torch.equal(kept, wide)                               # nothing beside the rows was written


def test_rotate_far_positions_keep_their_angle():
    x = torch.ones(4, 1, 128, device="cuda")
    positions = torch.tensor([0, 1, (1 << 31) + 5, 1 << 40], device="cuda")
    # at 2^40 positions the product of position and frequency is off by 2^-53 of itself
    y, size = turn(x.double()[None], positions[None], freqs(128))
    got = ops.rotate(x, positions, freqs(128)).double()[None]
    far = (positions.double() * 2 ** -52).view(1, 4, 1, 1)
    assert ((got - y).abs() <= U * y.abs() + TURN_ERROR * size + far * size).all()


def test_rotate_nothing():
    for shape in ((0, 4, 64), (3, 0, 64), (0, 5, 4, 64)):
        x = torch.empty(shape, device="cuda")
        assert ops.rotate(x, torch.zeros(shape[:-2], dtype=torch.int64, device="cuda"), freqs(64)).shape == x.shape


# ---------------------------------------------------------------------------
# norm and rotate
# ---------------------------------------------------------------------------

NORM_CASES = [  # tokens, heads, kv_heads, dim, rotary
    (1, 1, 1, 128, 128), (7, 32, 8, 128, 128), (700, 5, 2, 64, 64), (65, 3, 3, 80, 40), (33, 4, 1, 96, 24), (5, 2, 1, 33, 10),
    (9, 2, 2, 512, 64), (3, 1, 2, 20, 0), (301, 5, 2, 80, 20), (17, 3, 1, 504, 250), (40, 2, 1, 24, 22),
]


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype,wdtype", [(F32, F32), (F16, F16), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("tokens,heads,kv,dim,rotary", NORM_CASES)
def test_norm_rotate_and_its_gradient(layout, dtype, wdtype, tokens, heads, kv, dim, rotary):
    g = gen(tokens + dim)
    qkv = normal(g, tokens, heads + 2 * kv, dim, dtype=dtype)
    q, k = qkv[:, :heads], qkv[:, heads:heads + kv]
    qw, kw = (1 + 0.3 * normal(g, dim)).to(wdtype), (1 + 0.3 * normal(g, dim)).to(wdtype)
    positions = torch.randint(0, 1 << 17, (tokens,), generator=g, device="cuda")
    inv, eps, amp = freqs(rotary), 1e-5, 0.75
    got = ops.norm_rotate(q, k, qw, kw, positions, inv, layout=layout, amplitude=amp, eps=eps)
    for out, x, w in zip(got, (q, k), (qw, kw)):
        y, size = turn(norm(as_rows(x), w.double(), eps), positions[None], inv, layout, amp)
        check_turn(out[None], y, size, dtype, extra=NORM_ERROR)

    grads = normal(g, tokens, heads, dim, dtype=dtype), normal(g, tokens, kv, dim, dtype=dtype)
    dq, dk, dqw, dkw = ops.norm_rotate_backward(*grads, q, k, qw, kw, positions, inv, layout=layout, amplitude=amp,
                                                eps=eps)
    again = ops.norm_rotate_backward(*grads, q, k, qw, kw, positions, inv, layout=layout, amplitude=amp, eps=eps)
    for a, b in zip((dq, dk, dqw, dkw), again):
        assert torch.equal(a, b)                                     # sums in a fixed order
    for dx, dw, x, w, gy in ((dq, dqw, q, qw, grads[0]), (dk, dkw, k, kw, grads[1])):
        x64, w64 = as_rows(x).requires_grad_(), w.double().requires_grad_()
        y, _ = turn(norm(x64, w64, eps), positions[None], inv, layout, amp)
        ex, ew = torch.autograd.grad(y, (x64, w64), gy.double()[None])
        # dx = r (w g - xh m): g is off by TURN_ERROR of its two elements, r and xh by
        # NORM_ERROR, the mean m by 21 U of the mean of absolute products and its factors'
        # errors, three more operations
        gt, size = turn(gy.double()[None], positions[None], inv, layout, amp, inverse=True)
        r = (x64.detach().square().mean(-1, keepdim=True) + eps).rsqrt()
        xh = x64.detach() * r
        wg = w64.detach().abs() * size
        bound = r * (wg + xh.abs() * (wg * xh.abs()).mean(-1, keepdim=True))
        err = TURN_ERROR + 2 * NORM_ERROR + 21 * U + 6 * U
        assert ((dx.double()[None] - ex).abs() <= 1.01 * half_step(dtype, ex) + err * bound).all()
        # dw: the terms' errors, and one rounding for each of the rows summed
        terms = (size * xh.abs()).sum((0, 1, 2))
        rows = tokens * x.shape[1]
        assert ((dw.double() - ew).abs() <= (TURN_ERROR + NORM_ERROR + (rows + 64) * U) * terms).all()


def test_norm_rotate_gradient_against_differences():
    g = gen(11)
    q, k = normal(g, 50, 4, 64), normal(g, 50, 2, 64)
    qw, kw = 1 + 0.3 * normal(g, 64), 1 + 0.3 * normal(g, 64)
    gq, gk = normal(g, 50, 4, 64), normal(g, 50, 2, 64)
    positions, inv = torch.arange(50, device="cuda"), freqs(64)
    grads = ops.norm_rotate_backward(gq, gk, q, k, qw, kw, positions, inv)
    along = [normal(g, *t.shape).double() for t in (q, k, qw, kw)]

    def loss(h):
        a, b, c, d = (t.double() + h * v for t, v in zip((q, k, qw, kw), along))
        y, _ = turn(norm(a[None], c, 1e-6), positions[None], inv)
        z, _ = turn(norm(b[None], d, 1e-6), positions[None], inv)
        return ((y * gq.double()).sum() + (z * gk.double()).sum()).item()

    # fourth-order differences: what they leave out is h^4 = 1e-12 of the fifth derivative
    h = 1e-3
    slope = (8 * (loss(h) - loss(-h)) - (loss(2 * h) - loss(-2 * h))) / (12 * h)
    got = sum((d.double() * v).sum().item() for d, v in zip(grads, along))
    size = sum((d.double() * v).abs().sum().item() for d, v in zip(grads, along))
    assert abs(slope - got) <= 1e-5 * size


def test_norm_rotate_in_place_of_a_projection():
    g = gen(5)
    qkv = normal(g, 19, 6 + 2 * 2, 64, dtype=BF16)
    kept = qkv.clone()
    q, k = qkv[:, :6], qkv[:, 6:8]
    w = torch.ones(64, device="cuda")
    positions = torch.arange(19, device="cuda")
    want = ops.norm_rotate(q, k, w, w, positions, freqs(64))
    got = ops.norm_rotate(q, k, w, w, positions, freqs(64), q_out=q, k_out=k)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(qkv[:, 8:], kept[:, 8:])
    # the gradient in the place of what it is the gradient of
    gq, gk = normal(g, 19, 6, 64, dtype=BF16), normal(g, 19, 2, 64, dtype=BF16)
    q, k = kept[:, :6], kept[:, 6:8]
    want = ops.norm_rotate_backward(gq, gk, q, k, w, w, positions, freqs(64))
    got = ops.norm_rotate_backward(gq, gk, q, k, w, w, positions, freqs(64), dq=gq, dk=k)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_norm_gradient_of_no_tokens_is_zero():
    e = torch.empty(0, 4, 64, device="cuda")
    w = torch.ones(64, device="cuda")
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    dq, dk, dqw, dkw = ops.norm_rotate_backward(e, e[:, :2], e, e[:, :2], w, w, none, freqs(64))
    assert dq.shape == (0, 4, 64) and dk.shape == (0, 2, 64)
    assert not dqw.any() and not dkw.any()


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("tokens,heads,kv,dim,rotary,page,heads_first,index", [
    (1, 8, 8, 128, 128, 16, False, torch.int64), (37, 6, 2, 64, 32, 16, False, torch.int32),
    (300, 5, 1, 80, 80, 24, True, torch.int64), (64, 4, 4, 33, 10, 1, False, torch.int32), (9, 8, 2, 256, 64, 128, True, torch.int64),
])
def test_append_paged(dtype, tokens, heads, kv, dim, rotary, page, heads_first, index):
    g = gen(tokens)
    pages = -(-tokens // page) + 2
    shape = (pages, kv, page, dim) if heads_first else (pages, page, kv, dim)
    caches = [normal(g, *shape, dtype=dtype) for _ in range(2)]
    kc, vc = (c.transpose(1, 2) if heads_first else c for c in caches)
    before = kc.clone(), vc.clone()
    qkv = normal(g, tokens, heads + 2 * kv, dim, dtype=dtype)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens].to(index)
    slots[tokens // 3 + 1::7] = -1                                     # (none of a single token)
    positions = torch.randint(0, 100000, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    inv = freqs(rotary)
    w = 1 + 0.3 * normal(g, dim)
    got = ops.append_paged(k, v, kc, vc, slots, positions=positions, inv_freq=inv, layout="interleaved",
                           k_weight=w, q=q, q_weight=w, eps=1e-5)
    y, size = turn(norm(as_rows(q), w.double(), 1e-5), positions[None], inv, "interleaved")
    check_turn(got[None], y, size, dtype, extra=NORM_ERROR)
    y, size = turn(norm(as_rows(k), w.double(), 1e-5), positions[None], inv, "interleaved")
    put = slots >= 0
    at = slots[put].long()
    check_turn(kc[at // page, at % page][None], y[:, put], size[:, put], dtype, extra=NORM_ERROR)
    assert torch.equal(vc[at // page, at % page], v[put])
    other = torch.ones(pages, page, dtype=torch.bool, device="cuda")
    other[at // page, at % page] = False
    assert torch.equal(kc[other], before[0][other]) and torch.equal(vc[other], before[1][other])


def test_append_without_rotation_copies():
    g = gen(1)
    cache = normal(g, 5, 2, 8, 4, 64, dtype=F16)                     # both caches in one tensor
    kc, vc = cache[:, 0], cache[:, 1]
    k, v = normal(g, 11, 4, 64, dtype=F16), normal(g, 11, 4, 64, dtype=F16)
    slots = torch.arange(3, 14, device="cuda")
    assert ops.append_paged(k, v, kc, vc, slots) is None
    assert torch.equal(kc.reshape(-1, 4, 64)[3:14], k) and torch.equal(vc.reshape(-1, 4, 64)[3:14], v)


def test_append_reports_a_slot_outside_the_cache():
    """The kernel's own bounds check leaves the row out; the next call raises."""
    g = gen(2)
    kc, vc = torch.zeros(2, 4, 1, 64, device="cuda"), torch.zeros(2, 4, 1, 64, device="cuda")
    k = normal(g, 3, 1, 64)
    ops.append_paged(k, k, kc, vc, torch.tensor([0, 8, 1 << 40], device="cuda"))
    torch.cuda.synchronize()
    with pytest.raises(native.NativeError, match="outside its pool"):
        ops.append_paged(k, k, kc, vc, torch.tensor([0, 1, 2], device="cuda"))
    assert torch.equal(kc.view(8, 1, 64)[0], k[0]) and not kc.view(8, 1, 64)[1:].any()
    ops.append_paged(k, k, kc, vc, torch.tensor([0, 1, 2], device="cuda"))
    ops.check_errors()
    assert torch.equal(vc.view(8, 1, 64)[:3], k)


def test_an_error_met_in_a_capture_is_raised_again_after_it():
    """A capture cannot reset the device's record: the error stays until a call
    outside of one raises it, and later errors are recorded again."""
    g = gen(4)
    kc, vc = torch.zeros(1, 4, 1, 64, device="cuda"), torch.zeros(1, 4, 1, 64, device="cuda")
    k = normal(g, 1, 1, 64)
    good, bad = torch.tensor([1], device="cuda"), torch.tensor([4], device="cuda")
    ops.append_paged(k, k, kc, vc, good)
    for _ in range(2):
        ops.append_paged(k, k, kc, vc, bad)
        torch.cuda.synchronize()
        with pytest.raises(native.NativeError, match="outside its pool"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                ops.append_paged(k, k, kc, vc, good)
        with pytest.raises(native.NativeError, match="outside its pool"):
            ops.append_paged(k, k, kc, vc, good)
        ops.append_paged(k, k, kc, vc, good)
        torch.cuda.synchronize()
        ops.check_errors()


def test_strides_of_single_tokens_and_heads_may_be_any():
    x = normal(gen(6), 4, 64)
    positions, inv = torch.tensor([7], device="cuda"), freqs(64)
    want = ops.rotate(x.view(1, 4, 64), positions, inv)
    assert torch.equal(ops.rotate(x.as_strided((1, 4, 64), (1 << 33, 64, 1)), positions, inv), want)
    assert torch.equal(ops.rotate(x[:1].as_strided((1, 1, 64), (1 << 33, (1 << 40) + 1, 1)), positions, inv), want[:, :1])
    cache = torch.zeros(3, 64, device="cuda")
    pages = cache.as_strided((3, 1, 1, 64), (64, 1 << 40, 1 << 35, 1))
    values = torch.zeros(3, 1, 1, 64, device="cuda")
    ops.append_paged(x[:1].view(1, 1, 64), x[1:2].view(1, 1, 64), pages, values, torch.tensor([2], device="cuda"),
                     positions=positions, inv_freq=inv)
    assert torch.equal(cache[2], want[0, 0]) and torch.equal(values[2, 0, 0], x[1]) and not cache[:2].any()


# ---------------------------------------------------------------------------
# attention over the paged cache
# ---------------------------------------------------------------------------

def paged(seed, counts, lengths, prefix, heads, kv, dim, page, dtype, heads_first=False, spare=0):
    """Inputs of one call, every cache row that no sequence reaches NaN."""
    g = gen(seed)
    batch = len(counts)
    width = max([1] + [-(-n // page) for n in lengths]) + spare
    shared = -(-prefix // page)
    pool = shared + sum(-(-n // page) for n in lengths) + 3
    order = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    shape = (pool, kv, page, dim) if heads_first else (pool, page, kv, dim)
    caches = [torch.full(shape, float("nan"), dtype=dtype, device="cuda") for _ in range(2)]
    caches = [c.transpose(1, 2) if heads_first else c for c in caches]
    table = torch.full((batch, width), -7, dtype=torch.int32, device="cuda")
    at = shared
    fill = [(order[:shared], prefix)]
    for b, n in enumerate(lengths):
        pages = order[at:at + -(-n // page)]
        at += len(pages)
        table[b, :len(pages)] = pages
        fill.append((pages, n))
    for pages, n in fill:
        for i, x in enumerate(pages.tolist()):
            rows = min(page, n - i * page)
            for c in caches:
                c[x, :rows] = normal(g, rows, kv, dim, dtype=dtype)
    q = normal(g, sum(counts), heads, dim, dtype=dtype)
    offsets = torch.tensor([0] + counts, dtype=torch.int32).cumsum(0).to(torch.int32).cuda()
    return q, *caches, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), order[:shared].clone(), offsets


def check_attend(case, counts, lengths, prefix, scale=None, single=False):
    q, kc, vc, table, lens, pages, offsets = case
    extra = {} if single else dict(query_offsets=offsets, max_queries=max(counts + [1]))
    got, lse = ops.attend_shared_prefix(q, kc, vc, table, lens, prefix_pages=pages, prefix_length=prefix,
                                        scale=scale, return_lse=True, **extra)
    again = ops.attend_shared_prefix(q, kc, vc, table, lens, prefix_pages=pages, prefix_length=prefix, scale=scale,
                                     **extra)
    assert torch.equal(got, again)
    want, wlse, tol, ltol = attend(q, kc, vc, table, lens, pages, prefix, counts,
                                   q.shape[-1] ** -0.5 if scale is None else scale)
    ops.check_errors()
    off = (got.double() - want).abs() - tol
    assert off.max().item() <= 0, f"{off.max().item():.3g} beyond the bound"      # NaN fails too
    assert torch.equal(lse.isinf(), wlse.isinf())
    assert ((lse.double() - wlse).abs() <= ltol)[~wlse.isinf()].all()
    return got, lse


SINGLE = [  # own lengths, prefix, heads, kv_heads, dim, page
    ([1], 0, 1, 1, 64, 16), ([1, 0, 3], 0, 4, 2, 128, 16), ([0, 0], 5, 8, 8, 64, 8), ([17, 64, 1], 1, 8, 1, 128, 16),
    ([100] * 5, 127, 6, 2, 128, 32), ([300, 5, 77, 129], 1000, 32, 8, 128, 64), ([513, 1], 64, 7, 1, 80, 16),
    ([65, 200], 129, 5, 5, 96, 24), ([31, 1000], 333, 16, 4, 256, 128), ([9], 4097, 3, 3, 40, 1),
    ([2000, 3, 1999], 0, 20, 4, 64, 256), ([40] * 40, 260, 16, 2, 64, 16), ([3] * 130, 700, 8, 8, 128, 64),
    ([5, 600], 2000, 64, 1, 128, 128),
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lengths,prefix,heads,kv,dim,page", SINGLE)
def test_attend_single_tokens(dtype, lengths, prefix, heads, kv, dim, page):
    counts = [1] * len(lengths)
    case = paged(sum(lengths) + prefix, counts, lengths, prefix, heads, kv, dim, page, dtype)
    got, lse = check_attend(case, counts, lengths, prefix, single=True)
    if prefix == 0:
        for b, n in enumerate(lengths):
            if n == 0:
                assert not got[b].any() and bool((lse[b] == -math.inf).all())


RAGGED = [  # new tokens, own lengths, prefix, heads, kv_heads, dim, page
    ([1, 2, 3], [1, 2, 3], 0, 4, 4, 64, 16), ([5, 0, 1, 17], [5, 9, 40, 17], 100, 8, 2, 128, 16),
    ([130], [130], 0, 4, 1, 128, 64), ([64, 1, 33], [200, 70, 33], 300, 4, 4, 64, 32),
    ([200, 3], [513, 3], 129, 6, 2, 96, 24), ([7] * 20, [7 + 9 * i for i in range(20)], 515, 10, 2, 128, 128),
    ([1, 300], [1, 300], 64, 3, 1, 256, 16), ([40, 41], [1000, 41], 1111, 32, 8, 80, 8), ([0, 0], [4, 0], 10, 2, 1, 64, 16),
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads_first", [False, True])
@pytest.mark.parametrize("counts,lengths,prefix,heads,kv,dim,page", RAGGED)
def test_attend_several_tokens(dtype, heads_first, counts, lengths, prefix, heads, kv, dim, page):
    if sum(counts) == 0:
        case = paged(1, counts, lengths, prefix, heads, kv, dim, page, dtype, heads_first)
        q, kc, vc, table, lens, pages, offsets = case
        assert ops.attend_shared_prefix(q, kc, vc, table, lens, prefix_pages=pages, prefix_length=prefix,
                                        query_offsets=offsets).shape == (0, heads, dim)
        return
    case = paged(sum(lengths), counts, lengths, prefix, heads, kv, dim, page, dtype, heads_first, spare=3)
    check_attend(case, counts, lengths, prefix)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("count,prefix,heads,kv,dim,page", [
    (40, 13, 32, 8, 128, 16), (40, 200, 32, 8, 128, 128), (33, 128, 24, 8, 64, 32), (50, 257, 16, 8, 80, 8), (129, 1, 8, 8, 64, 256),
])
def test_attend_many_chunks_on_a_short_prefix(dtype, count, prefix, heads, kv, dim, page):
    """Sequences' own blocks take the prefix too; some sequences have fewer new
    tokens or none, none beside the new ones, or a tile and more."""
    counts = [count] * 20 + [0, 1, count - 1, 5]
    lengths = [n + (0, 1, 100, 250)[i % 4] for i, n in enumerate(counts)]
    lengths[20] = 0
    case = paged(prefix, counts, lengths, prefix, heads, kv, dim, page, dtype, spare=2)
    check_attend(case, counts, lengths, prefix)


@pytest.mark.parametrize("spare,hint", [(0, 300), (0, 1), (500, None), (500, 300)])
def test_attend_wide_tables_and_hints(spare, hint):
    """A table far wider than its sequences, and hints about the longest, right or
    wrong, split the work otherwise and change nothing else."""
    lengths = [300, 0, 64, 1]
    for counts in ([1] * 4, [40, 0, 64, 1]):
        q, kc, vc, table, lens, pages, offsets = paged(5, counts, lengths, 500, 8, 2, 128, 16, BF16, spare=spare)
        got = ops.attend_shared_prefix(q, kc, vc, table, lens, prefix_pages=pages, prefix_length=500, max_length=hint,
                                       query_offsets=offsets, max_queries=max(counts))
        want, _, tol, _ = attend(q, kc, vc, table, lens, pages, 500, counts, 128 ** -0.5)
        assert ((got.double() - want).abs() <= tol).all()
    ops.check_errors()


@pytest.mark.parametrize("scale", [0.0, 30.0, -0.5])
def test_attend_scales(scale):
    """Equal weights, weights that all go to one key, and a negative scale."""
    case = paged(4, [1, 1], [70, 300], 200, 4, 2, 64, 16, F16)
    check_attend(case, [1, 1], [70, 300], 200, scale=scale, single=True)


def test_attend_leaves_rows_behind_the_last_sequence():
    counts, lengths = [3, 1], [20, 9]
    q, kc, vc, table, lens, pages, offsets = paged(8, counts, lengths, 40, 8, 2, 128, 16, BF16)
    padded = torch.cat([q, torch.full((5, 8, 128), float("nan"), dtype=BF16, device="cuda")])
    out = torch.full((9, 8 * 2, 128), 7.0, dtype=BF16, device="cuda")[:, ::2]
    got = ops.attend_shared_prefix(padded, kc, vc, table, lens, prefix_pages=pages, prefix_length=40,
                                   query_offsets=offsets, max_queries=3, out=out)
    zeros = torch.cat([q, torch.zeros(5, 8, 128, dtype=BF16, device="cuda")])
    want = ops.attend_shared_prefix(zeros, kc, vc, table, lens, prefix_pages=pages, prefix_length=40,
                                    query_offsets=offsets, max_queries=3)
    assert got is out and torch.equal(out[:4], want[:4]) and bool((out[4:] == 7).all())
    check_attend((q, kc, vc, table, lens, pages, offsets), counts, lengths, 40)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("counts,lengths,prefix,heads,kv,dim", [
    ([6, 2], [40, 2], 30, 2, 2, 64), ([3], [20], 0, 4, 1, 128), ([150, 40], [300, 40], 64, 4, 2, 128), ([200], [210], 0, 1, 1, 64),
    ([5, 9], [100, 9], 20, 2, 1, 256), ([70, 3], [1000, 200], 0, 4, 2, 80), ([40] * 30, [50] * 30, 200, 16, 4, 64),
])
def test_attend_odd_values_reach_only_who_sees_them(dtype, counts, lengths, prefix, heads, kv, dim):
    """Keys and values of new tokens that are infinite or not a number: tokens
    before them keep their results, tokens from them on show them."""
    case = paged(7, counts, lengths, prefix, heads, kv, dim, 16, dtype)
    q, kc, vc, table, lens, pages, offsets = case
    args = dict(prefix_pages=pages, prefix_length=prefix, query_offsets=offsets, max_queries=max(counts))
    want, _, tol, _ = attend(q, kc, vc, table, lens, pages, prefix, counts, dim ** -0.5)
    group = heads // kv

    def as_before(got, rows):
        return bool(((got.double() - want).abs() <= tol)[rows].all())

    def place(b, token):                                             # of a sequence's own token in the cache
        return int(table[b, token // 16]), token % 16

    b, n = 0, counts[0]
    at = lengths[0] - n // 2                                         # the middle of the new tokens
    first = n - n // 2                                               # the first query that sees it
    page, row = place(b, at)
    old = vc[page, row].clone()
    for value, d in ((float("nan"), 3), (float("inf"), 0), (float("-inf"), dim - 1)):
        vc[page, row, kv - 1, d] = value
        got = ops.attend_shared_prefix(q, kc, vc, table, lens, **args)
        vc[page, row] = old
        heads_of = slice((kv - 1) * group, None)
        touched = torch.zeros_like(got, dtype=torch.bool)
        touched[first:n, heads_of, d] = True
        assert as_before(got, ~touched)
        seen = got[first:n, heads_of, d]
        assert bool((seen.isnan() if value != value else seen == value).all())
    # both infinities in one column, the second one token later: a number, then one, then none
    if n >= 4:
        vc[page, row, 0, 1], (p2, r2) = float("inf"), place(b, at + 1)
        keep = vc[p2, r2].clone()
        vc[p2, r2, 0, 1] = float("-inf")
        got = ops.attend_shared_prefix(q, kc, vc, table, lens, **args)
        vc[page, row], vc[p2, r2] = old, keep
        assert bool((got[first, :group, 1] == float("inf")).all()) and bool(got[first + 1:n, :group, 1].isnan().all())
        assert as_before(got, slice(0, first)) and as_before(got, slice(n, None))
    # a key that is not a number: rows that see it are lost, the others are not
    old = kc[page, row].clone()
    kc[page, row, 0, 2] = float("nan")
    got = ops.attend_shared_prefix(q, kc, vc, table, lens, **args)
    kc[page, row] = old
    touched = torch.zeros_like(got, dtype=torch.bool)
    touched[first:n, :group] = True
    assert as_before(got, ~touched) and bool(got[first:n, :group].isnan().all())
    ops.check_errors()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("counts,lengths,prefix,heads,kv,dim", [
    ([1] * 4, [50, 3, 200, 9], 300, 8, 2, 128), ([1] * 30, [50] * 30, 300, 8, 2, 128), ([40, 20], [100, 30], 200, 8, 2, 64),
    ([100], [150], 0, 4, 1, 128),
])
def test_attend_queries_that_are_no_numbers(dtype, counts, lengths, prefix, heads, kv, dim):
    """They show in their own row and nowhere else; scores of minus infinity
    throughout count as nothing seen."""
    q, kc, vc, table, lens, pages, offsets = paged(3, counts, lengths, prefix, heads, kv, dim, 16, dtype)
    args = dict(prefix_pages=pages, prefix_length=prefix, query_offsets=offsets, max_queries=max(counts), return_lse=True)
    want, wlse = ops.attend_shared_prefix(q, kc, vc, table, lens, **args)
    others = torch.ones(q.shape[:2], dtype=torch.bool, device="cuda")
    others[-1, -1] = False
    old = q[-1, -1].clone()
    for value in (math.nan, math.inf):
        q[-1, -1, 5] = value
        got, lse = ops.attend_shared_prefix(q, kc, vc, table, lens, **args)
        q[-1, -1] = old
        assert torch.equal(got[others], want[others]) and torch.equal(lse[others], wlse[others])
        assert got[-1, -1].isnan().all() and lse[-1, -1].isnan()
    q[-1, -1] = 0
    q[-1, -1, 5] = 1
    kc[..., kv - 1, :] = 0
    kc[..., kv - 1, 5] = -math.inf
    got, lse = ops.attend_shared_prefix(q, kc, vc, table, lens, **args)
    assert not got[-1, -1].any() and lse[-1, -1] == -math.inf


def test_attend_query_strides():
    counts, lengths = [1, 1, 1], [20, 9, 33]
    q, kc, vc, table, lens, pages, _ = paged(8, counts, lengths, 40, 6, 2, 64, 16, F16)
    want = ops.attend_shared_prefix(q, kc, vc, table, lens, prefix_pages=pages, prefix_length=40)
    odd = torch.zeros(3, 6, 65, dtype=F16, device="cuda")
    odd[..., 1:] = q
    heads_first = q.transpose(0, 1).contiguous().transpose(0, 1)
    for x in (odd[..., 1:], heads_first, torch.cat([q, q, q], 1)[:, 6:12]):
        assert torch.equal(ops.attend_shared_prefix(x, kc, vc, table, lens, prefix_pages=pages, prefix_length=40), want)


@pytest.mark.parametrize("heads,kv", [(4, 2), (64, 2)])
def test_attend_reports_bad_pages_lengths_and_offsets(heads, kv):
    """The kernels check what only the device sees: a bad page reads as zeros,
    a length beyond the table is cut to it, and the next call raises."""
    counts, lengths = [1, 1], [40, 64]
    case = paged(3, counts, lengths, 64, heads, kv, 64, 16, F16)
    q, kc, vc, table, lens, pages, offsets = case
    kc.nan_to_num_(0.0), vc.nan_to_num_(0.0)
    good = ops.attend_shared_prefix(q, kc, vc, table, lens, prefix_pages=pages, prefix_length=64)
    for bad in (kc.shape[0], -1, 1 << 30):
        t, shared = table.clone(), pages.clone()
        t[0, 1] = bad
        shared[2] = bad
        got = ops.attend_shared_prefix(q, kc, vc, t, lens, prefix_pages=pages, prefix_length=64)
        torch.cuda.synchronize()
        with pytest.raises(native.NativeError, match="outside its pool"):
            ops.check_errors()
        assert torch.equal(got[1], good[1]) and bool(got.isfinite().all())
        ops.attend_shared_prefix(q, kc, vc, table, lens, prefix_pages=shared, prefix_length=64)
        torch.cuda.synchronize()
        with pytest.raises(native.NativeError, match="outside its pool"):
            ops.check_errors()
    for n in (-3, 1 << 20):
        other = lens.clone()
        other[0] = n
        got = ops.attend_shared_prefix(q, kc, vc, table.clamp_min(0), other, prefix_pages=pages, prefix_length=64)
        torch.cuda.synchronize()
        with pytest.raises(native.NativeError, match="outside its pool"):
            ops.check_errors()
        assert torch.equal(got[1], good[1])
    for o in ([0, 1, 99], [-4, 1, 2], [0, 2, 1], [0, 0, 2]):
        ops.attend_shared_prefix(q, kc, vc, table, lens, prefix_pages=pages, prefix_length=64,
                                 query_offsets=torch.tensor(o, dtype=torch.int32, device="cuda"), max_queries=1)
        torch.cuda.synchronize()
        with pytest.raises(native.NativeError, match="outside its pool"):
            ops.check_errors()
    assert torch.equal(ops.attend_shared_prefix(q, kc, vc, table, lens, prefix_pages=pages, prefix_length=64), good)


def test_attend_far_into_a_large_cache():
    """Pages whose rows lie beyond 2^32 bytes of the cache's start."""
    pages, page, kv, dim = 40000, 64, 4, 256                         # 5.2 GB a cache
    kc = torch.zeros(pages, page, kv, dim, dtype=F16, device="cuda")
    vc = torch.zeros_like(kc)
    g = gen(6)
    table = torch.tensor([[39999, 3]], dtype=torch.int32, device="cuda")
    k, v = normal(g, 100, kv, dim, dtype=F16), normal(g, 100, kv, dim, dtype=F16)
    i = torch.arange(100, device="cuda")
    ops.append_paged(k, v, kc, vc, table[0].long()[i // page] * page + i % page)
    lens = torch.tensor([100], dtype=torch.int32, device="cuda")
    q = normal(g, 1, 8, dim, dtype=F16)
    shared = torch.tensor([39999, 39998], dtype=torch.int32, device="cuda")
    check_attend((q, kc, vc, table, lens, shared, None), [1], [100], 70, single=True)
    q = normal(g, 100, 8, dim, dtype=F16)
    check_attend((q, kc, vc, table, lens, shared, torch.tensor([0, 100], dtype=torch.int32, device="cuda")), [100], [100], 70)


def test_decode_step_through_all_operators():
    """A prompt and three decode steps of one layer: normed and rotated queries
    and keys into the cache, attention over prefix and own tokens; against dense
    attention over everything, in 64 bits of the rows that the operators stored."""
    g = gen(21)
    heads, kv, dim, page, batch, prefix = 8, 2, 64, 16, 3, 50
    inv = freqs(dim)
    w = 1 + 0.2 * normal(g, dim)
    kc = torch.full((40, page, kv, dim), float("nan"), dtype=BF16, device="cuda")
    vc = kc.clone()
    shared = torch.tensor([7, 2, 30, 11], dtype=torch.int32, device="cuda")
    table = torch.arange(12, 12 + batch * 4, dtype=torch.int32, device="cuda").view(batch, 4)

    def project(n):
        x = normal(g, n, heads + 2 * kv, dim, dtype=BF16)
        return x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:]

    def slots(pages, first, n):
        i = torch.arange(first, first + n, device="cuda")
        return pages.long()[i // page] * page + i % page

    q, k, v = project(prefix)
    ops.append_paged(k, v, kc, vc, slots(shared, 0, prefix), positions=torch.arange(prefix, device="cuda"), inv_freq=inv,
                     k_weight=w)
    have = [0] * batch
    for counts in ([9, 1, 5], [1, 1, 1], [1, 1, 1], [2, 1, 3]):
        n = sum(counts)
        q, k, v = project(n)
        at = torch.cat([slots(table[b], have[b], c) for b, c in enumerate(counts)])
        pos = torch.cat([torch.arange(prefix + have[b], prefix + have[b] + c, device="cuda") for b, c in enumerate(counts)])
        qr, _ = ops.norm_rotate(q, k, w, w, pos, inv)
        got = ops.append_paged(k, v, kc, vc, at, positions=pos, inv_freq=inv, k_weight=w, q=q, q_weight=w)
        assert torch.equal(got, qr)
        have = [h + c for h, c in zip(have, counts)]
        lens = torch.tensor(have, dtype=torch.int32, device="cuda")
        offsets = torch.tensor([0] + counts, device="cuda").cumsum(0).to(torch.int32)
        check_attend((qr, kc, vc, table, lens, shared, offsets), counts, have, prefix)


# ---------------------------------------------------------------------------
# streams and graphs
# ---------------------------------------------------------------------------

def test_other_stream_and_graph_replay():
    g = gen(9)
    x = normal(g, 64, 8, 128, dtype=BF16)
    gy = normal(g, 64, 8, 128, dtype=BF16)
    w = torch.ones(128, device="cuda")
    positions, inv = torch.arange(64, device="cuda"), freqs(128)

    def step():
        a, b = ops.norm_rotate(x, x[:, :2], w, w, positions, inv)
        return (a, b) + ops.norm_rotate_backward(gy, gy[:, :2], x, x[:, :2], w, w, positions, inv)

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs = [], []
    for _ in range(2):                                               # two graphs, each with its own workspace
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step())
        graphs.append(graph)
    x.copy_(normal(g, 64, 8, 128, dtype=BF16))
    want = step()
    for graph in graphs:
        graph.replay()
    torch.cuda.synchronize()
    for got in outs:
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_attend_on_another_stream_and_in_two_graphs():
    counts, lengths = [1] * 6, [100, 40, 260, 1, 77, 513]
    q, kc, vc, table, lens, pages, _ = paged(3, counts, lengths, 600, 32, 8, 128, 16, BF16)

    def step():
        return ops.attend_shared_prefix(q, kc, vc, table, lens, prefix_pages=pages, prefix_length=600, return_lse=True)

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    here = step()                                                    # two calls at once
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, got, here))
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step())
        graphs.append(graph)
    q.copy_(normal(gen(77), *q.shape, dtype=BF16))
    lens.sub_(1).clamp_min_(1)
    want = step()
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for graph, s in zip(graphs, streams):
        with torch.cuda.stream(s):
            graph.replay()
    torch.cuda.synchronize()
    for got in outs:
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---------------------------------------------------------------------------
# the C entries
# ---------------------------------------------------------------------------

def test_c_entry_of_a_tensor_without_heads():
    """It has no rows, and none of its addresses is read: they may all be 0."""
    from test_ops import FLAG_NORM, FLAG_ROTATE, HEAD, ROTARY_BYTES, ROWS
    g = gen(13)
    tokens, heads, dim = 5, 3, 64
    x, gy, w = normal(g, tokens, heads, dim), normal(g, tokens, heads, dim), 1 + 0.3 * normal(g, dim)
    positions, inv = torch.arange(tokens, device="cuda"), freqs(dim)
    none = x[:, :0]
    want = ops.norm_rotate(x, none, w, w, positions, inv)[0]
    want_dx, _, want_dw, _ = ops.norm_rotate_backward(gy, none, x, none, w, w, positions, inv)
    entries = native.library()
    entries.tila_rotary_workspace.restype = ctypes.c_uint64

    def call(entry, out, grad, weight_grads, first):
        flags = FLAG_ROTATE | FLAG_NORM
        full = ROWS.pack(x.data_ptr(), out.data_ptr(), w.data_ptr(), grad, 0, heads * dim, dim, 0, heads * dim, dim, 0,
                         heads * dim, dim, heads, flags | 8)
        empty = ROWS.pack(0, 0, 0, 0, *[0] * 9, 0, flags)
        rows = (full + empty if first else empty + full) + bytes(ROWS.size)

        def args(space, size):
            return HEAD.pack(ROTARY_BYTES, 0, 1, tokens, dim, dim, 0, 0, 1.0, 1e-6, positions.data_ptr(), 0, 1,
                             inv.data_ptr(), 0, 0, 0, 0, 1, 2, 0, 0, torch.cuda.current_stream().cuda_stream, space, size,
                             *weight_grads) + rows

        size = entries.tila_rotary_workspace(args(0, 0)) if grad else 0
        space = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
        log = ctypes.create_string_buffer(512)
        assert getattr(entries, entry)(args(space.data_ptr(), size), log, ctypes.c_size_t(512)) == native.TILA_OK, log.value
        torch.cuda.synchronize()

    for first in (True, False):
        out, dx = torch.empty_like(x), torch.empty_like(x)
        dw = torch.full((2, dim), 7.0, device="cuda")
        call("tila_rotary_rows", out, 0, (0, 0), first)
        call("tila_rotary_norm_backward", dx, gy.data_ptr(), (dw[0].data_ptr(), dw[1].data_ptr()), first)
        assert torch.equal(out, want) and torch.equal(dx, want_dx)
        assert torch.equal(dw[0 if first else 1], want_dw) and not dw[1 if first else 0].any()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("counts,prefix,heads,kv,dim,page", [
    ([256, 100, 156], 2000, 64, 8, 64, 24), ([130, 3, 77], 1700, 64, 8, 256, 16), ([300, 1], 1100, 96, 32, 80, 1),
])
def test_attend_many_rows_in_the_narrow_form(dtype, counts, prefix, heads, kv, dim, page):
    """Page and head sizes that the wide form does not take, with blocks enough
    for chunks of the prefix longer than 512 keys."""
    lengths = [n + 7 * i for i, n in enumerate(counts)]
    case = paged(sum(counts), counts, lengths, prefix, heads, kv, dim, page, dtype)
    check_attend(case, counts, lengths, prefix)


# ---------------------------------------------------------------------------
# beside autograd
# ---------------------------------------------------------------------------

def test_tensors_written_in_place_count_it():
    """A tensor that another operation saved for its backward pass and that an
    operator then wrote is found out, as after torch's own in-place operations."""
    g = gen(17)
    positions, inv, w = torch.arange(6, device="cuda"), freqs(64), torch.ones(64, device="cuda")
    q, k, gq, gk = (normal(g, 6, h, 64, dtype=BF16) for h in (4, 2, 4, 2))
    kc, vc = normal(g, 2, 16, 2, 64, dtype=BF16), normal(g, 2, 16, 2, 64, dtype=BF16)
    out = torch.empty_like(q)
    table, lens = torch.zeros(6, 1, dtype=torch.int32, device="cuda"), torch.ones(6, dtype=torch.int32, device="cuda")
    slots = torch.arange(6, device="cuda")
    calls = [
        (lambda: ops.rotate(q, positions, inv, out=out), [out]),
        (lambda: ops.rotate(q, positions, inv, out=q), [q]),
        (lambda: ops.rotate_backward(gq, positions, inv, out=gq), [gq]),
        (lambda: ops.norm_rotate(q, k, w, w, positions, inv, q_out=q, k_out=k), [q, k]),
        (lambda: ops.norm_rotate_backward(gq, gk, q, k, w, w, positions, inv, dq=q, dk=gk), [q, gk]),
        (lambda: ops.append_paged(k, k, kc, vc, slots), [kc, vc]),
        (lambda: ops.append_paged(k, k, kc, vc, slots, q=q, q_out=out), [kc, vc, out]),
        (lambda: ops.attend_shared_prefix(q, kc, vc, table, lens, out=out), [out]),
    ]
    everything = [q, k, gq, gk, kc, vc, out, w, inv, positions, table, lens, slots]
    for call, wrote in calls:
        before = [t._version for t in everything]
        call()
        for t, v in zip(everything, before):
            assert (t._version > v) == any(t is x for x in wrote)
    scale = torch.ones((), device="cuda", requires_grad=True)
    y = (q.float() * scale).sum() + (out * scale).float().sum()      # saves `out`
    ops.rotate(q, positions, inv, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():                                     # tensors without versions
        x = q.clone()
        assert ops.rotate(x, positions, inv, out=x) is x
        cache = kc.clone()
        ops.append_paged(k, k, cache, vc, slots)
    assert torch.equal(x, out)


def test_first_operator_in_inference_mode():
    """The error block that it makes outlives the mode: a device error is raised
    and reset outside of it too."""
    code = """
import torch
from tila_b200 import native, ops
kc, k = torch.zeros(1, 4, 1, 64, device="cuda"), torch.ones(1, 1, 64, device="cuda")
vc = kc.clone()
good, bad = torch.tensor([1], device="cuda"), torch.tensor([4], device="cuda")
with torch.inference_mode():
    ops.append_paged(k, k, kc, vc, good)
for _ in range(2):
    ops.append_paged(k, k, kc, vc, bad)
    torch.cuda.synchronize()
    try:
        ops.append_paged(k, k, kc, vc, good)
    except native.NativeError as e:
        assert "outside its pool" in str(e)
    else:
        raise SystemExit("no error")
    ops.append_paged(k, k, kc, vc, good)
    torch.cuda.synchronize()
    ops.check_errors()
print("raised and reset")
"""
    got = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120,
                         cwd=Path(__file__).resolve().parents[1])
    assert got.returncode == 0 and "raised and reset" in got.stdout, got.stderr


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotate_sines_near_zero(layout):
    """Angles close to whole half turns, whose sines are far smaller than the
    rounding of the angle itself to 32 bits."""
    g = gen(23)
    half, tokens = 32, 200
    positions = torch.arange(1, tokens + 1, device="cuda")
    # position * inv_freq = a few half turns and up to 1e-5 of one
    inv = math.pi * (1 + 1e-5 * torch.rand(half, generator=g, device="cuda", dtype=torch.float64)) * torch.arange(
        1, half + 1, device="cuda")
    x = torch.zeros(tokens, 1, 2 * half, device="cuda")
    first = slice(0, half) if layout == "half" else slice(0, None, 2)
    second = slice(half, None) if layout == "half" else slice(1, None, 2)
    x[..., first] = 1
    y = ops.rotate(x, positions, inv, layout=layout).double()[:, 0]
    angle = positions.double()[:, None] * inv
    c, s = angle.cos(), angle.sin()
    # sincospi is off by 2 ulp (4 U); the sum with its correction, the amplitude and the row's product by U each;
    # the correction itself (at most pi 2^-25 < 1e-7) by 3 U of it (remainder, pi, product); the angle in 64 bits by
    # 2^-51 of itself (position * inv_freq * 1/2pi, here and in the reference)
    bound, least = 8 * U, 2 ** -50 * angle + 4 * U * 1e-7
    assert ((y[:, second] - s).abs() <= bound * s.abs() + least).all()
    assert ((y[:, first] - c).abs() <= bound * c.abs() + least).all()
    assert bool((s.abs() < 1e-3).any())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("page", [16, 128])
@pytest.mark.parametrize("dim", [8, 40, 56, 72, 104, 136, 200, 248])
def test_attend_head_sizes_that_end_inside_a_box(dtype, page, dim):
    """Boxes of 64 elements that are wider than the rows, or lie behind them wholly: few
    rows (narrow form), many (wide form up to 128 elements: prefix and own tokens
    apart, and own blocks that take a short prefix too)."""
    for counts, lengths, prefix in (([1, 1, 1], [40, 129, 3], 300), ([40, 33, 2], [200, 33, 70], 300),
                                    ([70] * 20, [75] * 20, 13)):
        case = paged(dim + prefix, counts, lengths, prefix, 8, 2, dim, page, dtype)
        check_attend(case, counts, lengths, prefix)


@pytest.mark.parametrize("what", ["norm", "append", "attend narrow", "attend wide", "attend chunks"])
def test_first_call_of_an_operator_in_a_capture(what):
    """In a process where only another operator has run on the device: its kernels
    are loaded, and given their shared memory, while the graph is captured."""
    code = """
import sys, torch
sys.path.insert(0, "tests")
from test_gpu_ops import *
what = sys.argv[1]
x, w, inv, positions = normal(gen(1), 40, 4, 64, dtype=BF16), torch.ones(64, device="cuda"), freqs(64), torch.arange(40, device="cuda")
ops.rotate(x, positions, inv)
if what.startswith("attend"):
    counts = [40, 3] if "chunks" in what else [1] * (2 if "narrow" in what else 20)
    q, kc, vc, table, lens, pages, offsets = paged(1, counts, [60] * len(counts), 300, 8, 2, 64, 16, BF16)
    f = lambda: [ops.attend_shared_prefix(q, kc, vc, table, lens, prefix_pages=pages, prefix_length=300,
                                          query_offsets=offsets, max_queries=max(counts))]
elif what == "norm":
    f = lambda: [*ops.norm_rotate(x, x, w, w, positions, inv), *ops.norm_rotate_backward(x, x, x, x, w, w, positions, inv)]
else:
    caches = torch.zeros(2, 3, 16, 4, 64, dtype=BF16, device="cuda")
    f = lambda: [ops.append_paged(x, x, *caches, positions, positions=positions, inv_freq=inv, q=x), caches]
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = f()
for t in got:
    t.zero_()
graph.replay()
torch.cuda.synchronize()
got = [t.clone() for t in got]
assert all(torch.equal(a, b) for a, b in zip(got, f())) and bool(got[0].any())
ops.check_errors()
print("captured")
"""
    got = subprocess.run([sys.executable, "-c", code, what], capture_output=True, text=True, timeout=120,
                         cwd=Path(__file__).resolve().parents[1])
    assert got.returncode == 0 and "captured" in got.stdout, got.stderr
