"""The decode-path operators on the GPU against their definitions in 64 bits."""

import math

import pytest
import torch

from tila_b200 import native, ops
from ops_support import NORM_ERROR, TURN_ERROR, U, check_turn, half_step, norm, turn

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
    (9, 2, 2, 512, 64), (3, 1, 2, 20, 0),
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
