"""Operators that stand around a model's attention, as hand-written sm_100a
kernels behind the C ABI (``include/tila_b200.h``, ``csrc/ops``).

* :func:`rotate`, :func:`rotate_backward` - rotary positions;
* :func:`norm_rotate`, :func:`norm_rotate_backward` - the norm of each query
  and key head with the rotation in the same pass, and its gradients;
* :func:`append_paged` - keys and values into a paged cache, rotated (and
  normed) on the way, the queries in the same launch;
* :func:`attend_shared_prefix` - attention over such a cache, of a batch whose
  sequences share a prefix that is read once for all;
* :func:`rotary_frequencies` - the frequencies that these take, scaled for
  long contexts.

Like the kernels of a Tila program they take CUDA tensors of any strides whose
last dimension is contiguous, write into tensors that the caller may supply,
and run asynchronously on the current PyTorch stream of the tensors' device.
They are not recorded by autograd: a gradient is a call of its own.  Every call
can be captured into a CUDA graph once an operator has run on the device.
Wrong arguments raise ``ValueError`` before anything is launched.  What only the
device can see (a slot outside the cache) leaves the access out, is recorded as
a device error, and is raised by the next operator on that device or by
:func:`check_errors`.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import native

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_LAYOUTS = {"half": 0, "interleaved": 1}

# ---------------------------------------------------------------------------
# device errors
# ---------------------------------------------------------------------------

ERROR_CODES = {
    1: "a bounded wait timed out; the operator stopped early and its outputs are incomplete",
    2: "tensor memory allocation failed",
    5: "an index outside its pool (a cache slot or a page) was left out",
}


class _ErrorBlock:
    """The error block that every operator on a device is given, and the
    page-locked word that the kernels copy its first error to."""

    def __init__(self, index):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the first operator on a device cannot be captured into a CUDA graph: "
                               "call it once before the capture")
        with torch.cuda.device(index):
            self.block = torch.zeros(native.ERROR_BLOCK_BYTES // 4, dtype=torch.int32, device="cuda")
            host, address = native.host_word_alloc()
            self.block.view(torch.int64)[1] = address
            torch.cuda.current_stream().synchronize()   # operators on other streams read it
        self.word = ctypes.c_uint32.from_address(host)
        self.address = self.block.data_ptr()


_error_blocks = {}


def _error_block(index):
    b = _error_blocks.get(index)
    if b is None:
        b = _error_blocks[index] = _ErrorBlock(index)
    if b.word.value:
        check_errors(index)
    return b.address


def check_errors(device=None) -> None:
    """Raise :class:`native.NativeError` if an operator that ran on ``device``
    recorded a device error.  Does not synchronise: it sees the errors of
    kernels that have reached them."""
    index = device if isinstance(device, int) else None if device is None else torch.device(device).index
    if index is None:
        index = torch.cuda.current_device()
    b = _error_blocks.get(index)
    if b is None or not b.word.value:
        return
    word = b.word.value
    with torch.cuda.device(index):
        b.block[0].zero_()
    b.word.value = 0
    code, where = word >> 24, word & 0xFFFFFF
    raise native.NativeError(native.TILA_ERR_ARGUMENT if code == 5 else native.TILA_ERR_DRIVER,
                             f"an operator launched earlier on cuda:{index} failed: "
                             f"{ERROR_CODES.get(code, f'device error code {code}')} (at {where})")


# ---------------------------------------------------------------------------
# checks of arguments
# ---------------------------------------------------------------------------

def _fail(name, text):
    raise ValueError(f"{name}: {text}")


def _tensor(name, what, t, device=None, dtype=None, rank=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: {what} must be a tensor, not {type(t).__name__}")
    if not t.is_cuda:
        _fail(name, f"{what} must be a CUDA tensor")
    if device is not None and t.device != device:
        _fail(name, f"{what} is on {t.device}, the other tensors on {device}")
    if dtype is not None and t.dtype is not dtype:
        _fail(name, f"{what} must be {dtype}, not {t.dtype}")
    if rank is not None and t.dim() != rank:
        _fail(name, f"{what} must have {rank} dimensions, not {t.dim()}")


def _unit_last(name, what, t):
    """The tensor's strides, whose last must be 1."""
    st = t.stride()
    if st[-1] != 1 and t.shape[-1] > 1 and t.numel():
        _fail(name, f"the last dimension of {what} must be contiguous")
    return st


def _writable(name, what, t):
    """Refuses a result whose elements share memory (an expanded tensor)."""
    if t.is_contiguous():
        return
    span = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if stride < span:
            _fail(name, f"elements of {what} share memory")
        span += (size - 1) * stride


def _extent(sizes, strides):
    return 1 + sum((n - 1) * s for n, s in zip(sizes, strides))


def _range(t):
    """First and last address of a tensor's elements, the last one excluded."""
    p = t.data_ptr()
    n = t.numel() if t.is_contiguous() else _extent(t.shape, t.stride()) if t.numel() else 0
    return p, p + n * t.element_size()


def _apart(name, what, a, other, b, same=False):
    """Refuses a result ``a`` that overlaps ``b``.  It may lie between the rows
    or pages of ``b`` (two parts of one tensor) and, with ``same``, be exactly the
    elements of ``b`` (a result in the place of its source)."""
    pa, ea = _range(a)
    pb, eb = _range(b)
    if pa >= eb or pb >= ea or pa == ea or pb == eb:
        return
    sa, sb, size = a.stride(), b.stride(), a.element_size()
    if a.dtype is b.dtype:
        if same and pa == pb and a.shape == b.shape and sa == sb:
            return
        # equal steps in the outer dimensions: both lie in windows of one period
        for outer in range(1, a.dim()):
            period = sa[outer - 1]
            if b.dim() != a.dim() or a.shape[:outer] != b.shape[:outer] or sa[:outer] != sb[:outer] or \
                    period <= 0 or (pb - pa) % size:
                break
            shift = (pb - pa) // size % period
            if all(s % period == 0 for s in sa[:outer]) and shift >= _extent(a.shape[outer:], sa[outer:]) and \
                    period - shift >= _extent(b.shape[outer:], sb[outer:]):
                return
    _fail(name, f"{what} overlaps {other}")


def _rows_shape(name, what, x):
    _tensor(name, what, x)
    if x.dtype not in _DTYPES:
        _fail(name, f"{what} must be float32, float16 or bfloat16, not {x.dtype}")
    if x.dim() not in (3, 4):
        _fail(name, f"{what} must be (tokens, heads, dim) or (batch, tokens, heads, dim)")
    if not 1 <= x.shape[-1] <= 512:
        _fail(name, f"{what} must have heads of 1 to 512 elements, not {x.shape[-1]}")


def _strides3(st):
    """(batch, token, head) strides of a (batch,) tokens, heads, dim tensor."""
    return st[:3] if len(st) == 4 else (0, st[0], st[1])


def _result(name, what, out, like, own, others=()):
    """The result tensor: a new one, or the caller's after its checks.  It may
    take the place of one of ``own`` and overlaps none of ``others``."""
    if out is None:
        return like.new_empty(like.shape)
    _tensor(name, what, out, like.device, like.dtype)
    if out.shape != like.shape:
        _fail(name, f"{what} must have the shape {tuple(like.shape)}, not {tuple(out.shape)}")
    _unit_last(name, what, out)
    _writable(name, what, out)
    for other, t in own:
        _apart(name, what, out, other, t, same=True)
    for other, t in others:
        _apart(name, what, out, other, t)
    return out


def _positions(name, positions, inv_freq, x, layout):
    """(positions, batch step, token step, wide, inv_freq, rotary) of the call."""
    if layout not in _LAYOUTS:
        _fail(name, f"layout must be 'half' or 'interleaved', not {layout!r}")
    _tensor(name, "positions", positions, x.device)
    if positions.dtype is not torch.int64 and positions.dtype is not torch.int32:
        _fail(name, f"positions must be int32 or int64, not {positions.dtype}")
    tokens = x.shape[:-2]
    st = positions.stride()
    if positions.shape == tokens:
        step = st if len(st) == 2 else (0, st[0])
    elif len(tokens) == 2 and positions.shape == tokens[1:]:
        step = (0, st[0])
    else:
        _fail(name, f"positions must have one position per token, {tuple(tokens)}, not {tuple(positions.shape)}")
    _tensor(name, "inv_freq", inv_freq, x.device, torch.float64, 1)
    rotary = 2 * inv_freq.shape[0]
    if rotary > x.shape[-1]:
        _fail(name, f"inv_freq rotates {rotary} elements, the heads have {x.shape[-1]}")
    if rotary > 2 and inv_freq.stride(0) != 1:
        _fail(name, "inv_freq must be contiguous")
    return positions.data_ptr(), step[0], step[1], positions.dtype is torch.int64, inv_freq.data_ptr(), rotary


def _weight(name, what, w, x):
    _tensor(name, what, w, x.device, None, 1)
    if w.dtype is not torch.float32 and w.dtype is not x.dtype:
        _fail(name, f"{what} must be float32 or {x.dtype}, not {w.dtype}")
    if w.shape[0] != x.shape[-1] or (w.shape[0] > 1 and w.stride(0) != 1):
        _fail(name, f"{what} must be a contiguous vector of {x.shape[-1]} elements")
    return native.ROWS_WEIGHT_F32 if w.dtype is torch.float32 else 0


def _rows(src, dst, flags, weight=0, grad=None):
    """One tensor of a call, as tila_op_rows."""
    return native.ROWS.pack(src.data_ptr(), dst.data_ptr(), weight, 0 if grad is None else grad.data_ptr(),
                            *_strides3(src.stride()),
                            *(dst.stride()[:3] if flags & native.ROWS_PAGED else _strides3(dst.stride())),
                            *((0, 0, 0) if grad is None else _strides3(grad.stride())), src.shape[-2], flags)


_NO_ROTATION = (0, 0, 0, False, 0, 0)


def _run_rotary(entry, x, rows, turn, layout, amplitude, inverse=False, eps=0.0, slots=None, num_slots=0, page=0,
                workspace=False, weight_grad=(0, 0)):
    """Packs tila_rotary_args and launches ``entry`` on x's device and its
    current stream."""
    positions, step_b, step_t, index64, inv_freq, rotary = turn
    shape = x.shape
    batch, tokens = (1, shape[0]) if len(shape) == 3 else shape[:2]
    slot = slot_step = 0
    if slots is not None:
        slot, slot_step = slots.data_ptr(), slots.stride(0)
        index64 = index64 | (2 if slots.dtype is torch.int64 else 0)
    tail = b"".join(rows) + native.NO_ROWS * (native.ROTARY_ROWS - len(rows))
    index = x.device.index

    def go():
        head = [native.ROTARY_BYTES, _DTYPES[x.dtype], batch, tokens, shape[-1], rotary, _LAYOUTS[layout],
                int(inverse), float(amplitude), float(eps), positions, step_b, step_t, inv_freq, slot, slot_step,
                num_slots, page, index64, len(rows), 0, _error_block(index),
                torch.cuda.current_stream(index).cuda_stream, 0, 0, *weight_grad]
        if workspace:
            need = native.rotary_workspace(native.ROTARY_HEAD.pack(*head) + tail)
            space = torch.empty(need, dtype=torch.uint8, device=x.device)
            head[23], head[24] = space.data_ptr(), need
        native.call_op(entry, native.ROTARY_HEAD.pack(*head) + tail)

    if torch.cuda.current_device() == index:
        go()
    else:
        with torch.cuda.device(index):
            go()


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------

def rotary_frequencies(rotary, base=10000.0, scaling=None, factor=1.0, original_length=None, beta_fast=32.0,
                       beta_slow=1.0, device=None):
    """``(inv_freq, amplitude)`` of a rotation of ``rotary`` elements: the
    radians per position of each pair, ``base ** (-2 i / rotary)``, as a
    float64 tensor on ``device`` (default: the current CUDA device).

    ``scaling`` stretches them for contexts ``factor`` times as long as the
    model was trained on:

    * ``"linear"``: every frequency divided by ``factor``;
    * ``"ntk"``: the base times ``factor ** (rotary / (rotary - 2))``, so that the
      slowest pair is stretched by ``factor`` and the fastest not at all;
    * ``"yarn"`` (Peng et al., 2023): pairs that turn more than ``beta_fast`` times over
      ``original_length`` positions stay, those that turn less than ``beta_slow``
      times are divided by ``factor``, with a ramp over the pairs between; the
      amplitude is ``0.1 ln(factor) + 1``.
    """
    name = "rotary_frequencies"
    if rotary < 0 or rotary % 2:
        _fail(name, f"rotary must be an even number of elements, not {rotary}")
    if not (base > 0 and factor >= 1.0):
        _fail(name, "base must be positive and factor at least 1")
    if scaling not in (None, "linear", "ntk", "yarn"):
        _fail(name, f"scaling must be None, 'linear', 'ntk' or 'yarn', not {scaling!r}")
    if scaling == "ntk" and rotary > 2:
        base = base * factor ** (rotary / (rotary - 2))
    freq = [base ** (-2.0 * i / rotary) for i in range(rotary // 2)]
    amplitude = 1.0
    if scaling == "linear":
        freq = [f / factor for f in freq]
    elif scaling == "yarn":
        if not original_length or original_length < 1:
            _fail(name, "'yarn' needs original_length, the length that the model was trained on")
        if not beta_fast > beta_slow > 0:
            _fail(name, "beta_fast must be above beta_slow, and both positive")

        def pair(turns):     # the pair (not whole) that turns so often over original_length
            return rotary * math.log(original_length / (turns * 2 * math.pi)) / (2 * math.log(base))

        low = max(math.floor(pair(beta_fast)), 0)
        high = min(math.ceil(pair(beta_slow)), rotary - 1)
        high = high + 0.001 if high == low else high
        ramp = [min(1.0, max(0.0, (i - low) / (high - low))) for i in range(rotary // 2)]
        freq = [f * (1 - r) + f / factor * r for f, r in zip(freq, ramp)]
        amplitude = 0.1 * math.log(factor) + 1.0
    return torch.tensor(freq, dtype=torch.float64, device="cuda" if device is None else device), amplitude


def _rotate(name, what, x, positions, inv_freq, layout, amplitude, out, inverse):
    _rows_shape(name, what, x)
    _unit_last(name, what, x)
    turn = _positions(name, positions, inv_freq, x, layout)
    out = _result(name, "out", out, x, ((what, x),))
    _run_rotary("tila_rotary_rows", x, [_rows(x, out, native.ROWS_ROTATE)], turn, layout, amplitude, inverse)
    return out


def rotate(x, positions, inv_freq, *, layout="half", amplitude=1.0, out=None):
    """Rotary positions: each pair of ``x`` (tokens, heads, dim) or (batch,
    tokens, heads, dim) turned by ``position * inv_freq``.

    The first ``2 * len(inv_freq)`` elements of a head rotate, the others are
    copied.  ``layout``: pairs ``(i, i + rotary/2)`` (``"half"``) or ``(2i, 2i + 1)``
    (``"interleaved"``).  ``positions``: int32 or int64, one per token, or (tokens,) for
    every batch entry.  ``amplitude`` multiplies the rotated elements.  ``out`` may
    be ``x`` itself.  float32, float16, bfloat16.
    """
    return _rotate("rotate", "x", x, positions, inv_freq, layout, amplitude, out, False)


def rotate_backward(grad, positions, inv_freq, *, layout="half", amplitude=1.0, out=None):
    """Gradient of :func:`rotate` with respect to ``x``, given that of its
    result: the rotation back, with the same amplitude."""
    return _rotate("rotate_backward", "grad", grad, positions, inv_freq, layout, amplitude, out, True)


def _pair(name, q, k, q_weight, k_weight):
    _rows_shape(name, "q", q)
    _rows_shape(name, "k", k)
    if k.device != q.device or k.dtype is not q.dtype:
        _fail(name, "q and k must have one device and one dtype")
    if k.shape[:-2] != q.shape[:-2] or k.shape[-1] != q.shape[-1]:
        _fail(name, f"q and k must have the same tokens and dim: {tuple(q.shape)} and {tuple(k.shape)}")
    _unit_last(name, "q", q)
    _unit_last(name, "k", k)
    return _weight(name, "q_weight", q_weight, q), _weight(name, "k_weight", k_weight, k)


def norm_rotate(q, k, q_weight, k_weight, positions, inv_freq, *, layout="half", amplitude=1.0, eps=1e-6,
                q_out=None, k_out=None):
    """``(q_out, k_out)``: each head of ``q`` and ``k`` divided by its root mean
    square, times the weight, and rotated, in one pass.

    ``q`` (.., tokens, heads, dim) and ``k`` (.., tokens, kv_heads, dim) may be
    parts of one projection; the weights (dim,) are float32 or of q's dtype.
    The results may be ``q`` and ``k`` themselves.  The other arguments are those
    of :func:`rotate`.
    """
    name = "norm_rotate"
    wide_q, wide_k = _pair(name, q, k, q_weight, k_weight)
    turn = _positions(name, positions, inv_freq, q, layout)
    q_out = _result(name, "q_out", q_out, q, (("q", q),), (("k", k),))
    k_out = _result(name, "k_out", k_out, k, (("k", k),), (("q", q), ("q_out", q_out)))
    flags = native.ROWS_ROTATE | native.ROWS_NORM
    _run_rotary("tila_rotary_rows", q, [_rows(q, q_out, flags | wide_q, q_weight.data_ptr()),
                                        _rows(k, k_out, flags | wide_k, k_weight.data_ptr())],
                turn, layout, amplitude, eps=eps)
    return q_out, k_out


def append_paged(k, v, k_cache, v_cache, slots, *, positions=None, inv_freq=None, layout="half", amplitude=1.0,
                 k_weight=None, q=None, q_weight=None, q_out=None, eps=1e-6):
    """Appends the rows ``k`` and ``v`` (tokens, kv_heads, dim) to a paged cache,
    in place, and returns the queries that go with them (``None`` without ``q``).

    ``k_cache`` and ``v_cache`` are (pages, page_size, kv_heads, dim) in any strides
    (a cache that keeps its heads before its rows is passed transposed).
    ``slots``: int32 or int64, one per token, ``page * page_size + row``; a negative
    slot leaves its token out (padding of a batch), and no two others are equal.
    With ``positions`` and ``inv_freq`` the keys are rotated on the way, with
    ``k_weight`` normed before that (``eps``).  ``q`` (tokens, heads, dim), with
    ``q_weight`` where it is normed too, is prepared in the same launch into
    ``q_out`` (which may be ``q``); the queries of tokens left out are written too.
    """
    name = "append_paged"
    _rows_shape(name, "k", k)
    if k.dim() != 3:
        _fail(name, "k must be (tokens, kv_heads, dim)")
    _tensor(name, "v", v, k.device, k.dtype)
    if v.shape != k.shape:
        _fail(name, f"v must have the shape of k, {tuple(k.shape)}, not {tuple(v.shape)}")
    _unit_last(name, "k", k)
    _unit_last(name, "v", v)
    if (positions is None) != (inv_freq is None):
        _fail(name, "positions and inv_freq go together")
    turn = _NO_ROTATION if positions is None else _positions(name, positions, inv_freq, k, layout)
    turned = 0 if positions is None else native.ROWS_ROTATE
    tokens, kv_heads, dim = k.shape
    _tensor(name, "slots", slots, k.device, None, 1)
    if slots.dtype is not torch.int64 and slots.dtype is not torch.int32:
        _fail(name, f"slots must be int32 or int64, not {slots.dtype}")
    if slots.shape[0] != tokens:
        _fail(name, f"slots must have one slot per token, {tokens}, not {slots.shape[0]}")
    for what, cache in (("k_cache", k_cache), ("v_cache", v_cache)):
        _tensor(name, what, cache, k.device, k.dtype, 4)
        if cache.shape[2:] != k.shape[1:] or cache.shape[:2] != k_cache.shape[:2] or cache.shape[1] < 1:
            _fail(name, f"{what} must be (pages, page_size, {kv_heads}, {dim}), not {tuple(cache.shape)}")
        _unit_last(name, what, cache)
        _writable(name, what, cache)
        _apart(name, what, cache, "k", k)
        _apart(name, what, cache, "v", v)
    _apart(name, "k_cache", k_cache, "v_cache", v_cache)
    flags_k = turned
    weight_k = weight_q = 0
    if k_weight is not None:
        flags_k |= native.ROWS_NORM | _weight(name, "k_weight", k_weight, k)
        weight_k = k_weight.data_ptr()
    rows = [_rows(k, k_cache, flags_k | native.ROWS_PAGED, weight_k), _rows(v, v_cache, native.ROWS_PAGED)]
    if q is None:
        if q_weight is not None or q_out is not None:
            _fail(name, "q_weight and q_out need q")
    else:
        _rows_shape(name, "q", q)
        if q.dim() != 3 or q.device != k.device or q.dtype is not k.dtype or q.shape[0] != tokens or q.shape[2] != dim:
            _fail(name, f"q must be ({tokens}, heads, {dim}) of k's device and dtype")
        _unit_last(name, "q", q)
        flags_q = turned
        if q_weight is not None:
            flags_q |= native.ROWS_NORM | _weight(name, "q_weight", q_weight, q)
            weight_q = q_weight.data_ptr()
        given = (("k", k), ("v", v), ("k_cache", k_cache), ("v_cache", v_cache))
        q_out = _result(name, "q_out", q_out, q, (("q", q),), given)
        _apart(name, "k_cache", k_cache, "q", q)
        _apart(name, "v_cache", v_cache, "q", q)
        rows.append(_rows(q, q_out, flags_q, weight_q))
    _run_rotary("tila_rotary_rows", k, rows, turn, layout, amplitude, eps=eps, slots=slots,
                num_slots=k_cache.shape[0] * k_cache.shape[1], page=k_cache.shape[1])
    return q_out


def norm_rotate_backward(q_grad, k_grad, q, k, q_weight, k_weight, positions, inv_freq, *, layout="half",
                         amplitude=1.0, eps=1e-6, dq=None, dk=None):
    """Gradients ``(dq, dk, dq_weight, dk_weight)`` of :func:`norm_rotate`,
    given those of its results and its inputs.

    ``dq`` and ``dk`` have q's dtype, the weights' gradients are float32 whatever the
    weights' dtype.  The same call gives the same bits: sums run in a fixed
    order.  ``dq`` may be ``q`` or ``q_grad`` itself, and ``dk`` likewise.
    """
    name = "norm_rotate_backward"
    wide_q, wide_k = _pair(name, q, k, q_weight, k_weight)
    turn = _positions(name, positions, inv_freq, q, layout)
    for what, g, like in (("q_grad", q_grad, q), ("k_grad", k_grad, k)):
        _tensor(name, what, g, q.device, q.dtype)
        if g.shape != like.shape:
            _fail(name, f"{what} must have the shape {tuple(like.shape)}, not {tuple(g.shape)}")
        _unit_last(name, what, g)
    of_q, of_k = (("q", q), ("q_grad", q_grad)), (("k", k), ("k_grad", k_grad))
    dq = _result(name, "dq", dq, q, of_q, of_k)
    dk = _result(name, "dk", dk, k, of_k, of_q + (("dq", dq),))
    sums = torch.empty(2, q.shape[-1], dtype=torch.float32, device=q.device)
    flags = native.ROWS_ROTATE | native.ROWS_NORM
    _run_rotary("tila_rotary_norm_backward", q, [_rows(q, dq, flags | wide_q, q_weight.data_ptr(), q_grad),
                                                 _rows(k, dk, flags | wide_k, k_weight.data_ptr(), k_grad)],
                turn, layout, amplitude, eps=eps, workspace=True,
                weight_grad=(sums.data_ptr(), sums.data_ptr() + 4 * q.shape[-1]))
    return dq, dk, sums[0], sums[1]


# ---------------------------------------------------------------------------
# attention over the paged cache
# ---------------------------------------------------------------------------

def _indexes(name, what, t, device, rank, length=None):
    _tensor(name, what, t, device, torch.int32, rank)
    if t.numel() > 1 and t.stride(-1) != 1:
        _fail(name, f"the last dimension of {what} must be contiguous")
    if length is not None and t.shape[0] != length:
        _fail(name, f"{what} must have {length} entries, not {t.shape[0]}")
    return t.data_ptr()


def attend_shared_prefix(q, k_cache, v_cache, page_table, lengths, *, prefix_pages=None, prefix_length=0,
                         query_offsets=None, max_queries=None, scale=None, out=None, return_lse=False):
    """Attention of new tokens over a paged cache: ``softmax(scale q K^T) V`` over
    a prefix that all sequences share and each sequence's own tokens.

    ``q``: (tokens, heads, dim), float16 or bfloat16, dim a multiple of 8 up to 256.
    ``k_cache``, ``v_cache``: (pages, page_size, kv_heads, dim) in any strides whose rows
    start on 16-byte boundaries; query heads share key heads in groups.
    ``page_table`` (batch, width) and ``lengths`` (batch,), int32: the pages of each
    sequence's own tokens and how many they are, the new ones included (append
    them first).  ``prefix_pages`` (int32) holds the first ``prefix_length`` tokens of
    every sequence; it is read once for the whole batch.

    Without ``query_offsets`` row b of ``q`` is the one new token of sequence b.  With
    it (int32, batch + 1 entries) rows ``query_offsets[b]`` to ``query_offsets[b + 1]`` are
    its new tokens, at most ``max_queries`` of them; each sees the tokens up to
    itself.  Rows of ``q`` behind the last sequence may be anything, and theirs of
    ``out`` are left as they were.  A token that sees nothing gets zeros.

    ``scale`` is 1/sqrt(dim) by default.  Returns ``out`` (q's dtype), and with
    ``return_lse`` also the log of each row's sum of exponentials, float32 (tokens,
    heads).  Scores, weights' sums and results are kept in 32 bits; the weights are
    rounded to the values' type for their product.  The same call gives the same
    bits.  Values that a new token may not see yet must still be finite, as a
    weight of 0 is multiplied with them; what lies behind a sequence's length,
    or in pages that it does not reach, may be anything.
    """
    name = "attend_shared_prefix"
    _tensor(name, "q", q, None, None, 3)
    if q.dtype is not torch.float16 and q.dtype is not torch.bfloat16:
        _fail(name, f"q must be float16 or bfloat16, not {q.dtype}")
    tokens, heads, dim = q.shape
    if dim % 8 or not 8 <= dim <= 256:
        _fail(name, f"dim must be a multiple of 8 up to 256, not {dim}")
    q_stride = _unit_last(name, "q", q)
    device = q.device
    strides = []
    for what, cache in (("k_cache", k_cache), ("v_cache", v_cache)):
        _tensor(name, what, cache, device, q.dtype, 4)
        if cache.shape != k_cache.shape or cache.shape[3] != dim or cache.shape[1] < 1:
            _fail(name, f"{what} must be (pages, page_size, kv_heads, {dim}), both alike, not {tuple(cache.shape)}")
        st = _unit_last(name, what, cache)
        if cache.data_ptr() % 16 or st[0] % 8 or st[1] % 8 or st[2] % 8:
            _fail(name, f"rows of {what} must start on 16-byte boundaries")
        strides += st[:3]
    pages, page_size, kv_heads, _ = k_cache.shape
    if kv_heads < 1 or heads < 1 or heads % kv_heads:
        _fail(name, f"heads ({heads}) must be a multiple of kv_heads ({kv_heads})")
    table = _indexes(name, "page_table", page_table, device, 2)
    batch, width = page_table.shape
    lens = _indexes(name, "lengths", lengths, device, 1, batch)
    if query_offsets is None:
        if tokens != batch:
            _fail(name, f"q must have one row per sequence, {batch}, not {tokens} (or query_offsets is needed)")
        if max_queries not in (None, 1):
            _fail(name, "max_queries needs query_offsets")
        offsets, most = 0, 1
    else:
        offsets = _indexes(name, "query_offsets", query_offsets, device, 1, batch + 1)
        most = max(1, tokens if max_queries is None else min(max_queries, tokens))
        if max_queries is not None and max_queries < 1:
            _fail(name, f"max_queries must be at least 1, not {max_queries}")
    shared = 0
    if prefix_length < 0:
        _fail(name, f"prefix_length must not be negative, is {prefix_length}")
    if prefix_length > 0:
        if prefix_pages is None:
            _fail(name, "prefix_length needs prefix_pages")
        shared = _indexes(name, "prefix_pages", prefix_pages, device, 1)
        if prefix_pages.shape[0] * page_size < prefix_length:
            _fail(name, f"prefix_pages holds {prefix_pages.shape[0] * page_size} tokens, fewer than {prefix_length}")
    out = _result(name, "out", out, q, (), (("q", q), ("k_cache", k_cache), ("v_cache", v_cache)))
    lse = torch.empty(tokens, heads, dtype=torch.float32, device=device) if return_lse else None
    o_stride = out.stride()
    index = device.index

    def go():
        args = [native.ATTEND.size, _DTYPES[q.dtype], tokens, batch, heads, kv_heads, dim, page_size, width, most,
                dim ** -0.5 if scale is None else float(scale), pages, prefix_length, q.data_ptr(),
                k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), 0 if lse is None else lse.data_ptr(),
                q_stride[0], q_stride[1], o_stride[0], o_stride[1], *strides, table,
                page_table.stride(0), lens, offsets, shared, _error_block(index),
                torch.cuda.current_stream(index).cuda_stream, 0, 0]
        need = native.attend_workspace(native.ATTEND.pack(*args))
        if need:
            space = torch.empty(need, dtype=torch.uint8, device=device)
            args[-2], args[-1] = space.data_ptr(), need
        native.call_op("tila_attend_shared_prefix", native.ATTEND.pack(*args))

    if torch.cuda.current_device() == index:
        go()
    else:
        with torch.cuda.device(index):
            go()
    return (out, lse) if return_lse else out
