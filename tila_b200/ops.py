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
They are not recorded by autograd: a gradient is a call of its own, and with
gradients enabled a tensor that requires one is refused (``torch.no_grad()``, or a
``torch.autograd.Function`` around the call and its gradient's).  Every call
can be captured into a CUDA graph once an operator has run on the device.
Wrong arguments raise ``ValueError`` before anything is launched.  What only the
device can see is kept from any access outside the caches, recorded as a device
error, and raised by the next operator on that device or by :func:`check_errors`:
a row whose slot is outside the cache is left out; a page outside it reads as zeros
(its keys score 0 and take their weight in the softmax); lengths and offsets are cut
to the table and to ``q``.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import native

try:
    from . import _ops
except ImportError as exc:
    raise ImportError("tila_b200._ops is not built; run __graft_entry__.build() or `python -m tila_b200.build`") from exc

# ---------------------------------------------------------------------------
# device errors
# ---------------------------------------------------------------------------

ERROR_CODES = {
    1: "a bounded wait timed out; the operator stopped early and its outputs are incomplete",
    2: "tensor memory allocation failed",
    5: "an index outside its pool: a cache slot (its row was left out), a page (read as zeros), a length or an offset "
       "(cut to the table or to q)",
}


class _ErrorBlock:
    """The error block that every operator on a device is given, and the
    page-locked word that the kernels copy its first error to."""

    def __init__(self, index):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the first operator on a device cannot be captured into a CUDA graph: "
                               "call it once before the capture")
        # (in inference mode it would be a tensor that check_errors could not reset outside of it)
        with torch.inference_mode(False), torch.cuda.device(index):
            self.block = torch.zeros(native.ERROR_BLOCK_BYTES // 4, dtype=torch.int32, device="cuda")
            host, address = native.host_word_alloc()
            self.block.view(torch.int64)[1] = address
            torch.cuda.current_stream().synchronize()   # operators on other streams read it
        self.word = ctypes.c_uint32.from_address(host)
        _ops.set_error_block(index, self.block.data_ptr(), host)


_error_blocks = {}


def _prepare(index):
    """The error block of a device that no operator has run on yet."""
    if index not in _error_blocks:
        _error_blocks[index] = _ErrorBlock(index)


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
        if not torch.cuda.is_current_stream_capturing():    # (a graph would record the reset: the next call raises again)
            b.block[0].zero_()
            b.word.value = 0
    code, where = word >> 24, word & 0xFFFFFF
    raise native.NativeError(native.TILA_ERR_ARGUMENT if code == 5 else native.TILA_ERR_DRIVER,
                             f"an operator launched earlier on cuda:{index} failed: "
                             f"{ERROR_CODES.get(code, f'device error code {code}')} (at {where})")


_ops.setup(_prepare, check_errors, native.NativeError)


def _fail(name, text):
    raise ValueError(f"{name}: {text}")


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
    if not (0 < base < math.inf and 1.0 <= factor < math.inf):
        _fail(name, "base must be positive and factor at least 1, both finite")
    if scaling not in (None, "linear", "ntk", "yarn"):
        _fail(name, f"scaling must be None, 'linear', 'ntk' or 'yarn', not {scaling!r}")
    try:
        if scaling == "ntk" and rotary > 2:
            base = base * factor ** (rotary / (rotary - 2))
            if base == math.inf:
                raise OverflowError
        freq = [base ** (-2.0 * i / rotary) for i in range(rotary // 2)]
    except OverflowError:
        _fail(name, f"base {base} and factor {factor} give frequencies beyond 64-bit numbers")
    amplitude = 1.0
    if scaling == "linear":
        freq = [f / factor for f in freq]
    elif scaling == "yarn":
        if base <= 1:
            _fail(name, f"'yarn' needs frequencies that fall from pair to pair: a base above 1, not {base}")
        if not original_length or not 1 <= original_length < math.inf:
            _fail(name, "'yarn' needs original_length, the length that the model was trained on")
        if not math.inf > beta_fast > beta_slow > 0:
            _fail(name, "beta_fast must be above beta_slow, both positive and finite")

        def pair(turns):     # the pair (not whole) that turns so often over original_length
            return rotary * math.log(original_length / (turns * 2 * math.pi)) / (2 * math.log(base))

        low = max(math.floor(pair(beta_fast)), 0)
        high = min(math.ceil(pair(beta_slow)), rotary - 1)
        high = high + 0.001 if high == low else high
        ramp = [min(1.0, max(0.0, (i - low) / (high - low))) for i in range(rotary // 2)]
        freq = [f * (1 - r) + f / factor * r for f, r in zip(freq, ramp)]
        amplitude = 0.1 * math.log(factor) + 1.0
    return torch.tensor(freq, dtype=torch.float64, device="cuda" if device is None else device), amplitude


def rotate(x, positions, inv_freq, *, layout="half", amplitude=1.0, out=None):
    """Rotary positions: each pair of ``x`` (tokens, heads, dim) or (batch,
    tokens, heads, dim) turned by ``position * inv_freq``.

    The first ``2 * len(inv_freq)`` elements of a head rotate, the others are
    copied.  ``layout``: pairs ``(i, i + rotary/2)`` (``"half"``) or ``(2i, 2i + 1)``
    (``"interleaved"``).  ``positions``: int32 or int64, one per token, or (tokens,) for
    every batch entry.  ``amplitude`` multiplies the rotated elements.  ``out`` may
    be ``x`` itself.  float32, float16, bfloat16.
    """
    return _ops.rotate(x, positions, inv_freq, layout, amplitude, out, False)


def rotate_backward(grad, positions, inv_freq, *, layout="half", amplitude=1.0, out=None):
    """Gradient of :func:`rotate` with respect to ``x``, given that of its
    result: the rotation back, with the same amplitude."""
    return _ops.rotate(grad, positions, inv_freq, layout, amplitude, out, True)


def norm_rotate(q, k, q_weight, k_weight, positions, inv_freq, *, layout="half", amplitude=1.0, eps=1e-6,
                q_out=None, k_out=None):
    """``(q_out, k_out)``: each head of ``q`` and ``k`` divided by its root mean
    square, times the weight, and rotated, in one pass.

    ``q`` (.., tokens, heads, dim) and ``k`` (.., tokens, kv_heads, dim) may be
    parts of one projection; the weights (dim,) are float32 or of q's dtype.
    The results may be ``q`` and ``k`` themselves.  The other arguments are those
    of :func:`rotate`.
    """
    return _ops.norm_rotate(q, k, q_weight, k_weight, positions, inv_freq, layout, amplitude, eps, q_out, k_out)


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
    return _ops.append_paged(k, v, k_cache, v_cache, slots, positions, inv_freq, layout, amplitude, k_weight, q, q_weight,
                             q_out, eps)


def norm_rotate_backward(q_grad, k_grad, q, k, q_weight, k_weight, positions, inv_freq, *, layout="half",
                         amplitude=1.0, eps=1e-6, dq=None, dk=None):
    """Gradients ``(dq, dk, dq_weight, dk_weight)`` of :func:`norm_rotate`,
    given those of its results and its inputs.

    ``dq`` and ``dk`` have q's dtype, the weights' gradients are float32 whatever the
    weights' dtype.  The same call gives the same bits: sums run in a fixed
    order.  ``dq`` may be ``q`` or ``q_grad`` itself, and ``dk`` likewise.
    """
    return _ops.norm_rotate_backward(q_grad, k_grad, q, k, q_weight, k_weight, positions, inv_freq, layout, amplitude,
                                     eps, dq, dk)


# ---------------------------------------------------------------------------
# attention over the paged cache
# ---------------------------------------------------------------------------

def attend_shared_prefix(q, k_cache, v_cache, page_table, lengths, *, prefix_pages=None, prefix_length=0,
                         query_offsets=None, max_queries=None, max_length=None, scale=None, out=None,
                         return_lse=False):
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
    itself.  By default ``max_queries`` is the number of rows of ``q``: right, but every
    sequence is given blocks for so many (64 sequences of 128 of them 1219 us instead
    of 303), so pass it where the host knows it.  Rows of ``q`` behind the last sequence may be anything, and theirs of
    ``out`` are left as they were.  A token that sees nothing, or whose scores are all
    minus infinity, gets zeros (and -inf for its log).

    ``max_length``, the longest of ``lengths`` where the host knows it, only steers how
    the work is split (by default the table's width, which may be far more).
    ``scale`` is 1/sqrt(dim) by default.  Returns ``out`` (q's dtype), and with
    ``return_lse`` also the log of each row's sum of exponentials, float32 (tokens,
    heads).  Scores, weights' sums and results are kept in 32 bits; the weights are
    rounded to the values' type for their product.  The same call gives the same
    bits.  What a token does not see may be anything, infinities and NaN included:
    new tokens behind it, cache rows behind a sequence's length, pages that no
    sequence reaches.
    """
    return _ops.attend_shared_prefix(q, k_cache, v_cache, page_table, lengths, prefix_pages, prefix_length, query_offsets,
                                     max_queries, scale, out, bool(return_lse), max_length)
