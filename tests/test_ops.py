"""The operators' host side on the CPU: frequencies, and the calls they refuse
(nothing is launched: every refusal comes before that)."""

import ctypes
import math
import re
import shutil
import struct
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from tila_b200 import native, ops


def dev(*shape, dtype=torch.float32):
    """What stands for a CUDA tensor: that it is none is the last check."""
    return torch.zeros(*shape, dtype=dtype)


def test_frequencies():
    inv, amplitude = ops.rotary_frequencies(8, base=100.0, device="cpu")
    assert inv.dtype is torch.float64 and amplitude == 1.0
    assert inv.tolist() == [100.0 ** (-i / 4) for i in range(4)]
    linear, _ = ops.rotary_frequencies(8, base=100.0, scaling="linear", factor=4.0, device="cpu")
    assert torch.equal(linear, inv / 4)
    ntk, _ = ops.rotary_frequencies(64, scaling="ntk", factor=8.0, device="cpu")
    plain, _ = ops.rotary_frequencies(64, device="cpu")
    assert ntk[0] == plain[0] and abs(ntk[-1].item() * 8 / plain[-1].item() - 1) < 1e-12
    yarn, amplitude = ops.rotary_frequencies(64, scaling="yarn", factor=8.0, original_length=4096, device="cpu")
    turns = plain * 4096 / (2 * math.pi)
    assert torch.equal(yarn[turns > 40], plain[turns > 40])           # beyond the ramp's rounding outwards
    assert torch.allclose(yarn[turns < 0.7], plain[turns < 0.7] / 8, rtol=1e-15)
    assert bool((yarn <= plain).all()) and bool((yarn >= plain / 8 * (1 - 1e-15)).all())
    assert amplitude == 0.1 * math.log(8.0) + 1.0
    assert ops.rotary_frequencies(0, device="cpu")[0].numel() == 0
    assert ops.rotary_frequencies(2, scaling="ntk", factor=2.0, device="cpu")[0].tolist() == [1.0]


@pytest.mark.parametrize("kwargs", [dict(rotary=7), dict(rotary=-2), dict(rotary=8, base=0.0), dict(rotary=8, factor=0.5),
                                    dict(rotary=8, scaling="other"), dict(rotary=8, scaling="yarn"),
                                    dict(rotary=8, scaling="yarn", original_length=100, beta_fast=1.0, beta_slow=2.0)])
def test_frequencies_refuse(kwargs):
    with pytest.raises(ValueError):
        ops.rotary_frequencies(device="cpu", **kwargs)


INV = torch.ones(32, dtype=torch.float64)
POS = torch.arange(6)


@pytest.mark.parametrize("change,text", [
    (dict(), "x must be a CUDA|grad must be a CUDA"),
    (dict(x=dev(6, 2, 64, dtype=torch.float64)), "float32"),
    (dict(x=dev(6, 64)), "tokens, heads, dim"),
    (dict(x=dev(6, 2, 513)), "512"),
    (dict(x=dev(6, 1, 64).expand(6, (1 << 20) + 1, 64)), "2\\^20 heads"),
    (dict(x=dev(6, 2, 128)[..., ::2]), "contiguous"),
    (dict(x=dev(6, 2, 62)), "rotates 64"),
    (dict(positions=POS[:5]), "one position per token"),
    (dict(positions=POS.float()), "int32 or int64"),
    (dict(positions=torch.zeros(6, dtype=torch.int64, device="meta")), "other tensors on cpu"),
    (dict(inv_freq=INV.float()), "Double"),
    (dict(inv_freq=dev(64, dtype=torch.float64)[::2]), "contiguous"),
    (dict(layout="other"), "layout"),
    (dict(out=dev(6, 2, 32)), "shape"),
    (dict(out=dev(6, 2, 64, dtype=torch.float16)), "Float, not Half"),
    (dict(out=dev(6, 1, 64).expand(6, 2, 64)), "share memory"),
    (dict(out=dev(6, 2, 128)[..., ::2]), "contiguous"),
])
def test_rotate_refuses(change, text):
    args = dict(x=dev(6, 2, 64), positions=POS, inv_freq=INV) | change
    x, positions, inv = args.pop("x"), args.pop("positions"), args.pop("inv_freq")
    with pytest.raises(ValueError, match=text):
        ops.rotate(x, positions, inv, **args)
    with pytest.raises(ValueError, match=text):
        ops.rotate_backward(x, positions, inv, **args)


def test_not_a_tensor():
    with pytest.raises(TypeError):
        ops.rotate([1.0], POS, INV)


def test_rotate_refuses_a_result_across_its_source():
    flat = dev(6 * 2 * 64 + 64)
    with pytest.raises(ValueError, match="overlaps"):
        ops.rotate(flat[:768].view(6, 2, 64), POS, INV, out=flat[64:].view(6, 2, 64))


def test_overlap_rules():
    """Parts of one tensor lie between each other's rows; anything else that
    shares memory is refused."""
    qkv = dev(6, 5, 64)
    q, k = qkv[:, :3], qkv[:, 3:]
    def apart(a, b, same=False):
        ops._ops.check_apart("t", "a", a, "b", b, same)
    apart(q, k)
    apart(k, q)
    apart(q, q, same=True)
    both = dev(4, 2, 8, 3, 64)
    apart(both[:, 0], both[:, 1])
    batch = dev(2, 6, 5, 64)
    apart(batch[:, :, :3], batch[:, :, 3:])
    for a, b in ((q, q), (qkv[:, :3], qkv[:, 2:]), (q, qkv[:, :2]), (both[:, 0], both[:, 0]), (qkv, q)):
        with pytest.raises(ValueError, match="overlaps"):
            apart(a, b)


NORM = dict(q=dev(6, 4, 64), k=dev(6, 2, 64), q_weight=dev(64), k_weight=dev(64))


@pytest.mark.parametrize("change,text", [
    (dict(), "q must be a CUDA"),
    (dict(k=dev(5, 2, 64)), "same tokens"),
    (dict(k=dev(6, 2, 32)), "same tokens"),
    (dict(k=dev(6, 2, 64, dtype=torch.float16)), "one dtype"),
    (dict(q_weight=dev(32)), "64 elements"),
    (dict(k_weight=dev(64, dtype=torch.bfloat16)), "float32"),
    (dict(q_weight=dev(128)[::2]), "contiguous"),
    (dict(k=NORM["q"], k_out=NORM["q"]), "overlaps"),
    (dict(q_out=dev(6, 4, 32)), "shape"),
])
def test_norm_rotate_refuses(change, text):
    args = NORM | change
    first = [args.pop(n) for n in ("q", "k", "q_weight", "k_weight")]
    with pytest.raises(ValueError, match=text):
        ops.norm_rotate(*first, POS, INV, **args)


def test_norm_rotate_backward_refuses():
    a = list(NORM.values())
    for grads, kwargs, text in (((dev(6, 4, 32), dev(6, 2, 64)), {}, "shape"),
                                ((dev(6, 4, 64), dev(6, 2, 64, dtype=torch.float16)), {}, "Float, not Half"),
                                ((dev(6, 4, 64), dev(6, 2, 64)), dict(dk=NORM["q"][:, :2]), "overlaps")):
        with pytest.raises(ValueError, match=text):
            ops.norm_rotate_backward(*grads, *a, POS, INV, **kwargs)


APPEND = dict(k=dev(6, 2, 64), v=dev(6, 2, 64), k_cache=dev(3, 4, 2, 64), v_cache=dev(3, 4, 2, 64),
              slots=torch.arange(6))


@pytest.mark.parametrize("change,text", [
    (dict(), "k must be a CUDA"),
    (dict(k=dev(1, 6, 2, 64)), "tokens, kv_heads"),
    (dict(v=dev(6, 2, 32)), "shape of k"),
    (dict(v=dev(6, 2, 64, dtype=torch.float16)), "Float, not Half"),
    (dict(k_cache=dev(3, 4, 1, 64)), "k_cache must be"),
    (dict(v_cache=dev(3, 5, 2, 64)), "v_cache must be"),
    (dict(v_cache=dev(12, 2, 64)), "4 dimensions"),
    (dict(v_cache=APPEND["k_cache"]), "overlaps"),
    (dict(k_cache=dev(1, 4, 2, 64).expand(3, 4, 2, 64)), "share memory"),
    (dict(slots=POS[:4]), "one slot per token"),
    (dict(slots=POS.float()), "int32 or int64"),
    (dict(positions=POS), "go together"),
    (dict(q_out=dev(6, 4, 64)), "need q"),
    (dict(q=dev(5, 4, 64)), "q must be"),
    (dict(q=dev(6, 4, 64), q_weight=dev(5)), "64 elements"),
    (dict(k_weight=dev(64, dtype=torch.float16)), "float32"),
    (dict(q=dev(6, 2, 64), q_out=APPEND["k"]), "overlaps"),
])
def test_append_refuses(change, text):
    args = APPEND | change
    first = [args.pop(n) for n in ("k", "v", "k_cache", "v_cache", "slots")]
    with pytest.raises(ValueError, match=text):
        ops.append_paged(*first, **args)


# tila_op_rows, tila_rotary_args without its rows, tila_attend_args (include/tila_b200.h)
ROWS, HEAD, ATTEND_ARGS = struct.Struct("=4Q9qiI"), struct.Struct("=Iiqq4iffQ2qQQqq4i6Q"), struct.Struct("=Iiq8ifi2q5Q4q6qQq7Q")
ROTARY_BYTES = HEAD.size + 3 * ROWS.size
FLAG_ROTATE, FLAG_NORM, FLAG_PAGED = 1, 2, 4


def refused(entry, args):
    """The C entry's status is that of a bad argument, and the log says why."""
    log = ctypes.create_string_buffer(512)
    status = getattr(native.library(), entry)(args, log, ctypes.c_size_t(len(log)))
    assert status == native.TILA_ERR_ARGUMENT and log.value


def workspace(entry, args):
    f = getattr(native.library(), entry)
    f.restype = ctypes.c_uint64
    return f(args)


def rotary_args(rows=1, flags=FLAG_ROTATE, token_stride=128, **change):
    """tila_rotary_args with addresses that nothing reads (the call is refused)."""
    names = ("size", "dtype", "batch", "tokens", "dim", "rotary", "interleaved", "inverse", "amplitude", "eps",
             "positions", "step_b", "step_t", "inv_freq", "slots", "slot_step", "num_slots", "page", "index64",
             "num_rows", "reserved", "err", "stream", "workspace", "workspace_bytes", "dw0", "dw1")
    head = dict(zip(names, (ROTARY_BYTES, 0, 1, 4, 64, 64, 0, 0, 1.0, 0.0, 4096, 0, 1, 4096, 0, 0, 0, 0, 1, rows, 0,
                            0, 0, 0, 0, 0, 0))) | change
    row = ROWS.pack(4096, 4096, 0, 0, 0, token_stride, 64, 0, 128, 64, 0, 0, 0, 2, flags)
    return HEAD.pack(*(head[n] for n in names)) + row * rows + bytes(ROWS.size) * (3 - rows)


@pytest.mark.parametrize("entry,args", [
    ("tila_rotary_rows", rotary_args(size=8)),
    ("tila_rotary_rows", rotary_args(reserved=1)),
    ("tila_rotary_rows", rotary_args(dtype=3)),
    ("tila_rotary_rows", rotary_args(dim=513)),
    ("tila_rotary_rows", rotary_args(rotary=66)),
    ("tila_rotary_rows", rotary_args(rotary=63)),
    ("tila_rotary_rows", rotary_args(positions=0)),
    ("tila_rotary_rows", rotary_args(num_rows=4)),
    ("tila_rotary_rows", rotary_args(token_stride=1 << 32)),
    ("tila_rotary_rows", rotary_args(flags=FLAG_NORM)),
    ("tila_rotary_rows", rotary_args(flags=FLAG_PAGED)),
    ("tila_rotary_norm_backward", rotary_args()),
])
def test_c_entry_refuses(entry, args):
    refused(entry, args)
    assert workspace("tila_rotary_workspace", args) == 0


def ints(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


H = torch.float16
ATTEND = dict(q=dev(3, 4, 64, dtype=H), k_cache=dev(5, 8, 2, 64, dtype=H), v_cache=dev(5, 8, 2, 64, dtype=H),
              page_table=ints(3, 2), lengths=ints(3))


@pytest.mark.parametrize("change,text", [
    (dict(), "q must be a CUDA"),
    (dict(q=dev(3, 4, 64)), "float16 or bfloat16"),
    (dict(q=dev(3, 4, 60, dtype=H)), "multiple of 8"),
    (dict(q=dev(3, 4, 264, dtype=H)), "up to 256"),
    (dict(q=dev(3, 64, dtype=H)), "3 dimensions"),
    (dict(q=dev(3, 5, 64, dtype=H)), "multiple of kv_heads"),
    (dict(q=dev(4, 4, 64, dtype=H)), "one row per sequence"),
    (dict(k_cache=dev(5, 8, 2, 32, dtype=H)), "both alike"),
    (dict(v_cache=dev(5, 9, 2, 64, dtype=H)), "both alike"),
    (dict(v_cache=dev(5, 8, 2, 64, dtype=torch.bfloat16)), "Half"),
    (dict(k_cache=dev(5, 8, 2, 68, dtype=H)[..., 4:]), "16-byte"),
    (dict(page_table=ints(3, 2).long()), "Int, not Long"),
    (dict(page_table=ints(3)), "2 dimensions"),
    (dict(page_table=ints(3, 4)[:, ::2]), "contiguous"),
    (dict(lengths=ints(2)), "3 entries"),
    (dict(lengths=ints(3, 1)), "1 dimensions"),
    (dict(query_offsets=ints(3)), "4 entries"),
    (dict(query_offsets=ints(4), max_queries=0), "at least 1"),
    (dict(max_queries=2), "needs query_offsets"),
    (dict(max_length=0), "at least 1"),
    (dict(prefix_length=-1), "negative"),
    (dict(prefix_length=5), "needs prefix_pages"),
    (dict(prefix_length=17, prefix_pages=ints(2)), "fewer than 17"),
    (dict(out=dev(3, 4, 32, dtype=H)), "shape"),
    (dict(out=ATTEND["q"]), "overlaps"),
    (dict(out=ATTEND["k_cache"].view(-1)[:768].view(3, 4, 64)), "overlaps"),
])
def test_attend_refuses(change, text):
    args = ATTEND | change
    first = [args.pop(n) for n in ("q", "k_cache", "v_cache", "page_table", "lengths")]
    with pytest.raises(ValueError, match=text):
        ops.attend_shared_prefix(*first, **args)


def attend_args(**change):
    """tila_attend_args with addresses that nothing reads (the call is refused)."""
    names = ("size", "dtype", "tokens", "batch", "heads", "kv_heads", "dim", "page_size", "table_width", "max_queries",
             "max_length", "scale", "reserved", "num_pages", "prefix_length", "q", "k_cache", "v_cache", "out", "lse", "qt", "qh", "ot", "oh",
             "kp", "kr", "kh", "vp", "vr", "vh", "page_table", "table_stride", "lengths", "query_offsets",
             "prefix_pages", "err", "stream", "workspace", "workspace_bytes")
    v = dict(zip(names, (ATTEND_ARGS.size, 1, 4, 4, 8, 2, 64, 16, 10, 1, 0, 0.125, 0, 100, 300, 4096, 4096, 4096, 4096, 0,
                         512, 64, 512, 64, 2048, 128, 64, 2048, 128, 64, 4096, 10, 4096, 0, 4096, 0, 0, 0, 0))) | change
    return ATTEND_ARGS.pack(*(v[n] for n in names))


@pytest.mark.parametrize("change", [
    dict(size=8), dict(reserved=1), dict(max_length=-1), dict(dtype=0), dict(dtype=3), dict(heads=3), dict(kv_heads=0), dict(dim=12), dict(dim=264), dict(page_size=0),
    dict(max_queries=0), dict(tokens=3), dict(prefix_length=-1), dict(prefix_length=1 << 31), dict(q=0), dict(q=4097),
    dict(k_cache=4104), dict(vr=4), dict(lengths=0), dict(page_table=0), dict(prefix_pages=0), dict(lse=2),
    dict(workspace=4096, workspace_bytes=16), dict(workspace=4097, workspace_bytes=1 << 40),
])
def test_c_attend_refuses(change):
    refused("tila_attend_shared_prefix", attend_args(**change))


def test_c_attend_workspace():
    """One partial result (dim + 1 floats) for every row and chunk; none where one
    block does it all; none for a call of no rows."""
    assert workspace("tila_attend_workspace", attend_args()) % (4 * 8 * 65 * 4) == 0
    assert workspace("tila_attend_workspace", attend_args()) > 0
    assert workspace("tila_attend_workspace", attend_args(prefix_length=0, table_width=1)) == 0
    assert workspace("tila_attend_workspace", attend_args(tokens=0, batch=0)) == 0
    assert native.library().tila_attend_shared_prefix(attend_args(tokens=0, batch=0), None, ctypes.c_size_t(0)) == native.TILA_OK


def rotary_rows(flags, weight=4096, grad=0, heads=2):
    """One tensor of tila_rotary_args, as rotary_args makes it."""
    return ROWS.pack(4096, 4096, weight, grad, 0, 128, 64, 0, 128, 64, 0, 128, 64, heads, flags)


FLAG_WEIGHT_F32 = 8


@pytest.mark.parametrize("entry,change,row", [
    ("tila_rotary_rows", dict(positions=4100), rotary_rows(FLAG_ROTATE)),                            # 64-bit positions
    ("tila_rotary_rows", dict(positions=4098, index64=0), rotary_rows(FLAG_ROTATE)),
    ("tila_rotary_rows", dict(inv_freq=4100), rotary_rows(FLAG_ROTATE)),
    ("tila_rotary_rows", dict(err=4100), rotary_rows(FLAG_ROTATE)),
    ("tila_rotary_rows", dict(dtype=1), rotary_rows(FLAG_NORM, weight=4097)),
    ("tila_rotary_rows", dict(dtype=1), rotary_rows(FLAG_NORM | FLAG_WEIGHT_F32, weight=4098)),
    ("tila_rotary_rows", dict(slots=4100, num_slots=8, page=4, index64=2), rotary_rows(FLAG_PAGED)),
    ("tila_rotary_rows", dict(slots=4098, num_slots=8, page=4, index64=0), rotary_rows(FLAG_PAGED)),
    ("tila_rotary_norm_backward", dict(dw0=4098, workspace=4096, workspace_bytes=1 << 20),
     rotary_rows(FLAG_NORM | FLAG_WEIGHT_F32, grad=4096)),
])
def test_c_entry_refuses_unaligned_addresses(entry, change, row):
    refused(entry, rotary_args(rows=1, **change)[:HEAD.size] + row + bytes(2 * ROWS.size))


@pytest.mark.parametrize("change", [dict(lengths=4098), dict(page_table=4097), dict(prefix_pages=4098),
                                    dict(query_offsets=4098, max_queries=4), dict(err=4100)])
def test_c_attend_refuses_unaligned_addresses(change):
    # (a workspace that is large enough, so that only the address is at fault)
    refused("tila_attend_shared_prefix", attend_args(workspace=4096, workspace_bytes=1 << 40, **change))


def test_c_entries_refuse_sizes_whose_product_passes_64_bits():
    for batch in (1, 4):
        refused("tila_rotary_rows", rotary_args(batch=batch, tokens=1 << 62))
        args = rotary_args(batch=batch, tokens=1 << 62, dw0=4096)[:HEAD.size] + rotary_rows(FLAG_NORM, grad=4096) + bytes(2 * ROWS.size)
        refused("tila_rotary_norm_backward", args)
        assert workspace("tila_rotary_workspace", args) == 0
    refused("tila_attend_shared_prefix", attend_args(tokens=1 << 61, workspace=4096, workspace_bytes=1 << 60))
    assert workspace("tila_attend_workspace", attend_args(tokens=1 << 61)) == 0


def attend_slots(tokens, batch, heads, kv, dim, page, prefix, own, queries):
    """Partial results of each row that a call's workspace holds."""
    space = workspace("tila_attend_workspace", attend_args(
        tokens=tokens, batch=batch, heads=heads, kv_heads=kv, dim=dim, page_size=page, table_width=-(-own // page),
        prefix_length=prefix, max_queries=queries, query_offsets=0 if queries == 1 else 4096, kp=page * kv * dim,
        kr=kv * dim, kh=dim, vp=page * kv * dim, vr=kv * dim, vh=dim, num_pages=1 << 20))
    slots, rest = divmod(space, tokens * heads * (dim + 1) * 4)
    assert rest == 0
    return slots


@pytest.mark.parametrize("page", [1, 4, 24, 48, 96, 64])
@pytest.mark.parametrize("tokens,batch,heads,kv,dim,prefix,own,queries,most", [
    (64 * 128, 64, 32, 8, 128, 32768, 1024, 128, 2),       # chunks of prompts: 270 MB a slot
    (8192, 1, 32, 8, 128, 131072, 8192, 8192, 2),          # one prompt on a long document
    (2048, 16, 32, 8, 256, 32768, 512, 128, 4),
    (128, 128, 32, 8, 256, 32768, 4096, 1, 24),            # a decode step: 17 MB a slot, and a prefix of 134 MB
])
def test_attend_workspace_is_bounded_for_any_page_size(page, tokens, batch, heads, kv, dim, prefix, own, queries, most):
    """Where many rows are taken by the narrow form (these page sizes and heads of 256
    elements), chunks are not cut finer than the blocks need."""
    assert 1 <= attend_slots(tokens, batch, heads, kv, dim, page, prefix, own, queries) <= most


def test_attend_few_rows_keep_their_chunks():
    """One token each of few sequences: 74 chunks of a prefix fill the GPU, and
    none of a longer one passes 512 keys."""
    assert attend_slots(4, 4, 32, 8, 256, 16, 32768, 64, 1) == 74 + 1
    assert attend_slots(4, 4, 32, 32, 256, 16, 32768, 64, 1) == 64 + 1


def test_a_copy_of_the_package_uses_its_own_library(tmp_path):
    package = Path(ops.__file__).parent
    copy = tmp_path / "tila_b200"
    copy.mkdir()
    for f in [*package.glob("*.py"), *package.glob("*.so")]:
        shutil.copy(f, copy)
    code = ("import sys; sys.path.insert(0, sys.argv[1]); from tila_b200 import ops\n"
            "print({l.split()[-1] for l in open('/proc/self/maps') if 'libtila_b200.so' in l})")
    got = subprocess.run([sys.executable, "-c", code, str(tmp_path)], check=True, capture_output=True, text=True,
                         cwd=tmp_path).stdout
    assert got.strip() == str({str(copy / "libtila_b200.so")})


def test_what_autograd_would_have_to_record_is_refused():
    """With gradients enabled; without them (under no_grad, in a Function's forward)
    the call goes on to the next check, which here is that there is no GPU."""
    offsets = dict(query_offsets=ints(4), max_queries=2)
    calls = [
        (lambda x, inv: ops.rotate(x, POS, inv), [dev(6, 2, 64), INV.clone()]),
        (lambda x, out: ops.rotate(x, POS, INV, out=out), [dev(6, 2, 64), dev(6, 2, 64)]),
        (lambda x: ops.rotate_backward(x, POS, INV), [dev(6, 2, 64)]),
        (lambda *t: ops.norm_rotate(*t, POS, INV), [t.clone() for t in NORM.values()]),
        (lambda *t: ops.norm_rotate_backward(*t, POS, INV), [dev(6, 4, 64), dev(6, 2, 64), *(t.clone() for t in NORM.values())]),
        (lambda k, v, kc, vc, kw, q, qw: ops.append_paged(k, v, kc, vc, torch.arange(6), k_weight=kw, q=q, q_weight=qw),
         [dev(6, 2, 64), dev(6, 2, 64), dev(3, 4, 2, 64), dev(3, 4, 2, 64), dev(64), dev(6, 4, 64), dev(64)]),
        (lambda q, k, v: ops.attend_shared_prefix(q, k, v, ints(3, 2), ints(3), **offsets),
         [ATTEND[n].clone() for n in ("q", "k_cache", "v_cache")]),
    ]
    for call, tensors in calls:
        for t in tensors:
            t.requires_grad_()
            with pytest.raises(ValueError, match="requires a gradient"):
                call(*tensors)
            with torch.no_grad(), pytest.raises(ValueError, match="must be a CUDA"):
                call(*tensors)
            t.requires_grad_(False)


def apart_rows(*size, stride):
    """A tensor of that size whose rows lie far apart (nothing is allocated)."""
    return torch.empty_strided(size, stride, device="meta")


def test_sizes_and_strides_beyond_the_kernels_are_refused():
    """As wrong arguments, before anything is allocated."""
    far = 1 << 32
    x, near = apart_rows(6, 2, 64, stride=(1 << 34, far, 1)), apart_rows(6, 2, 64, stride=(128, 64, 1))
    pos, inv = torch.empty(6, dtype=torch.int64, device="meta"), torch.empty(32, dtype=torch.float64, device="meta")
    w, text = torch.empty(64, device="meta"), "below 2\\^32 elements"
    with pytest.raises(ValueError, match=f"x's.*{text}"):
        ops.rotate(x, pos, inv)
    with pytest.raises(ValueError, match=f"k's.*{text}"):
        ops.norm_rotate(near, x, w, w, pos, inv)
    with pytest.raises(ValueError, match=f"q_grad's.*{text}"):
        ops.norm_rotate_backward(x, near, near, near, w, w, pos, inv)
    # (empty ones, which do not overlap)
    x, near, pos = x[:0], near[:0], pos[:0]
    with pytest.raises(ValueError, match=f"out's.*{text}"):
        ops.rotate(near, pos, inv, out=x)
    cache = apart_rows(0, 4, 2, 64, stride=(512, 128, 64, 1))
    with pytest.raises(ValueError, match=f"v's.*{text}"):
        ops.append_paged(near, x, cache, cache, pos)
    with pytest.raises(ValueError, match=f"v_cache's.*{text}"):
        ops.append_paged(near, near, cache, apart_rows(0, 4, 2, 64, stride=(1 << 40, far, 64, 1)), pos)
    with pytest.raises(ValueError, match=f"q's.*{text}"):
        ops.append_paged(near, near, cache, cache, pos, q=x)

    q, k = dev(1, 1, 64, dtype=H), dev(1, 1, 1, 64, dtype=H)
    many = lambda rows, heads: q.expand(rows, heads, 64)                                  # noqa: E731
    offsets = dict(query_offsets=ints(4), max_queries=1 << 21)
    pages = k.expand(5, 1 << 20, 1, 64)
    for args, kwargs in (((many(1 << 21, 1 << 10), *[k.expand(5, 8, 1, 64)] * 2, ints(3, 2), ints(3)), offsets),
                         ((many(3, 1), pages, pages, ints(3, 1025), ints(3)), {}),
                         ((many(3, 1), pages, pages, ints(3, 1), ints(3)),
                          dict(prefix_pages=ints(1025), prefix_length=(1 << 30) + 1))):
        with pytest.raises(ValueError, match="more than 2\\^30"):
            ops.attend_shared_prefix(*args, **kwargs)


@pytest.mark.parametrize("kwargs", [
    dict(base=1.0, scaling="yarn", original_length=100), dict(base=0.5, scaling="yarn", original_length=100),
    dict(scaling="yarn", original_length=math.inf), dict(scaling="yarn", original_length=math.nan),
    dict(scaling="yarn", original_length=100, beta_fast=math.inf), dict(base=math.inf), dict(base=math.nan),
    dict(scaling="linear", factor=math.inf), dict(scaling="yarn", factor=math.inf, original_length=100),
    dict(scaling="ntk", factor=1e300), dict(scaling="ntk", factor=1e298, base=1e10), dict(base=1e-320),
])
def test_frequencies_that_do_not_exist_are_refused(kwargs):
    with pytest.raises(ValueError, match="rotary_frequencies"):
        ops.rotary_frequencies(64, device="cpu", **kwargs)
    assert ops.rotary_frequencies(64, base=1.0, device="cpu")[0].tolist() == [1.0] * 32


def test_views_that_negate_are_refused():
    """The imaginary part of a conjugate holds its values with the opposite sign."""
    lazy = torch.zeros(6, 2, 1, dtype=torch.complex64).conj().imag
    assert lazy.is_neg()
    none = torch.ones(0, dtype=torch.float64)
    for call in (lambda: ops.rotate(lazy, POS, none), lambda: ops.rotate(dev(6, 2, 1), POS, none, out=lazy),
                 lambda: ops.norm_rotate(lazy, dev(6, 2, 1), dev(1), dev(1), POS, none)):
        with pytest.raises(ValueError, match="negates"):
            call()
    with pytest.raises(ValueError, match="must be a CUDA"):
        ops.rotate(lazy.resolve_neg(), POS, none)


@pytest.mark.parametrize("scale", [math.nan, math.inf, -math.inf, 1e300, 3e38])
def test_attend_refuses_a_scale_that_is_no_number(scale):
    args = [ATTEND[n] for n in ("q", "k_cache", "v_cache", "page_table", "lengths")]
    with pytest.raises(ValueError, match="scale must be finite"):
        ops.attend_shared_prefix(*args, scale=scale)
    scale = math.copysign(min(abs(scale), 3.4e38), scale)             # in 32 bits
    refused("tila_attend_shared_prefix", attend_args(scale=scale, workspace=4096, workspace_bytes=1 << 40))


def test_wide_attention_kernels_have_the_registers_they_share_out(tmp_path):
    """Their warpgroups would otherwise wait for registers that do not exist (the
    library then takes the narrow form): a compiler that gives them others shows here."""
    from tila_b200 import build
    source = build.PKG / "csrc" / "ops" / "attend_wide.cu"
    text = source.read_text()
    two, one = map(int, re.search(r"kLaunchRegisters = G == 2 \? (\d+) : (\d+);", text).groups())
    r = subprocess.run([str(build.CUDA / "bin" / "nvcc"), "-std=c++17", "-O2", "-gencode", "arch=compute_100a,code=sm_100a",
                        "-lineinfo", "-diag-suppress", "550", "-Xptxas", "-v", "-cubin", "-o", str(tmp_path / "x.cubin"),
                        str(source)], check=True, capture_output=True, text=True)
    used = re.findall(r"entry function '\S*attend_wide_kernelI\S*Lb([01])E\S*'.*?Used (\d+) registers", r.stdout + r.stderr, re.S)
    assert sorted(used) == sorted([("0", str(two)), ("1", str(one))] * 4)
