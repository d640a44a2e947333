"""The operators of the decode path, as they are measured: rotary positions,
norms of queries and keys fused with the rotation, the append to a paged
key/value cache, and attention of a batch that shares a long prefix.

``run`` computes each in its plain form (elementary torch operations in 32
bits, angles in 64, rounded once at the end), or through ``tila_b200.ops``
where ``own`` is true.  ``exact`` states the same results in 64 bits.
"""

import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # one decode step of a small batch: queries alone, latency counts
        {"name": "rotate 8 tokens", "op": "rotate", "direction": "forward", "batch": 8, "tokens": 1, "heads": 32,
         "dim": 128, "rotary": 128, "layout": "half", "dtype": "bf16", "scaling": 1.0, "far": 100000},
        # two prompts of odd length whose heads rotate in their first half only
        {"name": "rotate prompts, part", "op": "rotate", "direction": "forward", "batch": 2, "tokens": 4099,
         "heads": 32, "dim": 128, "rotary": 64, "layout": "interleaved", "dtype": "f16", "scaling": 4.0, "far": 0},
        # the gradient in a training step (batch 4, 2048 tokens) in 32 bits
        {"name": "rotate gradient", "op": "rotate", "direction": "backward", "batch": 4, "tokens": 2048, "heads": 32,
         "dim": 128, "rotary": 128, "layout": "half", "dtype": "f32", "scaling": 1.0, "far": 0},
        # one decode step of 64 sequences: normed and rotated queries and keys
        {"name": "norm 64 tokens", "op": "norm", "direction": "forward", "tokens": 64, "heads": 32, "kv_heads": 8,
         "dim": 128, "rotary": 128, "layout": "half", "dtype": "bf16", "far": 100000},
        # a training batch of 8192 tokens, forward, read from one fused projection
        {"name": "norm 8192 tokens", "op": "norm", "direction": "forward", "tokens": 8192, "heads": 32,
         "kv_heads": 8, "dim": 128, "rotary": 128, "layout": "half", "dtype": "bf16", "far": 0},
        # its gradient: of queries, keys and both weights
        {"name": "norm gradient", "op": "norm", "direction": "backward", "tokens": 8192, "heads": 32, "kv_heads": 8,
         "dim": 128, "rotary": 128, "layout": "half", "dtype": "bf16", "far": 0},
        # one decode step of 64 sequences: one row each into its own page
        {"name": "append 64 tokens", "op": "append", "tokens": 64, "heads": 32, "kv_heads": 8, "dim": 128,
         "rotary": 128, "layout": "half", "page": 16, "run": 1, "padded": 0, "dtype": "bf16", "far": 100000},
        # prompts of 1021 tokens each, padded to a fixed batch, into pages of 64
        {"name": "append prompts", "op": "append", "tokens": 16384, "heads": 32, "kv_heads": 8, "dim": 128,
         "rotary": 64, "layout": "interleaved", "page": 64, "run": 1021, "padded": 48, "dtype": "f16", "far": 0},
        # four short chats on a system prompt: one token each
        {"name": "attend 4 chats", "op": "attend", "batch": 4, "queries": 1, "prefix": 1000, "own": 200, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "lens": 1, "dtype": "bf16"},
        # 64 sequences on a long shared document
        {"name": "attend 64 on 8192", "op": "attend", "batch": 64, "queries": 1, "prefix": 8192, "own": 1024,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "lens": 2, "dtype": "bf16"},
        # several new tokens for each sequence (chunks of prompts, drafted tokens), heads without groups
        {"name": "attend chunks", "op": "attend", "batch": 16, "queries": 128, "prefix": 4096, "own": 1000,
         "heads": 16, "kv_heads": 16, "dim": 64, "page": 32, "lens": 3, "dtype": "f16"},
        # the largest batch on the longest prefix
        {"name": "attend 128 on 32768", "op": "attend", "batch": 128, "queries": 1, "prefix": 32768, "own": 4096,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "lens": 4, "dtype": "bf16"},
    ]


# ---------------------------------------------------------------------------
# drawn cases
# ---------------------------------------------------------------------------

def _spread(rng, low, high):
    """A whole number, spread over the logarithm of its range."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def _within(case, field, most):
    """`case` with `field` halved until one pass moves at most `most` bytes."""
    while work(case)["bytes"] > most and case[field] > 1:
        case[field] //= 2
    return case


def draw(rng):
    op = rng.choice(["rotate", "norm", "append", "attend"])
    dim = rng.choice([64, 80, 96, 128])
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 2, 3, 4, 5, 7, 8])
    dtype = rng.choice(["bf16", "f16"] if op == "attend" else ["bf16", "f16", "f32"])
    part = rng.choice([1, 1, 2, 4])
    layout = rng.choice(["half", "interleaved"])
    far = rng.choice([0, rng.randrange(1, 1 << 20)])
    if op == "rotate":
        case = {"op": op, "direction": rng.choice(["forward", "backward"]), "batch": _spread(rng, 1, 16),
                "tokens": _spread(rng, 1, 8192), "heads": heads, "dim": dim, "rotary": dim // part, "layout": layout,
                "dtype": dtype, "scaling": rng.choice([1.0, 4.0, 8.0]), "far": far}
        return _within(case, "tokens", 250e6)
    if op == "norm":
        case = {"op": op, "direction": rng.choice(["forward", "backward"]), "tokens": _spread(rng, 1, 16384),
                "heads": heads, "kv_heads": kv, "dim": dim, "rotary": dim // part, "layout": layout, "dtype": dtype,
                "far": far}
        return _within(case, "tokens", 250e6)
    if op == "append":
        case = {"op": op, "tokens": _spread(rng, 1, 16384), "heads": heads, "kv_heads": kv, "dim": dim,
                "rotary": dim // part, "layout": layout, "page": rng.choice([16, 32, 64, 128]),
                "run": _spread(rng, 1, 2000), "padded": rng.choice([0, rng.randrange(0, 64)]), "dtype": dtype,
                "far": far}
        return _within(case, "tokens", 300e6)
    case = {"op": op, "batch": _spread(rng, 1, 128), "queries": rng.choice([1, 1, _spread(rng, 2, 128)]),
            "prefix": rng.choice([0, _spread(rng, 1, 32768), _spread(rng, 1000, 32768)]), "own": _spread(rng, 1, 4096),
            "heads": heads, "kv_heads": kv, "dim": dim, "page": rng.choice([16, 32, 64, 128]),
            "lens": rng.randrange(1, 1 << 20), "dtype": dtype}
    case["own"] = max(case["own"], case["queries"])
    # the scores of a chunk are what costs most here
    while work(case)["flops"] > 60e9 and case["batch"] > 1:
        case["batch"] //= 2
    while work(case)["flops"] > 60e9 and case["queries"] > 1:
        case["queries"] //= 2
    return case


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _frequencies(case):
    """Radians per position of each rotated pair, in 64 bits; long contexts
    are scaled by dividing them."""
    half = case["rotary"] // 2
    return torch.tensor([10000.0 ** (-i / half) / case.get("scaling", 1.0) for i in range(half)],
                        dtype=torch.float64, device="cuda")


def _lengths(case):
    """(own tokens in the cache, new tokens among them) of each sequence: part
    of the case, so that its work is known."""
    r = np.random.RandomState(case["lens"])
    new = r.randint(1, case["queries"] + 1, case["batch"]) if case["queries"] > 1 else np.ones(case["batch"], np.int64)
    new[0] = case["queries"]
    own_ = np.maximum(r.randint(1, case["own"] + 1, case["batch"]), new)
    own_[-1] = case["own"]
    return own_, new


def _positions(case, g, shape):
    n = shape[-1]
    start = torch.randint(0, max(1, case["far"]), shape[:-1] + (1,), generator=g, device="cuda")
    if n == 1 or case.get("run") == 1:
        return torch.randint(0, max(2, case["far"]), shape, generator=g, device="cuda")
    return (start + torch.arange(n, device="cuda")).contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)

    s = {"case": case}
    if case["op"] == "rotate":
        s["x"] = normal(case["batch"], case["tokens"], case["heads"], case["dim"])
        s["positions"] = _positions(case, g, (case["batch"], case["tokens"]))
        s["inv_freq"] = _frequencies(case)
    elif case["op"] == "norm":
        t, h, kv, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        qkv = normal(t, h + 2 * kv, d, scale=1.5)          # one fused projection: queries, keys, values
        s["q"], s["k"] = qkv[:, :h], qkv[:, h:h + kv]
        s["q_weight"] = (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(dtype)
        s["k_weight"] = (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(dtype)
        s["positions"] = _positions(case, g, (t,))
        s["inv_freq"] = _frequencies(case)
        if case["direction"] == "backward":
            s["q_grad"], s["k_grad"] = normal(t, h, d), normal(t, kv, d)
    elif case["op"] == "append":
        t, h, kv, d, page = case["tokens"], case["heads"], case["kv_heads"], case["dim"], case["page"]
        qkv = normal(t, h + 2 * kv, d)
        s["q"], s["k"], s["v"] = qkv[:, :h], qkv[:, h:h + kv], qkv[:, h + kv:]
        s["positions"] = _positions(case, g, (t,))
        s["inv_freq"] = _frequencies(case)
        # runs of tokens fill pages taken from the pool in any order
        run_ = min(case["run"], t)
        per = -(-run_ // page)
        runs = -(-t // run_)
        pool = runs * per + 3
        pages = torch.randperm(pool, generator=g, device="cuda")[:runs * per].view(runs, per)
        i = torch.arange(t, device="cuda")
        at = i % run_
        slots = pages[i // run_, at // page] * page + at % page
        s["kept"] = max(1, t - case["padded"])              # the rows behind are padding of the batch
        slots[s["kept"]:] = -1
        s["slots"] = slots
        s["k_cache"] = normal(pool, page, kv, d)
        s["v_cache"] = normal(pool, page, kv, d)
    else:
        b, kv, d, page, p = case["batch"], case["kv_heads"], case["dim"], case["page"], case["prefix"]
        lens, new = _lengths(case)
        wide = -(-case["own"] // page)
        shared = -(-p // page)
        need = -(-lens // page)
        pool = int(need.sum()) + shared + 2
        order = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
        starts = np.concatenate([[0], np.cumsum(need)[:-1]]) + shared
        at = np.minimum(starts[:, None] + np.arange(wide)[None], pool - 1)
        s["page_table"] = order[torch.from_numpy(at).cuda()].contiguous()
        s["prefix_pages"] = order[:shared].contiguous()
        s["lengths"] = torch.from_numpy(lens.astype(np.int32)).cuda()
        offsets = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        s["offsets"] = torch.from_numpy(offsets).cuda() if case["queries"] > 1 else None
        s["tokens"] = int(offsets[-1])
        # which sequence each new token is of, and its place there: a scheduler knows this
        s["of"] = torch.from_numpy(np.repeat(np.arange(b), new)).cuda()
        s["place"] = torch.from_numpy(np.concatenate([np.arange(n) for n in new])).cuda()
        s["new"] = torch.from_numpy(new.astype(np.int64)).cuda()
        s["q"] = normal(s["tokens"], case["heads"], d)
        s["k_cache"] = normal(pool, page, kv, d)
        s["v_cache"] = normal(pool, page, kv, d)
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------

def _turned(x, positions, inv_freq, layout, inverse=False):
    """The rotation of x (..., tokens, heads, dim; 32 bits)."""
    angle = positions.double().unsqueeze(-1) * inv_freq
    c, s = angle.cos().float().unsqueeze(-2), angle.sin().float().unsqueeze(-2)
    if inverse:
        s = -s
    half = inv_freq.numel()
    y = x.clone()
    if layout == "half":
        a, b = x[..., :half], x[..., half:2 * half]
        y[..., :half], y[..., half:2 * half] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        y[..., 0:2 * half:2], y[..., 1:2 * half:2] = a * c - b * s, b * c + a * s
    return y


EPS = 1e-6


def _normed(x, weight):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight


def _normed_gradient(g, x, weight):
    """Gradients of x and weight, where g is the gradient of _normed(x, weight)."""
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    xh = x * r
    gw = g * weight
    return r * (gw - xh * (gw * xh).mean(-1, keepdim=True)), (g * xh).sum(0).sum(0)


def _plain_rotate(s):
    x, back = s["x"], s["case"]["direction"] == "backward"
    return _turned(x.float(), s["positions"], s["inv_freq"], s["case"]["layout"], back).to(x.dtype)


def _plain_norm(s):
    pos, inv, layout = s["positions"], s["inv_freq"], s["case"]["layout"]
    q, k, qw, kw = s["q"], s["k"], s["q_weight"].float(), s["k_weight"].float()
    if s["case"]["direction"] == "forward":
        return [_turned(_normed(x.float(), w), pos, inv, layout).to(x.dtype) for x, w in ((q, qw), (k, kw))]
    gq = _turned(s["q_grad"].float(), pos, inv, layout, True)
    gk = _turned(s["k_grad"].float(), pos, inv, layout, True)
    dq, dqw = _normed_gradient(gq, q.float(), qw)
    dk, dkw = _normed_gradient(gk, k.float(), kw)
    return [dq.to(q.dtype), dk.to(k.dtype), dqw, dkw]


def _plain_append(s):
    pos, inv, layout = s["positions"], s["inv_freq"], s["case"]["layout"]
    q = _turned(s["q"].float(), pos, inv, layout).to(s["q"].dtype)
    k = _turned(s["k"].float(), pos, inv, layout).to(s["k"].dtype)
    kept = s["kept"]
    slots = s["slots"][:kept]
    s["k_cache"].flatten(0, 1)[slots] = k[:kept]
    s["v_cache"].flatten(0, 1)[slots] = s["v"][:kept]
    return [q, s["k_cache"], s["v_cache"]]


def _plain_attend(s):
    case = s["case"]
    b, kv, d, p, t = case["batch"], case["kv_heads"], case["dim"], case["prefix"], s["tokens"]
    g, most = case["heads"] // kv, case["queries"]
    q = s["q"].float().view(t, kv, g, d) * d ** -0.5
    # the shared prefix: every new token attends to all of it
    kp = s["k_cache"][s["prefix_pages"]].flatten(0, 1)[:p].float().permute(1, 2, 0)       # kv, d, p
    vp = s["v_cache"][s["prefix_pages"]].flatten(0, 1)[:p].float().permute(1, 0, 2)       # kv, p, d
    shared = q.permute(1, 0, 2, 3).reshape(kv, t * g, d) @ kp
    # each sequence's own tokens, causal among the new ones
    ko = s["k_cache"][s["page_table"]].flatten(1, 2).float().permute(0, 2, 3, 1)          # b, kv, d, n
    vo = s["v_cache"][s["page_table"]].flatten(1, 2).float().permute(0, 2, 1, 3)
    n = ko.shape[-1]
    padded = q.new_zeros(b, most, kv, g, d)
    padded[s["of"], s["place"]] = q
    own_ = (padded.permute(0, 2, 1, 3, 4).reshape(b, kv, most * g, d) @ ko).view(b, kv, most, g, n)
    last = (s["lengths"].long() - s["new"])[:, None] + torch.arange(most, device="cuda")   # b, most
    hidden = torch.arange(n, device="cuda") > last[:, :, None]
    own_ = own_.masked_fill(hidden[:, None, :, None, :], -math.inf)
    top_own = own_.amax(-1)                                                               # b, kv, most, g
    top_shared = shared.amax(-1).view(kv, t, g) if p else None
    rows = lambda x: x.permute(0, 2, 1, 3)[s["of"], s["place"]]                           # noqa: E731  t, kv, g
    top = rows(top_own)
    if p:
        top = torch.maximum(top, top_shared.permute(1, 0, 2))
    spread = top.new_zeros(b, most, kv, g)
    spread[s["of"], s["place"]] = top
    e = (own_ - spread.permute(0, 2, 1, 3)[..., None]).exp()
    total = rows(e.sum(-1))
    out = (e.view(b, kv, most * g, n) @ vo).view(b, kv, most, g, d).permute(0, 2, 1, 3, 4)[s["of"], s["place"]]
    if p:
        e = (shared - top.permute(1, 0, 2).reshape(kv, t * g, 1)).exp()
        total = total + e.sum(-1).view(kv, t, g).permute(1, 0, 2)
        out = out + (e @ vp).view(kv, t, g, d).permute(1, 0, 2, 3)
    out = (out / total[..., None]).view(t, kv * g, d).to(s["q"].dtype)
    return [out, (top + total.log()).view(t, kv * g)]


PLAIN = {"rotate": _plain_rotate, "norm": _plain_norm, "append": _plain_append, "attend": _plain_attend}


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------

def _own(s):
    from tila_b200 import ops
    case = s["case"]
    if case["op"] == "rotate":
        call = ops.rotate if case["direction"] == "forward" else ops.rotate_backward
        return call(s["x"], s["positions"], s["inv_freq"], layout=case["layout"])
    if case["op"] == "norm":
        args = (s["q"], s["k"], s["q_weight"], s["k_weight"], s["positions"], s["inv_freq"])
        if case["direction"] == "forward":
            return list(ops.norm_rotate(*args, layout=case["layout"], eps=EPS))
        return list(ops.norm_rotate_backward(s["q_grad"], s["k_grad"], *args, layout=case["layout"], eps=EPS))
    if case["op"] == "append":
        q = ops.append_paged(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"], positions=s["positions"],
                             inv_freq=s["inv_freq"], layout=case["layout"], q=s["q"])
        return [q, s["k_cache"], s["v_cache"]]
    return list(ops.attend_shared_prefix(s["q"], s["k_cache"], s["v_cache"], s["page_table"], s["lengths"],
                                         prefix_pages=s["prefix_pages"], prefix_length=case["prefix"],
                                         query_offsets=s["offsets"], max_queries=case["queries"], return_lse=True))


def run(state):
    if own:
        return _own(state)
    return PLAIN[state["case"]["op"]](state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    d = case["dim"]
    if case["op"] == "rotate":
        n = case["batch"] * case["tokens"]
        e = n * case["heads"] * d
        return {"bytes": 2 * e * size + 8 * n + 4 * case["rotary"], "flops": 3 * n * case["heads"] * case["rotary"]}
    if case["op"] == "norm":
        n = case["tokens"]
        e = n * (case["heads"] + case["kv_heads"]) * d
        if case["direction"] == "forward":
            return {"bytes": 2 * e * size + 2 * d * size + 8 * n, "flops": 7 * e}
        return {"bytes": 3 * e * size + 2 * d * (size + 4) + 8 * n, "flops": 14 * e}
    if case["op"] == "append":
        n = case["tokens"]
        kept = max(1, n - case["padded"])
        e = n * case["heads"] * d + 2 * kept * case["kv_heads"] * d
        return {"bytes": 2 * e * size + 16 * n, "flops": 3 * n * (case["heads"] + case["kv_heads"]) * case["rotary"]}
    lens, new = _lengths(case)
    t, kv, p = int(new.sum()), case["kv_heads"], case["prefix"]
    seen = int((new * lens - new * (new - 1) // 2).sum())
    cache = 2 * (p + int(lens.sum())) * kv * d * size
    pages = 4 * (-(-p // case["page"]) + int((-(-lens // case["page"])).sum()))
    rows = t * case["heads"]
    return {"bytes": cache + pages + 2 * rows * d * size + 4 * rows,
            "flops": 4 * case["heads"] * d * (t * p + seen)}


# ---------------------------------------------------------------------------
# the same results in 64 bits, from the definitions
# ---------------------------------------------------------------------------

def _exact_turn(x, s, sign=1.0):
    """Each pair as one complex number, times exp(i * angle)."""
    half = s["inv_freq"].numel()
    z = torch.polar(torch.ones_like(s["inv_freq"]), torch.zeros_like(s["inv_freq"]))
    angle = sign * torch.outer(s["positions"].reshape(-1).double(), s["inv_freq"])
    z = torch.polar(torch.ones_like(angle), angle).view(*s["positions"].shape, 1, half)
    head, rest = x[..., :2 * half], x[..., 2 * half:]
    if s["case"]["layout"] == "half":
        y = torch.complex(head[..., :half].contiguous(), head[..., half:].contiguous()) * z
        return torch.cat([y.real, y.imag, rest], -1)
    pairs = head.unflatten(-1, (half, 2))
    y = torch.complex(pairs[..., 0].contiguous(), pairs[..., 1].contiguous()) * z
    return torch.cat([torch.stack([y.real, y.imag], -1).flatten(-2), rest], -1)


def _exact_norm(x, w):
    return w * x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt()


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotate":
        return _exact_turn(s["x"].double(), s, 1.0 if case["direction"] == "forward" else -1.0)
    if case["op"] == "norm":
        leaves = [s[n].double().requires_grad_() for n in ("q", "k", "q_weight", "k_weight")]
        q, k, qw, kw = leaves
        out = [_exact_turn(_exact_norm(q, qw), s), _exact_turn(_exact_norm(k, kw), s)]
        if case["direction"] == "forward":
            return [x.detach() for x in out]
        return list(torch.autograd.grad(out, leaves, [s["q_grad"].double(), s["k_grad"].double()]))
    if case["op"] == "append":
        q, k, v = (s[n].double() for n in ("q", "k", "v"))
        q, k = _exact_turn(q, s), _exact_turn(k, s)
        page = case["page"]
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        kept = (s["slots"] >= 0).nonzero()[:, 0]
        at = s["slots"][kept]
        kc[at // page, at % page] = k[kept]
        vc[at // page, at % page] = v[kept]
        return [q, kc, vc]
    lens, new = _lengths(case)
    kv, d, p, page = case["kv_heads"], case["dim"], case["prefix"], case["page"]
    g = case["heads"] // kv
    shared = s["prefix_pages"].long()
    out, lse, at = [], [], 0
    for b in range(case["batch"]):
        n, m = int(lens[b]), int(new[b])
        mine = s["page_table"][b].long()[:-(-n // page)]
        k, v = (torch.cat([c[shared].reshape(-1, kv, d)[:p], c[mine].reshape(-1, kv, d)[:n]]).double()
                for c in (s["k_cache"], s["v_cache"]))
        q = s["q"][at:at + m].double().view(m, kv, g, d)
        at += m
        w = torch.einsum("mkgd,nkd->kgmn", q, k) / math.sqrt(d)
        allowed = torch.ones(m, p + n, dtype=torch.bool, device="cuda").tril(p + n - m)
        w = w.masked_fill(~allowed, -math.inf)
        lse.append(torch.logsumexp(w, -1).permute(2, 0, 1).reshape(m, kv * g))
        out.append(torch.einsum("kgmn,nkd->mkgd", torch.softmax(w, -1), v).reshape(m, kv * g, d))
    return [torch.cat(out), torch.cat(lse)]
