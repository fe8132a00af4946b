"""What the operators of a key/value cache held in 4 bits are measured on.

A cache in 4 bits: every 32 channels of a key or value that one head has at one position are a block with one scale, a power of
two; a number is one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign (bits: sign, two of exponent, one of fraction) times the scale.

    e     = exponent of the block's largest magnitude, less 2, and one more where that magnitude is over 1.75 times a power of two
            (it would be 7 or more in units of 2^(e), and rounds to 8 rather than to 6), within -119 .. 125
    code  = x / 2^e to the nearest of the sixteen numbers, ties to the even code, 6 at most
    byte  = e + 127; 255 where the block holds a NaN or an infinity: all of it reads as NaN

In pages of ``page`` positions: a key's codes ``[pages, heads, page, D / 2]`` (channel 2 j in byte j's low half), a value's
``[pages, heads, page / 8, D / 2, 8]`` (the same bytes of 8 positions side by side), the scales of either
``[pages, heads, page / 8, blocks, 8]``.

Kinds of case:

======  =========================================================================================================================
store   rotate a step's queries and keys, write keys and values to their pages, read the written rows back: ``requests`` of
        ``tokens`` new tokens each behind ``context`` cached ones
read    the pages of ``requests`` that have up to ``context`` tokens, as pages of ``dtype``
attend  causal attention of ``requests`` with up to ``context`` cached tokens each (the last ``tokens`` of them are the step's own),
        with a window or a sink a head where the case says so
======  =========================================================================================================================

``draw`` gives more cases of the same ranges.  Requests of a case have between half and all of ``context`` tokens; their pages are
scattered over a pool.  Heads and sizes are those of this repository's benchmark and tests.
"""
from __future__ import annotations

import math
import random

import torch

own = False

BLOCK = 32
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)
THETA = 500000.0
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
# (query heads, key/value heads, channels of a head)
HEADS = {"8b": (32, 8, 128), "70b": (64, 8, 128), "1b": (32, 8, 64), "7b": (32, 32, 128), "wide": (16, 1, 256), "small": (8, 4, 32)}


def _case(name, kind, heads, requests, tokens, context, page=64, window=0, sink=False, dtype="bfloat16"):
    return {"name": name, "kind": kind, "heads": heads, "requests": requests, "tokens": tokens, "context": context, "page": page,
            "window": window, "sink": sink, "dtype": dtype}


def listed():
    return [
        # a lone user's decoded token on the 8B shape: launches and dependent reads
        _case("store-1", "store", "8b", 1, 1, 2000),
        # a full batch's decoded tokens, heads of 64
        _case("store-64x1", "store", "1b", 64, 1, 900),
        # a whole portion of a prompt, as the scheduler cuts it
        _case("store-2048", "store", "8b", 1, 2048, 2048),
        # a short request's pages, its last one begun
        _case("read-333", "read", "8b", 1, 1, 333),
        # the pages behind a portion of a long prompt, in true 32 bits and in the engine's type
        _case("read-5000-f32", "read", "1b", 3, 1, 5000, dtype="float32"),
        _case("read-32768", "read", "8b", 1, 1, 32768),
        # decoded tokens: one user, a full batch of long requests, a head for every query, one very long request
        _case("attend-1x2000", "attend", "8b", 1, 1, 2000),
        _case("attend-64x8000", "attend", "8b", 64, 1, 8000),
        _case("attend-23x900-mha", "attend", "7b", 23, 1, 900),
        _case("attend-1x131072", "attend", "70b", 1, 1, 131072),
        # a window and a sink over heads of 64, three tokens a request
        _case("attend-32x3-window", "attend", "1b", 32, 3, 3000, window=1024, sink=True),
        # a portion of a prompt behind what earlier portions left
        _case("attend-2048-after-6144", "attend", "8b", 1, 2048, 8192),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["store", "read", "attend", "attend", "attend"])
    heads = rng.choice(list(HEADS))
    page = rng.choice([32, 64, 64, 128])
    H, Hk, D = HEADS[heads]
    if kind == "store":
        tokens = rng.choice([1, 1, _spread(rng, 2, 2048)])
        requests = _spread(rng, 1, 64 if tokens == 1 else max(1, 2048 // tokens))
        context = tokens + _spread(rng, 1, 4000)
        dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
        return {k: v for k, v in _case("", kind, heads, requests, tokens, context, page, dtype=dtype).items() if k != "name"}
    if kind == "read":
        requests = _spread(rng, 1, 16)
        context = _spread(rng, 17, min(32768, (1 << 25) // (requests * Hk * D)))
        dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
        return {k: v for k, v in _case("", kind, heads, requests, 1, context, page, dtype=dtype).items() if k != "name"}
    tokens = rng.choice([1, 1, 1, _spread(rng, 2, 16), _spread(rng, 17, 1024)])
    requests = _spread(rng, 1, max(1, min(64, 2048 // tokens)))
    # no more cached numbers, and no more of a key's products with rows, than the largest listed cases have
    most = min(131072, (1 << 29) // (requests * Hk * D), (1 << 36) // (requests * tokens * H * D))
    context = tokens + _spread(rng, 1, max(2, most))
    window = rng.choice([0, 0, _spread(rng, 1, 4096)])
    dtype = rng.choice(["bfloat16"] * 5 + ["float32"]) if context * requests <= 20000 and tokens <= 64 else "bfloat16"
    return {k: v for k, v in _case("", kind, heads, requests, tokens, context, page, window, rng.random() < 0.25, dtype).items() if k != "name"}


# ------------------------------------------------------------------------------------------------ the inputs
def _lengths(case):
    """Cached tokens of each request once the step has run: the first has all, the others half at least (a case's own, whatever its
    inputs: what comes back has one shape)."""
    n, top = case["requests"], case["context"]
    low = max(case["tokens"], (top + 1) // 2)
    some = random.Random(top * 8191 + n)
    return [top] + [some.randint(low, top) for _ in range(n - 1)]


def _channels(Hk, D, gen, dev):
    """What makes some channels of a head larger than others: a deviation and an offset a channel."""
    dev_ = torch.exp(0.5 * torch.randn((Hk, D), generator=gen, device=dev))
    return dev_, torch.randn((Hk, D), generator=gen, device=dev) * 0.5


def _fill(codes, scales, values, Hk, D, page, gen, dev):
    """A pool's pages, each with keys or values as a layer would have left them there."""
    spread, offset = _channels(Hk, D, gen, dev)
    step = max(1, (1 << 26) // (Hk * page * D))
    for p in range(0, codes.shape[0], step):
        n = min(step, codes.shape[0] - p)
        x = torch.randn((n, Hk, page, D), generator=gen, device=dev) * spread[:, None] + offset[:, None]
        c, s = _quantise(x)
        codes[p:p + n] = c.view(n, Hk, page // 8, 8, D // 2).transpose(3, 4) if values else c
        scales[p:p + n] = s.view(n, Hk, page // 8, 8, D // BLOCK).transpose(3, 4)


def prepare(case, seed):
    dev = torch.device("cuda")
    H, Hk, D = HEADS[case["heads"]]
    page, B, n, dtype = case["page"], case["requests"], case["tokens"], DTYPES[case["dtype"]]
    host = torch.Generator().manual_seed(seed)
    gen = torch.Generator(device=dev).manual_seed(seed)
    lens = _lengths(case)
    counts = [-(-x // page) for x in lens]
    pool = sum(counts) + 3                                      # the null page, and some that are nobody's
    order = (torch.randperm(pool - 1, generator=host) + 1).tolist()
    table = torch.full((B, max(counts)), -1, dtype=torch.int32)
    tables, at = [], 0
    for b, c in enumerate(counts):
        tables.append(order[at:at + c])
        table[b, :c] = torch.tensor(order[at:at + c], dtype=torch.int32)
        at += c
    state = {"case": case, "lens": lens, "tables": tables, "table": table.to(dev), "dtype": dtype}
    for name, values in (("k", False), ("v", True)):
        codes = torch.empty((pool, Hk, page // 8, D // 2, 8) if values else (pool, Hk, page, D // 2), dtype=torch.uint8, device=dev)
        scales = torch.empty((pool, Hk, page // 8, D // BLOCK, 8), dtype=torch.uint8, device=dev)
        _fill(codes, scales, values, Hk, D, page, gen, dev)
        state[name + "_codes"], state[name + "_scales"] = codes, scales
    pos = torch.cat([torch.arange(x - n, x, dtype=torch.int32) for x in lens])
    state["positions"] = pos.to(dev)
    state["req"] = torch.arange(B, dtype=torch.int32).repeat_interleave(n).to(dev)
    state["starts"] = (torch.tensor(lens) - n).to(dev)
    T = B * n
    if case["kind"] == "store":
        # the input projection's 32-bit rows: queries, keys and values of a layer
        qs, qo = _channels(H, D, gen, dev)
        ks, ko = _channels(Hk, D, gen, dev)
        proj = torch.randn((T, (H + 2 * Hk), D), generator=gen, device=dev)
        proj[:, :H] = proj[:, :H] * qs + qo
        proj[:, H:H + Hk] = proj[:, H:H + Hk] * ks + ko
        state["proj"] = proj.view(T, -1)
        state["inv_freq"] = (1.0 / THETA ** (torch.arange(0, D, 2, dtype=torch.float64) / D)).float().to(dev)
    elif case["kind"] == "attend":
        state["q"] = (1.5 * torch.randn((T, H * D), generator=gen, device=dev)).to(dtype)
        state["sinks"] = torch.randn((H,), generator=gen, device=dev) if case["sink"] else None
    return state


# ------------------------------------------------------------------------------------------------ plain forms
def _quantise(x):
    """(codes two to a byte, a byte of scale a block) of the last axis."""
    blocks = x.unflatten(-1, (-1, BLOCK))
    bits = blocks.abs().amax(-1).view(torch.int32)
    byte = (((bits + 0x1FFFFF) >> 23) - 2).clamp(8, 252)
    byte = torch.where(bits >= 0x7F800000, 255, byte)
    finite = torch.where((byte == 255)[..., None], 0.0, blocks)
    y = torch.ldexp(finite, (127 - byte.clamp(max=252))[..., None])
    a = y.abs()
    # borders between neighbouring numbers; a tie goes to the even code
    code = ((a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int() + (a > 2.5).int() + (a >= 3.5).int()
            + (a > 5.0).int())
    code = (code + 8 * torch.signbit(y).int()).flatten(-2).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), byte.to(torch.uint8)


def _values(codes, scales):
    """32-bit numbers of ``codes [..., D / 2]`` and ``scales [..., blocks]``."""
    level = torch.tensor(LEVELS, dtype=torch.float32, device=codes.device)
    both = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2)
    x = level[both.int()].unflatten(-1, (-1, BLOCK))
    x = torch.ldexp(x, scales.int()[..., None] - 127)
    return torch.where((scales == 255)[..., None], float("nan"), x).flatten(-2)


def _rows_of(state, name, pages, offs):
    """Numbers of the positions ``offs`` of ``pages``: ``[..., heads, D]``."""
    codes, scales = state[name + "_codes"], state[name + "_scales"]
    if name == "k":
        c = codes[pages, :, offs]
    else:
        c = codes[pages, :, offs // 8, :, offs % 8]
    return _values(c, scales[pages, :, offs // 8, :, offs % 8])


def _rotated(x, positions, inv_freq):
    angle = positions.double()[:, None] * inv_freq.double()
    c, s = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    a, b = x.chunk(2, dim=-1)
    return torch.cat([a * c - b * s, a * s + b * c], dim=-1)


def _plain_store(state):
    case = state["case"]
    H, Hk, D = HEADS[case["heads"]]
    page = case["page"]
    x = state["proj"].unflatten(1, (-1, D))
    pos = state["positions"].long()
    q = _rotated(x[:, :H], pos, state["inv_freq"])
    k = _rotated(x[:, H:H + Hk], pos, state["inv_freq"])
    pages, offs = state["table"][state["req"].long(), pos // page].long(), pos % page
    kc, ks = _quantise(k)
    vc, vs = _quantise(x[:, H + Hk:])
    state["k_codes"][pages, :, offs] = kc
    state["k_scales"][pages, :, offs // 8, :, offs % 8] = ks
    state["v_codes"][pages, :, offs // 8, :, offs % 8] = vc
    state["v_scales"][pages, :, offs // 8, :, offs % 8] = vs
    return {"q": q.flatten(1).to(state["dtype"]), "k": _rows_of(state, "k", pages, offs).flatten(1).to(torch.bfloat16),
            "v": _rows_of(state, "v", pages, offs).flatten(1).to(torch.bfloat16)}


def _plain_read(state):
    case, dtype = state["case"], state["dtype"]
    H, Hk, D = HEADS[case["heads"]]
    page = case["page"]
    lens = torch.tensor(state["lens"], device=state["table"].device)
    held = state["table"] >= 0
    pages = state["table"][held].long()
    left = (lens[:, None] - page * torch.arange(held.shape[1], device=lens.device))[held]      # positions of each that are the request's
    there = torch.arange(page, device=lens.device) < left[:, None]
    k = _values(state["k_codes"][pages], state["k_scales"][pages].transpose(3, 4).flatten(2, 3))
    v = _values(state["v_codes"][pages].transpose(3, 4).flatten(2, 3), state["v_scales"][pages].transpose(3, 4).flatten(2, 3))
    k, v = (torch.where(there[:, None, :, None], x, 0.0) for x in (k, v))
    number = torch.where(held, held.flatten().cumsum(0).view(held.shape) - 1, -1).int()
    return {"k": k.to(dtype), "v": v.transpose(2, 3).contiguous().to(dtype), "table": number}


def _plain_attend(state):
    case = state["case"]
    H, Hk, D = HEADS[case["heads"]]
    page, B, n = case["page"], case["requests"], case["tokens"]
    dev = state["table"].device
    L = max(state["lens"])
    keys = torch.arange(L, device=dev)
    pages = state["table"][:, keys // page].long().clamp(min=0)                # [B, L]
    offs = (keys % page).expand(B, L)
    k = _rows_of(state, "k", pages, offs).permute(0, 2, 3, 1).contiguous()    # [B, Hk, D, L]
    v = _rows_of(state, "v", pages, offs).permute(0, 2, 1, 3).contiguous()    # [B, Hk, L, D]
    q = state["q"].float().view(B, n, Hk, H // Hk, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, -1, D)
    s = torch.matmul(q, k).view(B, Hk, H // Hk, n, L) * D ** -0.5
    at = state["starts"][:, None] + torch.arange(n, device=dev)                # [B, n]
    seen = keys <= at[..., None]
    if case["window"]:
        seen = seen & (keys > at[..., None] - case["window"])
    s = torch.where(seen[:, None, None], s, float("-inf"))
    top = s.amax(-1, keepdim=True)
    if state["sinks"] is not None:
        sink = state["sinks"].view(1, Hk, H // Hk, 1, 1)
        top = torch.maximum(top, sink)
    p = torch.exp(s - top)
    whole = p.sum(-1, keepdim=True)
    if state["sinks"] is not None:
        whole = whole + torch.exp(sink - top)
    o = torch.matmul((p / whole).view(B, Hk, -1, L), v).view(B, Hk, H // Hk, n, D)
    return o.permute(0, 3, 1, 2, 4).reshape(B * n, H * D).to(state["dtype"])


# ------------------------------------------------------------------------------------------------ the framework's calls
def _step(state):
    """What a program keeps for a step and all its layers: the kernels, the cache as the framework holds it, the step's context."""
    if "step" not in state:
        from xyntetik_runner_amd.cache.manager import RequestCache
        from xyntetik_runner_amd.csrc.ops import FourBitPages, load_ops
        from xyntetik_runner_amd.engine.batch import StepContext, StepEntry
        case = state["case"]
        D = HEADS[case["heads"]][2]
        ops = load_ops()
        n = case["tokens"]
        entries = [StepEntry(b, [0] * n) for b in range(case["requests"])]
        held = [RequestCache(b, b, x - n, [t], False) for b, (x, t) in enumerate(zip(state["lens"], state["tables"]))]
        ctx = StepContext(ops, state["table"].device, entries, held, 1)
        state["step"] = (ops, FourBitPages(state["k_codes"], state["k_scales"], D), FourBitPages(state["v_codes"], state["v_scales"], D), ctx)
    return state["step"]


def _own_store(state):
    ops, k_pages, v_pages, _ = _step(state)
    H, Hk, D = HEADS[state["case"]["heads"]]
    proj = state["proj"]
    q = torch.empty((proj.shape[0], H * D), dtype=state["dtype"], device=proj.device)
    ops.rope_kv_write(proj[:, :H * D], proj[:, H * D:(H + Hk) * D], proj[:, (H + Hk) * D:], q, k_pages, v_pages, state["positions"],
                      state["req"], state["table"], state["inv_freq"], H, Hk, D, D, False, 1.0, state["case"]["page"])
    k, v = ops.read_rows(k_pages, v_pages, state["positions"], state["req"], state["table"], torch.bfloat16)
    return {"q": q, "k": k, "v": v}


def _own_read(state):
    ops, k_pages, v_pages, ctx = _step(state)
    k, v, table = ops.read_pages(k_pages, v_pages, ctx, 0, state["dtype"])
    return {"k": k, "v": v, "table": table}


def _own_attend(state):
    ops, k_pages, v_pages, ctx = _step(state)
    case = state["case"]
    H, Hk, D = HEADS[case["heads"]]
    return ops.attention(state["q"], k_pages, v_pages, ctx, 0, H, Hk, D, case["page"], D ** -0.5, window=case["window"] or None,
                         sinks=state["sinks"])


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"store": _own_store, "read": _own_read, "attend": _own_attend}[kind](state)
    return {"store": _plain_store, "read": _plain_read, "attend": _plain_attend}[kind](state)


# ------------------------------------------------------------------------------------------------ floors and the definition in 64 bits
def work(case):
    H, Hk, D = HEADS[case["heads"]]
    T, size = case["requests"] * case["tokens"], 2 if case["dtype"] == "bfloat16" else 4
    token = 2 * Hk * (D // 2 + D // BLOCK)              # a token's codes and scales, keys and values
    lens = _lengths(case)
    if case["kind"] == "store":
        return {"bytes": T * ((H + 2 * Hk) * D * 4 + H * D * size + token + 2 * Hk * D * 2), "flops": T * (6 * (H + Hk) * D + 8 * Hk * D)}
    if case["kind"] == "read":
        return {"bytes": sum(lens) * (token + 2 * Hk * D * size), "flops": sum(lens) * 2 * Hk * D}
    n, window = case["tokens"], case["window"] or case["context"]
    reach = sum(min(x, window + n - 1) for x in lens)                                   # keys that some row of their request sees
    seen = sum(min(p + 1, window) for x in lens for p in range(x - n, x))               # pairs of a row's position and a key it sees
    return {"bytes": reach * token + 2 * T * H * D * size, "flops": 4 * H * D * seen}


def _exact_numbers(codes, scales):
    """64-bit numbers from a code's fields: sign, exponent, fraction."""
    c = torch.stack([codes % 16, codes // 16], dim=-1).flatten(-2).long()
    sign = 1.0 - 2.0 * (c // 8).double()
    expo, frac = (c % 8) // 2, (c % 2).double()
    mag = torch.where(expo == 0, frac * 0.5, (1.0 + 0.5 * frac) * 2.0 ** (expo.double() - 1.0))
    byte = scales.repeat_interleave(BLOCK, dim=-1).double()
    return torch.where(byte == 255, math.nan, sign * mag * 2.0 ** (byte - 127.0))


def _exact_request(state, b, upto):
    """Keys and values ``[heads, upto, D]`` of request ``b``."""
    page = state["case"]["page"]
    ids = torch.tensor(state["tables"][b], device=state["table"].device)
    got = []
    for name in "kv":
        c, s = state[name + "_codes"][ids], state[name + "_scales"][ids]
        c = c.permute(0, 1, 2, 4, 3).flatten(2, 3) if name == "v" else c
        x = _exact_numbers(c, s.permute(0, 1, 2, 4, 3).flatten(2, 3))       # [pages, heads, page, D]
        got.append(x.permute(1, 0, 2, 3).flatten(1, 2)[:, :upto])
    return got


def _exact_rounded(x):
    """What a block of 32 numbers reads back as."""
    y = x.unflatten(-1, (-1, BLOCK))
    frac, expo = torch.frexp(y.abs().amax(-1, keepdim=True))
    e = (expo - 3 + (frac > 0.875).to(expo.dtype)).clamp(-119, 125)
    unit = 2.0 ** e.double()
    level = torch.tensor(LEVELS[:8], dtype=torch.float64, device=x.device)
    m = (y.abs() / unit).clamp(max=6.0)
    up = torch.searchsorted(level, m.contiguous()).clamp(1, 7)
    lo, hi = level[up - 1], level[up]
    down = (m - lo < hi - m) | ((m - lo == hi - m) & ((up - 1) % 2 == 0))
    return (torch.where(down, lo, hi) * torch.sign(y) * unit).flatten(-2)


def exact(case, seed):
    state = prepare(case, seed)
    H, Hk, D = HEADS[case["heads"]]
    n, page = case["tokens"], case["page"]
    if case["kind"] == "store":
        x = state["proj"].double().view(-1, H + 2 * Hk, D)
        turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device),
                           state["positions"].double()[:, None] * state["inv_freq"].double())[:, None]
        z = torch.complex(x[:, :H + Hk, :D // 2], x[:, :H + Hk, D // 2:]) * turn
        r = torch.cat([z.real, z.imag], dim=-1)
        return {"q": r[:, :H].flatten(1), "k": _exact_rounded(r[:, H:]).flatten(1), "v": _exact_rounded(x[:, H + Hk:]).flatten(1)}
    if case["kind"] == "read":
        ks, vs = [], []
        for b, length in enumerate(state["lens"]):
            k, v = _exact_request(state, b, length)
            more = len(state["tables"][b]) * page - length
            k, v = (torch.nn.functional.pad(t, (0, 0, 0, more)).view(Hk, -1, page, D).transpose(0, 1) for t in (k, v))
            ks.append(k)
            vs.append(v.transpose(2, 3))
        return {"k": torch.cat(ks), "v": torch.cat(vs), "table": None}
    out = []
    q = state["q"].double().view(case["requests"], n, Hk, H // Hk, D)
    for b, length in enumerate(state["lens"]):
        k, v = _exact_request(state, b, length)
        heads = []
        for j in range(Hk):
            s = (q[b, :, j].reshape(-1, D) @ k[j].T).view(n, H // Hk, length) / math.sqrt(D)
            far = torch.arange(length - n, length, device=s.device)[:, None] - torch.arange(length, device=s.device)
            hidden = (far < 0) | (far >= case["window"]) if case["window"] else far < 0
            s = s.masked_fill(hidden[:, None], -math.inf)
            if case["sink"]:
                s = torch.cat([s, state["sinks"].double().view(Hk, 1, -1, 1)[j].expand(n, -1, 1)], dim=-1)
            p = torch.softmax(s, dim=-1)[..., :length]
            heads.append((p.reshape(-1, length) @ v[j]).view(n, H // Hk, D))
        out.append(torch.stack(heads, dim=1).reshape(n, H * D))
    return torch.cat(out)
