"""An 8-bit paged KV cache, what fills it and what reads it, as timed cases.

* ``rotate``: ``torch.ops.trianglemix.rotate_positions.out``: the position rotation of query and key rows that do not
  go into the cache yet (drafted tokens, a prompt whose pages are written elsewhere);
* ``append``: ``torch.ops.trianglemix.rotate_and_cache``: a step's projection output: Q rotated into a buffer of its
  own, K rotated, scaled and stored, V scaled and stored, in the pages' slots;
* ``attend``: ``torch.ops.trianglemix.cached_attention.out``: causal attention of the last T tokens of each request
  over its pages, all of them or a window behind the first few tokens.

Caches hold e4m3 numbers with one scale for each KV head, or the queries' own 16-bit type.  Pages hold 128 tokens, heads
128 dims.  Head layouts are the framework's 32 query and 8 KV heads, its tensor-parallel shards, and other groups.
"""

import math
import os
import sys

import torch

own = False

D, PAGE = 128, 128
SCALE = D ** -0.5
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
E4M3, E4M3_MAX = torch.float8_e4m3fn, 448.0


def listed():
    return [
        # the drafted tokens of a batch that verifies them, deep in long contexts, Q and K of a fused projection
        _rotate("rotate_drafts", tokens=57, low=900, high=131072, heads=40),
        # a prompt's chunk, positions in neighbouring pairs and in half of the head only
        _rotate("rotate_chunk", tokens=8191, low=24000, high=24000, heads=40, rotary=64, interleaved=True, dtype="fp16"),
        # a decoding step of a batch into an 8-bit cache, captured with 61 requests where 64 fit
        _append("append_decode", batch=64, rows=1, low=900, high=8192, pad=3),
        # a chunk of a long prompt into an 8-bit cache, frequencies stretched for eight times the trained length
        _append("append_chunk", batch=1, rows=4096, low=100001, high=100001, stretch=8.0),
        # a chunk into a cache of the queries' own type, in front of the prefill kernel
        _append("append_same", batch=1, rows=2048, low=8320, high=8320, cache="same"),
        # one request, one token, on one of four tensor-parallel ranks
        _attend("attend_single", batch=1, rows=1, low=8111, high=8111, heads=8, kv_heads=2),
        # a decoding step of a batch over an 8-bit cache
        _attend("attend_decode", batch=64, rows=1, low=2000, high=16384),
        # a batch that verifies four drafted tokens behind its last one
        _attend("attend_verify", batch=32, rows=5, low=500, high=9000, dtype="fp16"),
        # a batch whose layers see the first tokens and a window alone, a cache of the queries' own type
        _attend("attend_window", batch=64, rows=1, low=900, high=32768, cache="same", window=512, sinks=8),
        # few requests over very long contexts
        _attend("attend_long", batch=4, rows=1, low=65536, high=131072),
        # a chunk of one prompt behind the pages of its earlier chunks
        _attend("attend_chunk", batch=1, rows=512, low=8192, high=8192),
        # a large chunk deep in a long prompt
        _attend("attend_prompt", batch=1, rows=2048, low=32749, high=32749),
    ]


def _rotate(name, tokens, low, high, heads, rotary=128, interleaved=False, base=500000.0, stretch=1.0, dtype="bf16"):
    return {"name": name, "kind": "rotate", "batch": 1 if low == high else tokens, "rows": tokens if low == high else 1,
            "low": low, "high": high, "heads": heads, "rotary": rotary, "interleaved": interleaved, "base": base,
            "stretch": stretch, "dtype": dtype}


def _append(name, batch, rows, low, high, heads=32, kv_heads=8, rotary=128, interleaved=False, base=500000.0, stretch=1.0,
            dtype="bf16", cache="e4m3", pad=0):
    return {"name": name, "kind": "append", "batch": batch, "rows": rows, "low": low, "high": high, "heads": heads,
            "kv_heads": kv_heads, "rotary": rotary, "interleaved": interleaved, "base": base, "stretch": stretch,
            "dtype": dtype, "cache": cache, "pad": pad}


def _attend(name, batch, rows, low, high, heads=32, kv_heads=8, dtype="bf16", cache="e4m3", window=-1, sinks=0):
    return {"name": name, "kind": "attend", "batch": batch, "rows": rows, "low": low, "high": high, "heads": heads,
            "kv_heads": kv_heads, "dtype": dtype, "cache": cache, "window": window, "sinks": sinks}


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["rotate", "append", "append", "attend", "attend", "attend"])
    most = max(_cost(work(c)) for c in listed() if c["kind"] == kind)
    while True:
        heads, kv_heads = rng.choice([(32, 8), (32, 8), (32, 8), (16, 4), (8, 2), (4, 1), (8, 8), (16, 8), (32, 4), (12, 4)])
        dtype, cache = rng.choice(["bf16", "bf16", "fp16"]), rng.choice(["e4m3", "e4m3", "same"])
        long = _log(rng, 300, 131072)
        if rng.random() < 0.6:  # a batch decodes or verifies drafts: ragged contexts
            batch, rows = _log(rng, 1, 64), rng.choice([1, 1, 1, 2, 5, 8, 16])
            low, high = sorted((_log(rng, 100, long), long))
        else:  # a chunk of one prompt, starting and ending anywhere
            batch, low, high = 1, long, long
            rows = min(long, rng.choice([128, 512, 2048, _log(rng, 17, 4096)]))
        turn = {"rotary": rng.choice([128, 128, 64, 96, 32]), "interleaved": rng.random() < 0.4,
                "base": rng.choice([10000.0, 500000.0]), "stretch": rng.choice([1.0, 1.0, 4.0, 8.0])}
        if kind == "rotate":
            tokens = batch * rows
            case = _rotate("", tokens, low, high if batch > 1 else low, heads + kv_heads, dtype=dtype, **turn)
        elif kind == "append":
            case = _append("", batch, rows, low, high, heads, kv_heads, dtype=dtype, cache=cache,
                           pad=rng.choice([0, 0, batch // 4]), **turn)
        else:
            window, sinks = rng.choice([(-1, 0), (-1, 0), (512, 8), (_log(rng, 1, 8192), rng.choice([0, 4, 130]))])
            case = _attend("", batch, rows, low, high, heads, kv_heads, dtype, cache, window, sinks)
        del case["name"]
        if _cost(work(case)) <= most and batch * high <= 1 << 20:
            return case


def _cost(w):
    return max(w["bytes"], w["flops"] / 50)


def _lens(case):
    """The requests' token counts, this step's among them, spread over low .. high."""
    span = case["high"] - case["low"]
    return [case["low"] + int(span * ((b + 1) * 0.6180339887498949 % 1.0)) for b in range(case["batch"])]


def _pages(n):
    return -(-n // PAGE)


def _cached(case):
    """Bytes of one number in the cache."""
    return 1 if case["cache"] == "e4m3" else 2


def _real(case):
    """Tokens of the step that are some: not before their request's first, not of a batch's padding."""
    return sum(min(case["rows"], n) for n in _lens(case)[:case["batch"] - case.get("pad", 0)])


def work(case):
    heads, rows, lens = case["heads"], case["rows"], _lens(case)
    if case["kind"] == "rotate":
        tokens = _real(case)
        return {"bytes": 2 * tokens * heads * D * 2 + tokens * 8, "flops": tokens * heads * 3 * case["rotary"]}
    kv = case["kv_heads"]
    if case["kind"] == "append":
        tokens = _real(case)
        read = tokens * ((heads + 2 * kv) * D * 2 + 16)
        return {"bytes": read + tokens * (heads * D * 2 + 2 * kv * D * _cached(case)),
                "flops": tokens * ((heads + kv) * 3 * case["rotary"] + 2 * kv * D)}
    total = {"bytes": 0, "flops": 0}
    for n in lens:
        first = max(0, n - rows)
        held = n - first
        if case["window"] < 0:
            seen, keys = held * first + held * (held + 1) // 2, n
        else:
            reach, sinks = case["window"] + 1, case["sinks"]
            at = range(first, n)
            seen = sum(min(p + 1, reach + min(sinks, max(0, p + 1 - reach))) for p in at)
            start = max(0, first + 1 - reach)
            keys = n - start + min(sinks, start)
        total["bytes"] += 2 * held * heads * D * 2 + keys * 2 * kv * D * _cached(case)
        total["flops"] += 4 * D * heads * seen
    return total


def _randn(shape, g, dtype):
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype)


def _frequencies(case):
    """Radians a position for each pair of dims; stretched by parts: slow pairs slowed down, fast ones left alone."""
    pairs = case["rotary"] // 2
    f = case["base"] ** (-torch.arange(pairs, dtype=torch.float64) / pairs)
    if case["stretch"] > 1.0:
        turns = 8192 * f / (2 * math.pi)  # over the length that was trained
        keep = ((turns - 1) / 31).clamp(0, 1)
        f = f * keep + f / case["stretch"] * (1 - keep)
    return f.cuda()


def _magnitude(case):
    return 0.1 * math.log(case["stretch"]) + 1.0


def _scales(kv, g):
    """What a calibration leaves: the largest number of a head, or nearly so, at the largest of the type."""
    return (4.0 + torch.rand(kv, generator=g, device="cuda")) / E4M3_MAX


def prepare(case, seed):
    if own:
        _native()
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype, heads, batch, rows = TYPES[case["dtype"]], case["heads"], case["batch"], case["rows"]
    lens = torch.tensor(_lens(case), dtype=torch.int32, device="cuda")
    s = {"case": case, "lens": lens}
    position = (lens.long()[:, None] - rows + torch.arange(rows, device="cuda")).clamp(min=-1)
    if case["kind"] != "attend":
        s["frequencies"], s["magnitude"] = _frequencies(case), _magnitude(case)
    if case["kind"] == "rotate":
        s["positions"] = position.flatten()
        # Q and K of the projection's output, V behind them
        s["qkv"] = _randn((batch * rows, heads + 8, D), g, dtype)
        s["out"] = torch.zeros((batch * rows, heads, D), dtype=dtype, device="cuda")
        return s
    kv = case["kv_heads"]
    used = [_pages(n) for n in _lens(case)]
    pages = sum(used) + 7  # the pages of all requests, anywhere in a cache with some pages more
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    s["table"] = torch.zeros(batch, max(used), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(used):
        s["table"][b, :n] = order[at:at + n]
        at += n
    s["key_scale"] = s["value_scale"] = None
    if case["cache"] == "e4m3":
        s["key_scale"], s["value_scale"] = _scales(kv, g), _scales(kv, g)
    s["keys"] = _stored(_randn((pages, PAGE, kv, D), g, dtype), s["key_scale"])
    s["values"] = _stored(_randn((pages, PAGE, kv, D), g, dtype), s["value_scale"])
    if case["kind"] == "append":
        page = s["table"].long().gather(1, position.clamp(min=0) // PAGE)
        slots = torch.where(position >= 0, page * PAGE + position % PAGE, -1)
        if case["pad"]:
            position[-case["pad"]:], slots[-case["pad"]:] = -1, -1
        s["positions"], s["slots"] = position.flatten().contiguous(), slots.flatten().contiguous()
        s["stored"] = torch.nonzero(s["slots"] >= 0).flatten()
        s["qkv"] = _randn((batch * rows, heads + 2 * kv, D), g, dtype)
        s["query"] = torch.zeros((batch * rows, heads, D), dtype=dtype, device="cuda")
    else:
        s["query"] = _randn((batch * rows, heads, D), g, dtype)
        s["query"] += _randn((1, heads, D), g, dtype)  # the queries of a head have much in common
        s["out"] = torch.zeros_like(s["query"])
    return s


def _stored(x, scale):
    """Rows as a cache holds them: the type's nearest number of x / scale, the largest one beyond its range."""
    if scale is None:
        return x
    return (x.float() / scale[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(E4M3)


def run(s):
    return (_own if own else _plain)(s)


# ---- the framework's kernels ----

def _native():
    package = os.path.abspath("sparse-attention-op-for-ascend-npu-_amd")
    if package not in sys.path:
        sys.path.insert(1, package)
    from trianglemix import native

    native.require_adapter()


def _own(s):
    case, heads = s["case"], s["case"]["heads"]
    ops = torch.ops.trianglemix
    if case["kind"] == "rotate":
        return ops.rotate_positions.out(s["qkv"][:, :heads], s["positions"], s["frequencies"], case["interleaved"],
                                        s["magnitude"], out=s["out"])
    kv = case["kv_heads"]
    if case["kind"] == "append":
        ops.rotate_and_cache(s["qkv"][:, :heads], s["qkv"][:, heads:heads + kv], s["qkv"][:, heads + kv:], s["positions"],
                             s["slots"], s["frequencies"], case["interleaved"], s["magnitude"], s["query"], s["keys"],
                             s["values"], s["key_scale"], s["value_scale"])
        return s["query"], s["keys"], s["values"]
    return ops.cached_attention.out(s["query"], s["keys"], s["values"], s["table"], s["lens"], SCALE, case["window"],
                                    case["sinks"], s["key_scale"], s["value_scale"], out=s["out"])


# ---- the plain forms ----

def _plain(s):
    return {"rotate": _plain_rotate, "append": _plain_append, "attend": _plain_attend}[s["case"]["kind"]](s)


def _turned(x, s):
    """Rows x [tokens, heads, 128] rotated by their positions, in 32 bits; the angles are formed in 64."""
    case = s["case"]
    angle = s["positions"].double()[:, None, None] * s["frequencies"]
    c, t = (angle.cos() * s["magnitude"]).float(), (angle.sin() * s["magnitude"]).float()
    x, n = x.float(), case["rotary"]
    if case["interleaved"]:
        a, b = x[..., 0:n:2], x[..., 1:n:2]
        turned = torch.stack([a * c - b * t, b * c + a * t], dim=-1).flatten(-2)
    else:
        a, b = x[..., :n // 2], x[..., n // 2:n]
        turned = torch.cat([a * c - b * t, b * c + a * t], dim=-1)
    return torch.cat([turned, x[..., n:]], dim=-1)


def _plain_rotate(s):
    x = s["qkv"][:, :s["case"]["heads"]]
    held = (s["positions"] >= 0)[:, None, None]
    s["out"].copy_(torch.where(held, _turned(x, s).to(x.dtype), s["out"]))
    return s["out"]


def _plain_append(s):
    heads, kv = s["case"]["heads"], s["case"]["kv_heads"]
    turned = _turned(s["qkv"][:, :heads + kv], s)
    held = (s["positions"] >= 0)[:, None, None]
    s["query"].copy_(torch.where(held, turned[:, :heads].to(s["query"].dtype), s["query"]))
    rows = s["stored"]
    slots = s["slots"][rows]
    kind = s["keys"].dtype
    bits = torch.uint8 if kind == E4M3 else kind  # indexed writes know no 8-bit floats
    new = _stored(turned[:, heads:][rows], s["key_scale"]).to(kind).view(bits)
    s["keys"].view(bits).view(-1, kv, D)[slots] = new
    new = _stored(s["qkv"][:, heads + kv:][rows], s["value_scale"]).to(kind).view(bits)
    s["values"].view(bits).view(-1, kv, D)[slots] = new
    return s["query"], s["keys"], s["values"]


def _seen(case, position, key):
    """Which keys a query at this position attends."""
    seen = (key <= position) & (position >= 0)
    if case["window"] >= 0:
        seen &= (key >= position - case["window"]) | (key < case["sinks"])
    return seen


def _plain_attend(s):
    case = s["case"]
    batch, rows, heads, kv = case["batch"], case["rows"], case["heads"], case["kv_heads"]
    group = heads // kv
    table = s["table"].long()
    tokens = table.shape[1] * PAGE
    position = s["lens"].long()[:, None] - rows + torch.arange(rows, device="cuda")
    seen = _seen(case, position[:, :, None], torch.arange(tokens, device="cuda"))

    def gathered(cache, scale):  # [batch, KV heads, tokens, 128]
        x = cache.view(torch.uint8)[table].view(cache.dtype) if cache.dtype == E4M3 else cache[table]
        x = x.view(batch, tokens, kv, D).permute(0, 2, 1, 3).float()
        return x if scale is None else x * scale[:, None, None]

    q = s["query"].float().view(batch, rows, kv, group, D).permute(0, 2, 3, 1, 4).reshape(batch, kv, group * rows, D)
    score = (q * SCALE) @ gathered(s["keys"], s["key_scale"]).transpose(2, 3)
    score = score.view(batch, kv, group, rows, tokens).masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(dim=-1, keepdim=True)
    p = score.sub_(torch.where(top > -math.inf, top, 0.0)).exp_()
    total = p.sum(dim=-1, keepdim=True)
    out = p.view(batch, kv, group * rows, tokens) @ gathered(s["values"], s["value_scale"])
    out = out.view(batch, kv, group, rows, D) / torch.where(total > 0, total, 1.0)
    out = out.permute(0, 3, 1, 2, 4).reshape(batch * rows, heads, D)
    held = (position >= 0).view(-1, 1, 1)  # rows before a request's first are left alone
    s["out"].copy_(torch.where(held, out.to(s["out"].dtype), s["out"]))
    return s["out"]


# ---- the definitions in 64 bits ----

def exact(case, seed):
    s = prepare(case, seed)
    return {"rotate": _exact_rotate, "append": _exact_append, "attend": _exact_attend}[case["kind"]](s, case)


def _exact_turned(x, s, case):
    x = x.double().clone()
    n = case["rotary"]
    for i in range(n // 2):
        a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, n // 2 + i)
        angle = (s["positions"].double() * s["frequencies"][i])[:, None]
        c, t = s["magnitude"] * torch.cos(angle), s["magnitude"] * torch.sin(angle)
        x[..., a], x[..., b] = x[..., a] * c - x[..., b] * t, x[..., a] * t + x[..., b] * c
    return x


def _exact_rotate(s, case):
    out = _exact_turned(s["qkv"][:, :case["heads"]], s, case)
    return torch.where((s["positions"] < 0)[:, None, None], s["out"].double(), out)


def _exact_append(s, case):
    heads, kv = case["heads"], case["kv_heads"]
    fresh = {"keys": _exact_turned(s["qkv"][:, heads:heads + kv], s, case), "values": s["qkv"][:, heads + kv:].double()}
    query = _exact_turned(s["qkv"][:, :heads], s, case)
    query = torch.where((s["positions"] < 0)[:, None, None], s["query"].double(), query)
    result = [query]
    row = s["stored"]
    for name, scale in (("keys", s["key_scale"]), ("values", s["value_scale"])):
        cache = s[name].double()
        x = fresh[name][row]
        if scale is not None:
            x = (x / scale.double()[:, None]).clamp(-E4M3_MAX, E4M3_MAX)
        cache[s["slots"][row] // PAGE, s["slots"][row] % PAGE] = x
        result.append(cache)
    return tuple(result)


def _exact_attend(s, case):
    kv, rows, group = case["kv_heads"], case["rows"], case["heads"] // case["kv_heads"]
    out = s["out"].double()
    for b, n in enumerate(_lens(case)):
        phys = s["table"][b, :_pages(n)].long()
        keys = s["keys"].view(torch.uint8)[phys].view(s["keys"].dtype).double().flatten(0, 1)[:n]
        values = s["values"].view(torch.uint8)[phys].view(s["values"].dtype).double().flatten(0, 1)[:n]
        if case["cache"] == "e4m3":
            keys = keys * s["key_scale"].double()[:, None]
            values = values * s["value_scale"].double()[:, None]
        for first in range(max(0, n - rows), n, 256):
            position = torch.arange(first, min(n, first + 256), device="cuda")
            at = b * rows + first - (n - rows)
            unseen = ~_seen(case, position[:, None], torch.arange(n, device="cuda"))
            for h in range(case["heads"]):
                score = s["query"][at:at + len(position), h].double() @ keys[:, h // group].t() * SCALE
                weight = torch.softmax(score.masked_fill(unseen, -math.inf), dim=-1)
                out[at:at + len(position), h] = weight @ values[:, h // group]
    return out
