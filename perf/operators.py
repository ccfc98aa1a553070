"""Serving over a long paged KV cache, as timed cases: attention over selected pages, and over draft trees.

* ``bounds``: ``torch.ops.trianglemix.update_page_bounds``, after a step has written its K rows into their pages: the
  elementwise smallest and largest key of every page the step wrote to;
* ``select``: ``torch.ops.trianglemix.select_pages``: for each block of 32 query rows and each KV head, the pages that
  a cheap score, an upper bound of the block's summed dot products with any key of a page, ranks highest;
* ``attend``: ``torch.ops.trianglemix.selected_page_attention.out``: causal attention of those rows over those pages;
* ``tree``: ``torch.ops.trianglemix.tree_attention.out``: one verification step of speculative decoding, each node
  of a request's draft tree attending the whole cache of its request and its ancestors in the tree; a tree of one
  node is a plain decoding step.

The query of a batch is ``[B * T, Hq, 128]``: the last T tokens of each of B requests (a prefill chunk is one request
with many rows, a decoding step many requests with one row).  Pages hold 128 tokens.  Head layouts are the
framework's 32 query and 8 KV heads, its tensor-parallel shards, and other group sizes.
"""

import math
import os
import sys

import torch

own = False

D, PAGE, BLOCK = 128, 128, 32
SCALE = D ** -0.5
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # a decoding step of a batch: one more key in the last page of each request
        _case("bounds_decode", "bounds", batch=64, rows=1, low=900, high=32768),
        # a prefill chunk of one request, deep in a long prompt, off the page borders
        _case("bounds_chunk", "bounds", batch=1, rows=2048, low=131000, high=131000),
        # a decoding step of a batch over long contexts
        _case("select_decode", "select", batch=32, rows=1, low=16384, high=131072, count=32),
        # one request, one token, on one of two tensor-parallel ranks
        _case("select_single", "select", batch=1, rows=1, low=8111, high=8111, count=16, heads=16, kv_heads=4),
        # a prefill chunk of a long prompt
        _case("select_chunk", "select", batch=1, rows=2048, low=131072, high=131072, count=32),
        # the smallest call: one request decodes one token
        _case("attend_single", "attend", batch=1, rows=1, low=8192, high=8192, count=16),
        # a decoding step of a ragged batch
        _case("attend_decode", "attend", batch=64, rows=1, low=2000, high=16384, count=24),
        # a chunk of 512 at the end of an 8192-token prompt
        _case("attend_chunk", "attend", batch=1, rows=512, low=8192, high=8192, count=16),
        # a chunk of 2048 of a long prompt
        _case("attend_long", "attend", batch=1, rows=2048, low=131072, high=131072, count=32),
        # one request verifies a small tree right after a short prompt
        _case("tree_single", "tree", batch=1, nodes=7, low=77, high=77),
        # a ragged batch verifies trees of up to 24 nodes, in fp16 on a tensor-parallel rank
        _case("tree_batch", "tree", batch=32, nodes=24, low=500, high=9000, heads=16, kv_heads=4, dtype="fp16"),
        # a few requests with very long contexts and large trees
        _case("tree_long", "tree", batch=4, nodes=60, low=65000, high=131072),
    ]


def _case(name, kind, batch, low, high, rows=1, count=0, nodes=0, heads=32, kv_heads=8, dtype="bf16"):
    return {"name": name, "kind": kind, "batch": batch, "rows": rows, "low": low, "high": high, "count": count,
            "nodes": nodes, "heads": heads, "kv_heads": kv_heads, "dtype": dtype}


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["bounds", "select", "attend", "attend", "tree", "tree"])
    most = max((work(c) for c in listed() if c["kind"] == kind), key=_cost)
    while True:
        heads, kv_heads = rng.choice([(32, 8), (32, 8), (32, 8), (16, 4), (8, 2), (4, 1), (8, 8), (16, 8), (32, 4)])
        case = _case("", kind, batch=1, low=1, high=1, heads=heads, kv_heads=kv_heads,
                     dtype=rng.choice(["bf16", "bf16", "fp16"]))
        del case["name"]
        long = _log(rng, 300, 131072)
        if kind == "tree" or rng.random() < 0.5:  # a batch decodes: ragged contexts
            case["batch"] = _log(rng, 1, 64)
            case["low"], case["high"] = sorted((_log(rng, 100, long), long))
            case["rows"] = rng.choice([1, 1, 1, 2, 5, 16])
        else:  # a chunk of one prompt, starting and ending anywhere
            case["low"] = case["high"] = long
            case["rows"] = min(long, rng.choice([128, 256, 512, 1024, 2048, rng.randrange(17, 2048)]))
        if kind in ("select", "attend"):
            case["count"] = rng.choice([4, 8, 16, 16, 32, 32, rng.randrange(4, 65)])
        if kind == "tree":
            case["rows"], case["nodes"] = 1, rng.choice([1, 1, rng.randrange(2, 65), rng.randrange(2, 65)])
        if _cost(work(case)) <= _cost(most) and _tokens(case) <= 1 << 20:
            return case


def _cost(w):
    return max(w["bytes"], w["flops"] / 50)


def _lens(case):
    """The requests' token counts, spread over low .. high; a tree's context does not count its nodes."""
    span = case["high"] - case["low"]
    return [case["low"] + int(span * ((b + 1) * 0.6180339887498949 % 1.0)) for b in range(case["batch"])]


def _nodes(case):
    """The requests' tree sizes: the full one first, smaller ones among the rest."""
    return [max(1, case["nodes"] - (b * 7) % (case["nodes"] // 2 + 1)) for b in range(case["batch"])]


def _pages(n):
    return -(-n // PAGE)


def _tokens(case):
    return sum(_lens(case))


def _blocks(case):
    return -(-case["rows"] // BLOCK)


def work(case):
    heads, kv, rows, lens = case["heads"], case["kv_heads"], case["rows"], _lens(case)
    row = kv * D * 2  # bytes of one token's K
    if case["kind"] == "bounds":
        read = pages = 0
        for n in lens:
            first = max(0, n - rows) // PAGE
            read += n - first * PAGE
            pages += _pages(n) - first
        return {"bytes": read * row + pages * 2 * row, "flops": read * kv * D * 2}
    if case["kind"] == "select":
        total = {"bytes": 0, "flops": 0}
        for n in lens:
            total["bytes"] += min(rows, n) * heads * D * 2 + _pages(n) * 2 * row
            total["bytes"] += _blocks(case) * kv * case["count"] * 4
            for i in range(_blocks(case)):
                last = n - rows + min(rows, BLOCK * (i + 1)) - 1
                total["flops"] += 2 * heads * D * _pages(last + 1) + BLOCK * heads * D if last >= 0 else 0
        return total
    total = {"bytes": 0, "flops": 0}
    if case["kind"] == "attend":
        for n in lens:
            total["bytes"] += 2 * min(rows, n) * heads * D * 2 + _blocks(case) * kv * case["count"] * 4
            total["bytes"] += min(n, _blocks(case) * case["count"] * PAGE) * 2 * row
            for i in range(_blocks(case)):
                first, last = n - rows + BLOCK * i, n - rows + min(rows, BLOCK * (i + 1)) - 1
                held = max(0, last - max(first, 0) + 1)
                keys = min(case["count"] * PAGE - (PAGE - 1 - last % PAGE), last + 1)
                total["flops"] += 4 * D * heads * held * max(0, keys)
        return total
    for n, t in zip(lens, _nodes(case)):
        total["bytes"] += 2 * t * heads * D * 2 + (n + t) * 2 * row
        total["flops"] += 4 * D * heads * t * n
    return total


def _randn(shape, g, dtype):
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype)


def _ancestors(parents):
    """Bit j of entry i: node i attends node j (itself and its ancestors), as signed 64-bit numbers."""
    bits = []
    for i, p in enumerate(parents):
        bits.append((bits[p] if p >= 0 else 0) | 1 << i)
    return [b - (1 << 64) if b >> 63 else b for b in bits]


def prepare(case, seed):
    if own:
        _native()
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    host = torch.Generator().manual_seed(int(seed))
    dtype, heads, kv, batch, rows = TYPES[case["dtype"]], case["heads"], case["kv_heads"], case["batch"], case["rows"]
    lens = _lens(case)
    used = [_pages(n) for n in lens]
    pages = sum(used) + 7  # the pages of all requests, anywhere in a cache with some pages more
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(batch, max(used), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    s = {"case": case, "table": table, "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"), "pages": pages}
    if case["kind"] == "select":
        # the bounds of pages of 128 keys around a centre of their own
        centre = _randn((pages, kv, D), g, torch.float32) * 0.7
        reach = 2.0 + 0.5 * torch.rand((2, pages, kv, D), generator=g, device="cuda")
        s["low"], s["high"] = (centre - reach[0]).to(dtype), (centre + reach[1]).to(dtype)
    else:
        s["keys"] = _randn((pages, PAGE, kv, D), g, dtype)
        s["keys"] += _randn((pages, 1, kv, D), g, dtype) * 0.7  # the keys of a page have much in common
    if case["kind"] in ("attend", "tree"):
        s["values"] = _randn((pages, PAGE, kv, D), g, dtype)
    if case["kind"] == "bounds":
        # what the pages held before this step
        s["low"], s["high"] = _randn((pages, kv, D), g, dtype), _randn((pages, kv, D), g, dtype)
    if case["kind"] in ("select", "attend"):
        s["query"] = _randn((batch * rows, heads, D), g, dtype)
        s["query"] += _randn((1, heads, D), g, dtype)  # the queries of a head have much in common
    if case["kind"] == "attend":
        s["out"] = torch.zeros_like(s["query"])
        # the first page, the pages of the block's rows and others at random
        n = torch.tensor(lens, device="cuda").view(batch, 1, 1, 1)
        first = n - rows + BLOCK * torch.arange(_blocks(case), device="cuda").view(1, -1, 1, 1)
        last = (first + BLOCK).clamp(max=n) - 1
        j = torch.arange(max(used), device="cuda").view(1, 1, 1, -1)
        liking = torch.rand((batch, _blocks(case), kv, max(used)), generator=g, device="cuda")
        liking = torch.where((j == 0) | (j >= first // PAGE), 2.0, liking).masked_fill(j > last // PAGE, -1.0)
        best = liking.topk(min(case["count"], max(used)), dim=-1)
        chosen = torch.where(best.values >= 0, best.indices, 1 << 30).sort(dim=-1).values
        chosen = torch.where(chosen < 1 << 30, chosen, -1).to(torch.int32)
        s["chosen"] = torch.full((batch, _blocks(case), kv, case["count"]), -1, dtype=torch.int32, device="cuda")
        s["chosen"][..., :chosen.shape[-1]] = chosen
    if case["kind"] == "tree":
        nodes = _nodes(case)
        total = sum(nodes)
        masks, offsets = [], [0]
        for t in nodes:  # each node hangs on one of the few before it, or begins a branch of its own
            back = torch.randint(1, 5, (t,), generator=host).tolist()
            masks += _ancestors([i - k if i >= k else -1 for i, k in enumerate(back)])
            offsets.append(offsets[-1] + t)
        s["mask"] = torch.tensor(masks, dtype=torch.int64, device="cuda")
        s["offsets"] = torch.tensor(offsets, dtype=torch.int32, device="cuda")
        # the projection's output: Q, K and V of a token side by side; the rotary embedding gives Q its own buffer
        s["qkv"] = _randn((total, heads + 2 * kv, D), g, dtype)
        s["query"] = s["qkv"][:, :heads].contiguous()
        s["out"] = torch.zeros_like(s["query"])
        s["sizes"], s["contexts"] = nodes, lens
    return s


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
    case, kind = s["case"], s["case"]["kind"]
    ops = torch.ops.trianglemix
    if kind == "bounds":
        ops.update_page_bounds(s["keys"], s["table"], s["lens"], case["rows"], s["low"], s["high"])
        return s["low"], s["high"]
    if kind == "select":
        return ops.select_pages(s["query"], s["low"], s["high"], s["table"], s["lens"], case["count"], 1, 1)
    if kind == "attend":
        ops.selected_page_attention.out(s["query"], s["keys"], s["values"], s["table"], s["lens"], s["chosen"], SCALE,
                                        out=s["out"])
        return s["out"]
    heads, kv = case["heads"], case["kv_heads"]
    ops.tree_attention.out(s["query"], s["qkv"][:, heads:heads + kv], s["qkv"][:, heads + kv:], s["keys"], s["values"],
                           s["table"], s["lens"], s["offsets"], s["mask"], SCALE, out=s["out"])
    return s["out"]


# ---- the plain forms ----

def _plain(s):
    return {"bounds": _plain_bounds, "select": _plain_select, "attend": _plain_attend, "tree": _plain_tree}[
        s["case"]["kind"]](s)


def _plain_bounds(s):
    rows, lens, table = s["case"]["rows"], s["lens"].long(), s["table"].long()
    first = (lens - rows).clamp(min=0) // PAGE
    j = first[:, None] + torch.arange(_pages(rows) + 1, device="cuda")  # the pages a request's last rows can lie in
    written = j * PAGE < lens[:, None]
    phys = table.gather(1, j.clamp(max=table.shape[1] - 1))
    keys = s["keys"][phys].float()
    held = (j[:, :, None] * PAGE + torch.arange(PAGE, device="cuda") < lens[:, None, None])[..., None, None]
    low = keys.masked_fill(~held, math.inf).amin(dim=2).to(s["low"].dtype)
    high = keys.masked_fill(~held, -math.inf).amax(dim=2).to(s["low"].dtype)
    s["low"][phys[written]] = low[written]
    s["high"][phys[written]] = high[written]
    return s["low"], s["high"]


def _rows(s):
    """The positions of the query rows as [B, blocks, 32], and which of them are rows of their request."""
    case = s["case"]
    t = torch.arange(_blocks(case) * BLOCK, device="cuda")
    pos = (s["lens"].long() - case["rows"])[:, None] + t
    real = (pos >= 0) & (t < case["rows"])
    return pos.view(case["batch"], -1, BLOCK), real.view(case["batch"], -1, BLOCK)


def _blocked(x, case):
    """[B * T, H, D] as [B, blocks, 32, H, D], zeros behind the last row."""
    x = x.view(case["batch"], case["rows"], *x.shape[1:])
    pad = _blocks(case) * BLOCK - case["rows"]
    if pad:
        x = torch.cat([x, x.new_zeros(case["batch"], pad, *x.shape[2:])], dim=1)
    return x.view(case["batch"], -1, BLOCK, *x.shape[2:])


def _plain_select(s):
    case = s["case"]
    kv, count = case["kv_heads"], case["count"]
    pos, real = _rows(s)
    # in 64 bits: which page comes last may hang on the last bits
    q = (_blocked(s["query"], case).double() * real[..., None, None]).sum(dim=2)  # [B, blocks, Hq, D]
    n = s["table"].shape[1]
    j = torch.arange(n, device="cuda")
    big = 1 << 40
    first = torch.where(real, pos, big).amin(dim=2)[:, :, None]
    last = torch.where(real, pos, -1).amax(dim=2)[:, :, None]
    last_page = torch.div(last, PAGE, rounding_mode="floor")
    forced = (j < 1) | (j >= first // PAGE)
    result = []
    for b in range(case["batch"]):
        phys = s["table"][b].long()
        low = s["low"][phys].double().permute(1, 2, 0).contiguous()  # [Hkv, D, pages]
        high = s["high"][phys].double().permute(1, 2, 0).contiguous()
        qb = q[b].view(-1, kv, case["heads"] // kv, D).permute(1, 0, 2, 3).reshape(kv, -1, D)
        score = qb.clamp(min=0) @ high + qb.clamp(max=0) @ low
        score = score.view(kv, -1, case["heads"] // kv, n).amax(dim=2).permute(1, 0, 2)  # [blocks, Hkv, pages]
        score = score.masked_fill(forced[b][:, None], math.inf)
        score = score.masked_fill((j > last_page[b])[:, None], -math.inf)
        order = score.sort(dim=-1, descending=True, stable=True).indices[..., :count]  # ties: the lowest first
        order = order.masked_fill(order > last_page[b][:, :, None], big).sort(dim=-1).values
        chosen = torch.full((*order.shape[:2], count), -1, dtype=torch.int32, device="cuda")
        chosen[..., :order.shape[-1]] = torch.where(order < big, order, -1)
        result.append(chosen)
    return torch.stack(result)


def _softmax_values(score, seen, values):
    """softmax(score over what is seen) @ values; rows that see nothing give zeros."""
    score = score.masked_fill(~seen, -math.inf)
    top = score.amax(dim=-1, keepdim=True)
    p = (score - torch.where(top > -math.inf, top, 0.0)).exp()
    total = p.sum(dim=-1, keepdim=True)
    return (p @ values) / torch.where(total > 0, total, 1.0)


def _plain_attend(s):
    case = s["case"]
    batch, heads, kv, count = case["batch"], case["heads"], case["kv_heads"], case["count"]
    group, blocks = heads // kv, _blocks(case)
    pos, real = _rows(s)
    q = _blocked(s["query"], case).float() * SCALE
    q = q.view(batch * blocks, BLOCK, kv, group, D).permute(0, 2, 1, 3, 4).reshape(batch * blocks, kv, BLOCK * group, D)
    pos, chosen = pos.reshape(-1, BLOCK), s["chosen"].view(batch * blocks, kv, count).long()
    request = torch.arange(batch, device="cuda").repeat_interleave(blocks)
    head = torch.arange(kv, device="cuda").view(1, kv, 1, 1)
    slot = torch.arange(PAGE, device="cuda")
    out = torch.empty(batch * blocks, kv, BLOCK * group, D, device="cuda")
    step = max(1, (1 << 28) // (kv * count * PAGE * D))
    for at in range(0, batch * blocks, step):
        part = slice(at, at + step)
        logical = chosen[part]
        phys = s["table"][request[part].view(-1, 1, 1), logical.clamp(min=0)].long()[..., None]
        keys = s["keys"][phys, slot, head].float().flatten(2, 3)
        values = s["values"][phys, slot, head].float().flatten(2, 3)
        at_keys = torch.where(logical[..., None] >= 0, logical[..., None] * PAGE + slot, 1 << 40).flatten(2)
        row = pos[part].repeat_interleave(group, dim=1)
        seen = at_keys[:, :, None, :] <= row[:, None, :, None]
        out[part] = _softmax_values(q[part] @ keys.transpose(2, 3), seen, values)
    out = out.view(batch, blocks, kv, BLOCK, group, D).permute(0, 1, 3, 2, 4, 5)
    out = out.reshape(batch, blocks * BLOCK, heads, D)[:, :case["rows"]].reshape(-1, heads, D)
    held = real.view(batch, -1)[:, :case["rows"]].reshape(-1, 1, 1)  # rows before a request's first are left alone
    s["out"].copy_(torch.where(held, out.to(s["out"].dtype), s["out"]))
    return s["out"]


def _plain_tree(s):
    case = s["case"]
    heads, kv = case["heads"], case["kv_heads"]
    group = heads // kv
    at = 0
    for b, (t, n) in enumerate(zip(s["sizes"], s["contexts"])):
        phys = s["table"][b, :_pages(n)].long()
        fresh = s["qkv"][at:at + t, heads:].float()
        keys = torch.cat([s["keys"][phys].view(-1, kv, D)[:n].float(), fresh[:, :kv]]).transpose(0, 1)
        values = torch.cat([s["values"][phys].view(-1, kv, D)[:n].float(), fresh[:, kv:]]).transpose(0, 1)
        q = s["query"][at:at + t].float().view(t, kv, group, D).permute(1, 0, 2, 3).reshape(kv, t * group, D) * SCALE
        bit = torch.arange(t, device="cuda")
        seen = torch.ones(t, n + t, dtype=torch.bool, device="cuda")
        seen[:, n:] = (s["mask"][at:at + t, None] >> bit) & 1 != 0
        out = _softmax_values(q @ keys.transpose(1, 2), seen.repeat_interleave(group, dim=0), values)
        s["out"][at:at + t] = out.view(kv, t, group, D).permute(1, 0, 2, 3).reshape(t, heads, D).to(s["out"].dtype)
        at += t
    return s["out"]


# ---- the definitions in 64 bits ----

def exact(case, seed):
    s = prepare(case, seed)
    return {"bounds": _exact_bounds, "select": _exact_select, "attend": _exact_attend, "tree": _exact_tree}[
        case["kind"]](s, case)


def _exact_bounds(s, case):
    low, high = s["low"].double(), s["high"].double()
    for b, n in enumerate(_lens(case)):
        for j in range(max(0, n - case["rows"]) // PAGE, _pages(n)):
            page = int(s["table"][b, j])
            keys = s["keys"][page, :min(PAGE, n - j * PAGE)].double()
            low[page], high[page] = keys.min(dim=0).values, keys.max(dim=0).values
    return low, high


def _exact_select(s, case):
    kv, count, rows = case["kv_heads"], case["count"], case["rows"]
    group = case["heads"] // kv
    result = torch.full((case["batch"], _blocks(case), kv, count), -1, dtype=torch.int32, device="cuda")
    for b, n in enumerate(_lens(case)):
        phys = s["table"][b, :_pages(n)].long()
        low, high = s["low"][phys].double(), s["high"][phys].double()
        for i in range(_blocks(case)):
            first, last = max(0, n - rows + BLOCK * i), n - rows + min(rows, BLOCK * (i + 1)) - 1
            if last < 0:
                continue
            at = b * rows + first - (n - rows)
            total = s["query"][at:at + last - first + 1].double().sum(dim=0)
            pages = last // PAGE + 1
            for h in range(kv):
                best = None
                for q in total[h * group:(h + 1) * group]:
                    score = torch.where(q >= 0, q * high[:pages, h], q * low[:pages, h]).sum(dim=1)
                    best = score if best is None else torch.maximum(best, score)
                best[:1] = math.inf
                best[first // PAGE:] = math.inf
                chosen = torch.argsort(best, descending=True, stable=True)[:count].sort().values
                result[b, i, h, :len(chosen)] = chosen.int()
    return result


def _exact_attend(s, case):
    kv, rows = case["kv_heads"], case["rows"]
    group = case["heads"] // kv
    out = s["out"].double()
    chosen, table = s["chosen"].cpu(), s["table"].cpu()
    for b, n in enumerate(_lens(case)):
        for i in range(_blocks(case)):
            first, last = max(0, n - rows + BLOCK * i), n - rows + min(rows, BLOCK * (i + 1)) - 1
            if last < first:
                continue
            at = b * rows + first - (n - rows)
            pos = torch.arange(first, last + 1, device="cuda")
            for h in range(kv):
                logical = chosen[b, i, h][chosen[b, i, h] >= 0].long()
                phys = table[b, logical].long().cuda()
                where = (logical[:, None] * PAGE + torch.arange(PAGE)).flatten().cuda()
                keys, values = s["keys"][phys, :, h].double().flatten(0, 1), s["values"][phys, :, h].double().flatten(0, 1)
                seen = where[None, :] <= pos[:, None]
                q = s["query"][at:at + len(pos), h * group:(h + 1) * group].double()
                score = (q.reshape(-1, D) @ keys.t()).view(len(pos), group, -1) * SCALE
                weight = torch.softmax(score.masked_fill(~seen[:, None], -math.inf), dim=-1).nan_to_num(0.0)
                out[at:at + len(pos), h * group:(h + 1) * group] = weight @ values
    return out


def _exact_tree(s, case):
    heads, kv = case["heads"], case["kv_heads"]
    group = heads // kv
    out = s["out"].double()
    at = 0
    for b, (t, n) in enumerate(zip(_nodes(case), _lens(case))):
        phys = s["table"][b, :_pages(n)].long()
        bits = s["mask"][at:at + t].tolist()
        seen = torch.tensor([[m >> j & 1 for j in range(t)] for m in bits], dtype=torch.bool, device="cuda")
        seen = torch.cat([torch.ones(t, n, dtype=torch.bool, device="cuda"), seen], dim=1)
        for h in range(kv):
            keys = torch.cat([s["keys"][phys, :, h].flatten(0, 1)[:n], s["qkv"][at:at + t, heads + h]]).double()
            values = torch.cat([s["values"][phys, :, h].flatten(0, 1)[:n], s["qkv"][at:at + t, heads + kv + h]]).double()
            for q in range(h * group, (h + 1) * group):
                score = s["query"][at:at + t, q].double() @ keys.t() * SCALE
                out[at:at + t, q] = torch.softmax(score.masked_fill(~seen, -math.inf), dim=-1) @ values
        at += t
    return out
