"""Oracle of the paged serving operators, in 64 bits on the CPU, request by request and row by row.

``page_bounds``, ``select_pages``, ``selected_attention`` and ``tree_attention`` restate the definitions in
``include/trianglemix_pages.h``.  The attention oracles also return, per output, the sum of weight * |value|, which
the tests' tolerances are derived from.
"""

from __future__ import annotations

import math

import torch

PAGE, BLOCK = 128, 32


def _physical(table, b: int, j: int, pages: int) -> int | None:
    """The cache page of logical page j, None where there is none."""
    if not 0 <= j < table.shape[1]:
        return None
    page = int(table[b, j])
    return page if 0 <= page < pages else None


def page_bounds(keys, table, lens, num_tokens: int, low, high):
    """Updated copies of the bounds."""
    low, high = low.clone(), high.clone()
    for b, n in enumerate(lens.tolist()):
        n = min(max(n, 0), table.shape[1] * PAGE)
        for j in range(max(0, n - num_tokens) // PAGE, -(-n // PAGE)):
            page = _physical(table, b, j, keys.shape[0])
            if page is not None:
                held = keys[page, :n - j * PAGE].double()
                low[page], high[page] = held.amin(dim=0).to(low.dtype), held.amax(dim=0).to(low.dtype)
    return low, high


def block_rows(seq_len: int, rows: int, block: int) -> tuple[int, int]:
    """Positions [first, last] of the rows of a block that are rows of the request; last < first: none."""
    start = max(seq_len, 0) - rows
    return max(0, start + BLOCK * block), start + min(rows, BLOCK * (block + 1)) - 1


def select_pages(query, low, high, table, lens, count: int, sink: int, recent: int):
    batch, kv = table.shape[0], low.shape[1]
    rows, group = query.shape[0] // batch, query.shape[1] // low.shape[1]
    blocks = -(-rows // BLOCK)
    out = torch.full((batch, blocks, kv, count), -1, dtype=torch.int32)
    for b, n in enumerate(lens.tolist()):
        for i in range(blocks):
            first, last = block_rows(n, rows, i)
            if last < first:
                continue
            at = b * rows + first - (max(n, 0) - rows)
            total = query[at:at + last - first + 1].double().sum(dim=0)
            for h in range(kv):
                ranked = []
                for j in range(min(table.shape[1], last // PAGE + 1)):
                    page = _physical(table, b, j, low.shape[0])
                    if page is None:
                        continue
                    best = None  # scores that are no number rank last
                    for q in total[h * group:(h + 1) * group]:
                        score = float(torch.where(q >= 0, q * high[page, h].double(), q * low[page, h].double()).sum())
                        if not math.isnan(score) and (best is None or score > best):
                            best = score
                    forced = j < sink or (recent > 0 and j >= first // PAGE - recent + 1)
                    ranked.append((0 if forced else 1 if best is not None else 2, -best if best is not None else 0.0, j))
                chosen = sorted(j for _, _, j in sorted(ranked)[:count])
                out[b, i, h, :len(chosen)] = torch.tensor(chosen, dtype=torch.int32)
    return out


def _attend(q, keys, values, scale):
    """softmax(scale q keys) values in 64 bits over keys [n, D], and sum of weight * |value|."""
    if keys.shape[0] == 0:
        return torch.zeros(q.shape[0], dtype=torch.float64), torch.zeros(q.shape[0], dtype=torch.float64)
    w = torch.softmax(keys.double() @ q.double() * scale, dim=0)
    return w @ values.double(), w @ values.double().abs()


def selected_attention(query, keys, values, table, lens, pages, scale: float, out):
    """(out updated, sum of weight * |value|, which rows are rows of a request)."""
    batch, kv = table.shape[0], keys.shape[2]
    rows, group = query.shape[0] // batch, query.shape[1] // kv
    out, size = out.double().clone(), torch.zeros(query.shape, dtype=torch.float64)
    written = torch.zeros(query.shape[0], dtype=torch.bool)
    for b, n in enumerate(lens.tolist()):
        for t in range(rows):
            pos = max(n, 0) - rows + t
            if pos < 0:
                continue
            written[b * rows + t] = True
            for h in range(kv):
                ks, vs = [keys[:0, 0, h]], [values[:0, 0, h]]
                for j in sorted(set(pages[b, t // BLOCK, h].tolist())):
                    page = _physical(table, b, j, keys.shape[0])
                    if page is not None and j * PAGE <= pos:
                        ks.append(keys[page, :pos - j * PAGE + 1, h])
                        vs.append(values[page, :pos - j * PAGE + 1, h])
                k, v = torch.cat(ks), torch.cat(vs)
                for g in range(h * group, (h + 1) * group):
                    out[b * rows + t, g], size[b * rows + t, g] = _attend(query[b * rows + t, g], k, v, scale)
    return out, size, written


def tree_attention(query, key, value, keys, values, table, contexts, offsets, mask, scale: float, out):
    """(out updated, sum of weight * |value|, which rows are nodes of a tree)."""
    kv = keys.shape[2]
    group = query.shape[1] // kv
    out, size = out.double().clone(), torch.zeros(query.shape, dtype=torch.float64)
    written = torch.zeros(query.shape[0], dtype=torch.bool)
    for b, n in enumerate(contexts.tolist()):
        n = min(max(n, 0), table.shape[1] * PAGE)
        start, end = int(offsets[b]), int(offsets[b + 1])
        nodes = min(end - start, 64)
        for i in range(nodes):
            written[start + i] = True
            seen = [start + j for j in range(nodes) if int(mask[start + i]) >> j & 1]
            for h in range(kv):
                ks, vs = [key[seen, h]], [value[seen, h]]
                for j in range(-(-n // PAGE)):
                    page = _physical(table, b, j, keys.shape[0])
                    if page is not None:
                        ks.append(keys[page, :n - j * PAGE, h])
                        vs.append(values[page, :n - j * PAGE, h])
                k, v = torch.cat(ks), torch.cat(vs)
                for g in range(h * group, (h + 1) * group):
                    out[start + i, g], size[start + i, g] = _attend(query[start + i, g], k, v, scale)
    return out, size, written


