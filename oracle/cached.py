"""Oracle of the cached-attention operators, in 64 bits on the CPU.

``rotate``, ``stored`` and ``attention`` restate the definitions in ``include/trianglemix_cached.h``; the attention
oracle also returns, per output, the sum of weight * |value|, which the tests' tolerances are derived from.
"""

from __future__ import annotations

import torch

PAGE = 128
E4M3_MAX = 448.0


def rotate(x, positions, freqs, interleaved: bool, magnitude: float):
    """Rows ``[rows, heads, 128]`` in 64 bits; rows at negative positions are what they were."""
    out = x.double().clone()
    pairs = freqs.shape[0]
    for r, p in enumerate(positions.tolist()):
        if p < 0:
            continue
        angle = p * freqs.double()
        cos, sin = magnitude * torch.cos(angle), magnitude * torch.sin(angle)
        for i in range(pairs):
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + pairs)
            u, v = x[r, :, a].double(), x[r, :, b].double()
            out[r, :, a], out[r, :, b] = u * cos[i] - v * sin[i], v * cos[i] + u * sin[i]
    return out


def quotient(x, scale):
    """``x [..., heads, 128]`` by the heads' scales, within the range of an 8-bit cache; NaN stays."""
    return (x.double() / scale.double()[:, None]).clamp(-E4M3_MAX, E4M3_MAX)


def attention(query, keys, values, table, lens, scale: float, window: int, sinks: int, key_scale=None, value_scale=None):
    """(out, size) ``[batch * rows, heads, 128]``; rows that are none hold zeros."""
    batch, kv = table.shape[0], keys.shape[2]
    rows, heads = query.shape[0] // max(batch, 1), query.shape[1]
    group = heads // kv
    all_keys, all_values = keys.double(), values.double()
    out = torch.zeros(query.shape, dtype=torch.float64)
    size = torch.zeros_like(out)
    for b, n in enumerate(lens.tolist()):
        n = max(n, 0)
        tokens = min(n, table.shape[1] * PAGE)
        pages = table[b, :-(-tokens // PAGE)].long()
        real = ((pages >= 0) & (pages < keys.shape[0])).repeat_interleave(PAGE)[:tokens]
        at = pages.clamp(0, keys.shape[0] - 1)
        k, v = all_keys[at].flatten(0, 1)[:tokens], all_values[at].flatten(0, 1)[:tokens]
        if key_scale is not None:
            k, v = k * key_scale.double()[:, None], v * value_scale.double()[:, None]
        j = torch.arange(tokens)
        for t in range(rows):
            p = n - rows + t
            if p < 0:
                continue
            seen = real & (j <= p)
            if window >= 0:
                seen &= (j >= p - window) | (j < sinks)
            if not seen.any():
                continue
            r = b * rows + t
            for h in range(heads):
                score = k[seen, h // group] @ query[r, h].double() * scale
                weight = torch.softmax(score, dim=0)
                out[r, h] = weight @ v[seen, h // group]
                size[r, h] = weight @ v[seen, h // group].abs()
    return out, size
