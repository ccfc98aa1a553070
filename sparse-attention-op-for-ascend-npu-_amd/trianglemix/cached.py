"""Attention over a paged cache of 8-bit or 16-bit numbers: decoding steps, verification of drafts, whole chunks.

``rotary.rotate_and_cache`` fills the cache, ``cached_attention`` reads it: the last ``rows`` tokens of each request attend
causally over its pages, all of them or a window behind the first few tokens.  An 8-bit cache
(``torch.float8_e4m3fn``) holds e4m3 numbers with one fp32 scale for each KV head of K and of V: half the memory and
half the traffic of a 16-bit one.  The package's other operators (the sparse prefill and its dense companion, the
cache write, page selection, trees) take 16-bit caches alone: ``new_cache(..., dtype=torch.bfloat16)`` makes one
that both can use.  ``block_table`` and ``seq_lens`` are int32 on the GPU and are read there: a captured
call can be replayed with others.  ``include/trianglemix_cached.h`` states every rule.
"""

from __future__ import annotations

PAGE_SIZE = 128
E4M3_MAX = 448.0


def new_cache(num_pages: int, kv_heads: int, dtype=None, *, device=None):
    """(key_cache, value_cache) ``[num_pages, 128, kv_heads, 128]`` of zeros; default type ``torch.float8_e4m3fn``."""
    import torch

    shape = (num_pages, PAGE_SIZE, kv_heads, 128)
    dtype = torch.float8_e4m3fn if dtype is None else dtype
    return torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device)


def head_scales(rows, margin: float = 1.0):
    """fp32 ``[kv_heads]`` scales that give the largest finite number of each head of ``rows [tokens, kv_heads, 128]``,
    times ``margin``, the largest of an 8-bit cache; 1 for a head of zeros (and of numbers too small for a normal scale)."""
    import torch

    size = rows.detach().abs()
    largest = size.masked_fill(~size.isfinite(), 0.0).amax(dim=(0, 2)).float() * (margin / E4M3_MAX)
    normal = largest >= torch.finfo(torch.float32).tiny
    return torch.where(normal, largest.clamp(max=2.0 ** 126), torch.ones_like(largest)).contiguous()


def cached_attention(query, key_cache, value_cache, block_table, seq_lens, softmax_scale: float, *, window: int = -1,
                     sinks: int = 0, key_scale=None, value_scale=None, out=None):
    """Attention of ``query [batch * rows, heads, 128]``, the last ``rows`` tokens of each request.

    ``window``: keys in front of its own position that a row attends, -1 for all; ``sinks``: the first keys, attended
    besides.  ``out`` keeps its rows at negative positions (zeros without it).
    """
    import torch

    from .native import require_adapter

    require_adapter()  # no CPU fallback: fails loudly without the native library
    op = torch.ops.trianglemix.cached_attention
    args = (query, key_cache, value_cache, block_table, seq_lens, softmax_scale, window, sinks, key_scale, value_scale)
    return op(*args) if out is None else op.out(*args, out=out)
