"""Attention over selected pages of a paged KV cache.

For requests whose context is much longer than what their queries need: after a step's K rows are in their pages
(``cache.write_chunk_kv``, ``cache.reshape_and_cache``),

1. ``update_page_bounds`` brings the elementwise smallest and largest key of the pages it wrote to up to date;
2. ``select_pages`` picks, for each block of 32 query rows and each KV head, the pages whose bounds promise the
   largest dot products with the block's summed queries, next to the first and the most recent pages;
3. ``selected_page_attention`` attends causally over those pages alone.

A batch is ``query [batch * rows, heads, 128]`` with the last ``rows`` tokens of each request: a prefill chunk is one
request with many rows, a decoding step many requests with one row.  ``block_table [batch, max_pages]`` and ``seq_lens
[batch]`` are int32 on the GPU and are read there: a captured call can be replayed with others.  Heads of 128 dims,
pages of 128 tokens, bf16 or fp16, any number of query heads per KV head up to 32.  The operators are
``torch.ops.trianglemix`` ones; ``include/trianglemix_pages.h`` is their C ABI and states every rule.
"""

from __future__ import annotations

SELECT_ROWS = 32  # query rows that share one selection


def page_bounds_like(key_cache):
    """Bounds buffers ``[pages, kv_heads, 128]`` for a key cache, of no page yet."""
    shape = (key_cache.shape[0], *key_cache.shape[2:])
    return key_cache.new_zeros(shape), key_cache.new_zeros(shape)


def update_page_bounds(key_cache, block_table, seq_lens, num_tokens: int, page_min, page_max) -> None:
    """Key bounds of the pages that hold the last ``num_tokens`` tokens of each request."""
    import torch

    from .native import require_adapter

    require_adapter()  # no CPU fallback: fails loudly without the native library
    torch.ops.trianglemix.update_page_bounds(key_cache, block_table, seq_lens, num_tokens, page_min, page_max)


def select_pages(query, page_min, page_max, block_table, seq_lens, count: int, *, sink_pages: int = 1,
                 recent_pages: int = 1, out=None):
    """int32 ``[batch, ceil(rows / 32), kv_heads, count]``: logical pages in ascending order, -1 behind them."""
    import torch

    from .native import require_adapter

    require_adapter()
    op = torch.ops.trianglemix.select_pages
    if out is None:
        return op(query, page_min, page_max, block_table, seq_lens, count, sink_pages, recent_pages)
    return op.out(query, page_min, page_max, block_table, seq_lens, count, sink_pages, recent_pages, out=out)


def selected_page_attention(query, key_cache, value_cache, block_table, seq_lens, pages, softmax_scale: float, *,
                            out=None):
    """Causal attention over the listed pages; ``out`` keeps its rows at negative positions (zeros without it)."""
    import torch

    from .native import require_adapter

    require_adapter()
    op = torch.ops.trianglemix.selected_page_attention
    if out is None:
        return op(query, key_cache, value_cache, block_table, seq_lens, pages, softmax_scale)
    return op.out(query, key_cache, value_cache, block_table, seq_lens, pages, softmax_scale, out=out)
