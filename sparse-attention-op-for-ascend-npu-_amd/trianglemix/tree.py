"""Attention of drafted tokens over a paged KV cache: the verification step of speculative decoding.

``tree_attention`` computes, for a batch of requests with one draft tree each, the attention of every node over its
request's cache and over the nodes of the tree that its mask names.  The drafts' K and V are read from the projection's
output, not from the cache: once the accepted path is known, ``cache.reshape_and_cache`` writes its rows (the rejected
ones with slot -1).  A tree of one node is a decoding step.  ``include/trianglemix_pages.h`` states every rule.
"""

from __future__ import annotations

from collections.abc import Sequence

MAX_TREE_NODES = 64


def ancestor_masks(parents: Sequence[int]) -> list[int]:
    """Mask words of one tree: bit j of entry i is set where node j is node i or one of its ancestors.

    ``parents[i]`` is the parent of node i, an earlier node, or -1 for a node that follows the context directly.  The
    words are signed, as an int64 tensor holds them.
    """
    if len(parents) > MAX_TREE_NODES:
        raise ValueError(f"a draft tree has at most {MAX_TREE_NODES} nodes")
    words: list[int] = []
    for node, parent in enumerate(parents):
        if not -1 <= parent < node:
            raise ValueError("a node's parent must be -1 or an earlier node")
        words.append((words[parent] if parent >= 0 else 0) | 1 << node)
    return [word - (1 << 64) if word >> 63 else word for word in words]


def tree_attention(query, key, value, key_cache, value_cache, block_table, context_lens, tree_offsets, tree_mask,
                   softmax_scale: float, *, out=None):
    """Attention of the nodes ``tree_offsets[b] .. tree_offsets[b + 1] - 1`` of each request b.

    ``query [nodes, heads, 128]``, ``key`` / ``value [nodes, kv_heads, 128]`` (row-strided views allowed),
    ``context_lens [batch]`` and ``tree_offsets [batch + 1]`` int32, ``tree_mask [nodes]`` int64 (``ancestor_masks``).
    Rows of ``out`` that are no node keep what they hold (zeros without ``out``).
    """
    import torch

    from .native import require_adapter

    require_adapter()  # no CPU fallback: fails loudly without the native library
    op = torch.ops.trianglemix.tree_attention
    args = (query, key, value, key_cache, value_cache, block_table, context_lens, tree_offsets, tree_mask, softmax_scale)
    return op(*args) if out is None else op.out(*args, out=out)
