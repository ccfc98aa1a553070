"""The paged serving operators at their limits: 1024 requests, 256 heads, 32 heads a group, trees of 64 nodes."""

from __future__ import annotations

import pytest
import torch
from oracle import pages as OP
from pages_cases import SCALE, make_cache, make_rows, tolerance
from test_gpu_tree import check as check_tree
from test_gpu_tree import make_trees
from trianglemix import pages as TP

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def ints(x, device="cpu"):
    return torch.tensor(x, dtype=torch.int32, device=device)


@pytest.mark.parametrize("lens,rows,heads,kv_heads,count", [
    ([(37 * b) % 300 for b in range(1024)], 1, 2, 1, 2),
    ([(53 * b) % 200 for b in range(1024)], 3, 1, 1, 3),
    ([300, 129], 1, 256, 256, 2),
    ([300], 2, 256, 8, 2),
    ([500], 33, 32, 1, 3),  # 1024 rows a group and 32
])
def test_pages(gpu, lens, rows, heads, kv_heads, count):
    print(f"limits {len(lens)} {rows} {heads}/{kv_heads}", flush=True)
    keys, values, table = make_cache(lens, kv_heads, BF16, seed=rows + heads)
    query = make_rows(len(lens) * rows, heads, BF16, 5)
    low, high = TP.page_bounds_like(keys)
    bounds = OP.page_bounds(keys, table, ints(lens), 1000, low, high)
    chosen = OP.select_pages(query, *bounds, table, ints(lens), count, 1, 0)
    want, size, written = OP.selected_attention(query, keys, values, table, ints(lens), chosen, SCALE,
                                                torch.zeros_like(query))
    keys_d, table_d, lens_d, query_d, low, high = (t.to(gpu) for t in (keys, table, ints(lens), query, low, high))
    TP.update_page_bounds(keys_d, table_d, lens_d, 1000, low, high)
    assert torch.equal(low.cpu(), bounds[0]) and torch.equal(high.cpu(), bounds[1])
    picked = TP.select_pages(query_d, low, high, table_d, lens_d, count, sink_pages=1, recent_pages=0)
    assert torch.equal(picked.cpu(), chosen)
    got = TP.selected_page_attention(query_d, keys_d, values.to(gpu), table_d, lens_d, picked, SCALE).cpu().double()
    assert (got[~written] == 0).all()
    assert bool(((got - want).abs() <= tolerance(want, size, values, 500, BF16)).all())


@pytest.mark.parametrize("contexts,sizes,heads,kv_heads", [
    ([(29 * b) % 140 for b in range(1024)], [b % 3 for b in range(1024)], 2, 1),
    ([129, 5], [3, 1], 256, 256),
    ([300, 0, 128], [64, 1, 2], 32, 1),  # 2048 rows a group
])
def test_trees(gpu, contexts, sizes, heads, kv_heads):
    print(f"limits trees {len(sizes)} {heads}/{kv_heads}", flush=True)
    keys, values, table = make_cache(contexts, kv_heads, BF16, seed=heads)
    offsets, mask = make_trees(sizes, 6)
    qkv = make_rows(int(offsets[-1]), heads + 2 * kv_heads, BF16, 7)
    check_tree(gpu, qkv, heads, kv_heads, keys, values, table, contexts, offsets, mask, max(contexts))
