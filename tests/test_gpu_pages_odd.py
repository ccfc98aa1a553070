"""Paged serving operators: scores of -infinity, and pages that requests share."""

from __future__ import annotations

import pytest
import torch
from oracle import pages as OP
from pages_cases import SCALE, make_cache, make_rows, tolerance
from trianglemix import pages as TP
from trianglemix import tree as TT

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def ints(x, device="cpu"):
    return torch.tensor(x, dtype=torch.int32, device=device)


def check(got, want, size, values, keys, dtype):
    """Rows whose scores are all -infinity (no number in the oracle) give zeros."""
    nothing = want.isnan()
    got = got.cpu().double()
    assert (got[nothing] == 0).all()
    off = (got - want).abs()[~nothing]
    tol = tolerance(want, size, values, keys, dtype)[~nothing]
    assert bool((off <= tol).all()), f"off by {(off / tol.clamp(min=1e-30)).max():.2f} of the tolerance"
    return nothing


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("length,rows,heads,kv", [
    (1, 1, 4, 1), (300, 1, 8, 1), (300, 4, 8, 1),              # groups of 4, 8 and 32 rows
    (200, 200, 4, 1), (200, 200, 16, 1), (150, 150, 128, 64),  # 128 and 512 rows; two workgroups a CU
])
def test_scores_of_minus_infinity_selected(gpu, dtype, length, rows, heads, kv):
    print(f"attend -inf {length} {rows} {heads}/{kv} {dtype}", flush=True)
    keys, values, table = make_cache([length], kv, dtype, seed=31)
    query = make_rows(rows, heads, dtype, 32)
    query[..., 0] = query[..., 0].abs() + 0.5
    for token in [0, *range(5, 70), 129]:  # a row's only key, whole tiles, single keys
        if token < length:
            keys[table[0, token // 128].item(), token % 128, :, 0] = -float("inf")
    count = -(-length // 128)
    pages = torch.arange(count, dtype=torch.int32).expand(1, -(-rows // 32), kv, count).contiguous()
    want, size, _ = OP.selected_attention(query, keys, values, table, ints([length]), pages, SCALE,
                                          torch.zeros_like(query))
    got = TP.selected_page_attention(query.to(gpu), keys.to(gpu), values.to(gpu), table.to(gpu), ints([length], gpu),
                                     pages.to(gpu), SCALE)
    nothing = check(got, want, size, values, length, dtype)
    assert nothing[0].all() == (rows == length) and not nothing[1:].any()


@pytest.mark.parametrize("nodes,heads", [(3, 4), (40, 4), (60, 8)])
def test_scores_of_minus_infinity_tree(gpu, nodes, heads):
    print(f"tree -inf {nodes} {heads}", flush=True)
    keys, values, table = make_cache([0], 1, BF16, seed=41)
    query, key, value = make_rows(nodes, heads, BF16, 42), make_rows(nodes, 1, BF16, 43), make_rows(nodes, 1, BF16, 44)
    query[..., 0] = query[..., 0].abs() + 0.5
    key[0, :, 0] = -float("inf")  # the first node attends nothing else
    mask = torch.tensor(TT.ancestor_masks([-1] + [i // 2 for i in range(nodes - 1)]), dtype=torch.int64)
    offsets = ints([0, nodes])
    want, size, _ = OP.tree_attention(query, key, value, keys, values, table, ints([0]), offsets, mask, SCALE,
                                      torch.zeros_like(query))
    got = TT.tree_attention(*(t.to(gpu) for t in (query, key, value, keys, values, table, ints([0]), offsets, mask)), SCALE)
    nothing = check(got, want, size, value, nodes, BF16)
    assert nothing[0].all() and not nothing[1:].any()


def test_requests_that_share_a_prefix(gpu):
    """Full pages in several tables of one batch, all updated, selected and attended at once."""
    print("shared prefix", flush=True)
    lens = [700, 400, 389, 384]
    keys, values, table = make_cache(lens, 2, BF16, seed=51)
    table[1:, :3] = table[0, :3]  # 384 tokens
    low, high = TP.page_bounds_like(keys)
    want = OP.page_bounds(keys, table, ints(lens), 1000, low, high)
    query = make_rows(4, 8, BF16, 52)
    chosen = OP.select_pages(query, *want, table, ints(lens), 3, 1, 1)
    low, high, lens_d = low.to(gpu), high.to(gpu), ints(lens, gpu)
    keys_d, values_d, table_d, query_d = keys.to(gpu), values.to(gpu), table.to(gpu), query.to(gpu)
    TP.update_page_bounds(keys_d, table_d, lens_d, 1000, low, high)
    assert torch.equal(low.cpu(), want[0]) and torch.equal(high.cpu(), want[1])
    picked = TP.select_pages(query_d, low, high, table_d, lens_d, 3)
    assert torch.equal(picked.cpu(), chosen)
    out, size, _ = OP.selected_attention(query, keys, values, table, ints(lens), chosen, SCALE, torch.zeros_like(query))
    got = TP.selected_page_attention(query_d, keys_d, values_d, table_d, lens_d, picked, SCALE)
    check(got, out, size, values, 384, BF16)
