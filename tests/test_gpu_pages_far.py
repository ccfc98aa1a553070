"""The paged serving operators over caches larger than 4 GiB, with runs of hundreds of pages a workgroup.

1024 logical pages stand for 16 physical ones near the end of a cache of 6 GiB, 64 in a row for each: the softmax over
them is the softmax over the 16, which a plain product in 64 bits gives.  A page of the wrong 64 shows, as the values of
each physical page lie around a mean of its own.
"""

from __future__ import annotations

import pytest
import torch
from pages_cases import SCALE, make_rows, tolerance
from trianglemix import pages as TP
from trianglemix import tree as TT

pytestmark = pytest.mark.gpu
KV, HEADS, PAGES, REAL, EACH = 64, 128, 3000, 16, 64
LENGTH = REAL * EACH * 128


@pytest.fixture(scope="module")
def far(gpu):
    g = torch.Generator(device=gpu).manual_seed(3)
    keys = torch.empty(PAGES, 128, KV, 128, dtype=torch.bfloat16, device=gpu)
    values = torch.empty_like(keys)
    at = PAGES - 1 - 2 * torch.randperm(REAL, generator=g, device=gpu)
    assert int(at.min()) * keys.stride(0) * 2 > 1 << 32
    keys[at] = torch.randn(REAL, 128, KV, 128, generator=g, device=gpu).bfloat16()
    mean = torch.randn(REAL, 1, 1, 128, generator=g, device=gpu)
    values[at] = (torch.randn(REAL, 128, KV, 128, generator=g, device=gpu) + mean).bfloat16()
    table = at.repeat_interleave(EACH).to(torch.int32)
    table = torch.cat([table, torch.full((3,), -1, dtype=torch.int32, device=gpu)])[None].contiguous()
    return keys, values, table, at


def check(got, query, far):
    keys, values, _, at = far
    for head in (0, 1, 62, 63, 126, 127):
        k, v = (x[at, :, head // 2].reshape(-1, 128).double().cpu() for x in (keys, values))
        w = torch.softmax(query[:, head].double() @ k.t() * SCALE, dim=1)
        want = w @ v
        tol = tolerance(want, w @ v.abs(), v, LENGTH, torch.bfloat16)
        assert bool(((got[:, head].cpu().double() - want).abs() <= tol).all()), head


@pytest.mark.parametrize("rows", [1, 20, 64])  # 2, 40 and twice 64 rows a group
def test_selected_pages(gpu, far, rows):
    print(f"far pages {rows}", flush=True)
    keys, values, table, _ = far
    query = make_rows(rows, HEADS, torch.bfloat16, 4)
    lens = torch.tensor([LENGTH + 200], dtype=torch.int32, device=gpu)
    chosen = torch.arange(REAL * EACH, dtype=torch.int32, device=gpu).expand(1, -(-rows // 32), KV, -1).contiguous()
    check(TP.selected_page_attention(query.to(gpu), keys, values, table, lens, chosen, SCALE), query, far)


@pytest.mark.parametrize("nodes", [1, 16, 20])  # 2, 32 and 40 rows a group
def test_trees(gpu, far, nodes):
    print(f"far trees {nodes}", flush=True)
    keys, values, table, _ = far
    query = make_rows(nodes, HEADS, torch.bfloat16, 5)
    draft = torch.full((nodes, KV, 128), float("nan"), dtype=torch.bfloat16, device=gpu)  # attended by no node
    context = torch.tensor([LENGTH], dtype=torch.int32, device=gpu)
    offsets = torch.tensor([0, nodes], dtype=torch.int32, device=gpu)
    mask = torch.zeros(nodes, dtype=torch.int64, device=gpu)
    check(TT.tree_attention(query.to(gpu), draft, draft, keys, values, table, context, offsets, mask, SCALE), query, far)


def test_bounds(gpu, far):
    print("far bounds", flush=True)
    keys, _, table, at = far
    low, high = TP.page_bounds_like(keys)
    lens = torch.tensor([LENGTH], dtype=torch.int32, device=gpu)
    TP.update_page_bounds(keys, table, lens, LENGTH, low, high)
    assert torch.equal(low[at], keys[at].amin(dim=1)) and torch.equal(high[at], keys[at].amax(dim=1))
    low[at] = high[at] = 0
    assert not low.any() and not high.any()
