"""Page selection of batches that decode over wide tables, against a ranking of all pages in 64 bits.

Scoring takes two tiles of 16 pages a wave once requests x KV heads x chunks of 128 pages reach 1024.
"""

from __future__ import annotations

import pytest
import torch
from oracle import pages as OP
from pages_cases import make_rows
from trianglemix import pages as TP

BF16, FP16 = torch.bfloat16, torch.float16


def ranked(query, low, high, table, lens, count, sink, recent):
    """``oracle.pages.select_pages`` of finite bounds, with the scores of a request as one product."""
    batch, kv = table.shape[0], low.shape[1]
    rows, group = query.shape[0] // batch, query.shape[1] // kv
    blocks = -(-rows // 32)
    out = torch.full((batch, blocks, kv, count), -1, dtype=torch.int32)
    low, high = low.double(), high.double()
    for b, n in enumerate(lens.tolist()):
        for i in range(blocks):
            first, last = OP.block_rows(n, rows, i)
            if last < first:
                continue
            at = b * rows + first - (max(n, 0) - rows)
            total = query[at:at + last - first + 1].double().sum(dim=0).view(kv, group, 128)
            j = torch.arange(min(table.shape[1], last // 128 + 1))
            there = (table[b, j] >= 0) & (table[b, j] < low.shape[0])
            phys = table[b, j].long() * there
            score = (total.clamp(min=0) @ high[phys].permute(1, 2, 0) + total.clamp(max=0) @ low[phys].permute(1, 2, 0))
            score = score.amax(dim=1)  # [kv, pages]
            forced = (j < sink) | ((j >= first // 128 - recent + 1) if recent > 0 else False)
            score = score.masked_fill(forced, float("inf"))[:, there]
            best = score.sort(dim=1, descending=True, stable=True).indices[:, :count].sort(dim=1).values
            out[b, i, :, :best.shape[1]] = j[there][best].to(torch.int32)
    return out


def make_batch(batch, kv_heads, cols, pages, dtype, seed):
    """(low, high, table, lens): random bounds, a third of the table's entries no page of the cache.

    Physical page 0 has by far the largest bounds and is in no request's table.
    """
    g = torch.Generator().manual_seed(seed)
    low = torch.randn(pages, kv_heads, 128, generator=g) - 1
    high = low + 2 + torch.rand(pages, kv_heads, 128, generator=g)
    low[0], high[0] = -60.0, 60.0
    table = torch.randint(1, pages, (batch, cols), generator=g).to(torch.int32)
    nothing = torch.tensor([-1, pages, -2 ** 31, 2 ** 31 - 1], dtype=torch.int32)
    bad = torch.rand(batch, cols, generator=g) < 1 / 3
    table[bad] = nothing[torch.randint(0, 4, (int(bad.sum()),), generator=g)]
    lens = torch.randint(1, cols * 128 + 1, (batch,), generator=g).to(torch.int32)
    lens[:4] = torch.tensor([cols * 128, 0, 1, 17 * 128 + 5])[:batch]
    table[0, 0] = table[0, -1] = -1  # the first and the most recent page
    table[3:4, 17] = -1
    return low.to(dtype), high.to(dtype), table, lens


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("rows,group,batch,kv_heads,cols", [
    (1, 1, 32, 8, 512), (1, 2, 64, 4, 500), (1, 4, 32, 8, 512), (1, 3, 64, 8, 300),  # decoding, 1 to 4 heads a group
    (3, 4, 32, 8, 512), (32, 1, 64, 8, 257),                                        # one block of several rows
    (40, 2, 32, 8, 512), (128, 1, 64, 4, 512),                                      # two blocks, four
])
def test_pages_that_are_none_in_every_tile(gpu, dtype, rows, group, batch, kv_heads, cols):
    print(f"select two tiles {rows} {group} {batch} {kv_heads} {cols} {dtype}", flush=True)
    assert -(-cols // 128) * kv_heads * batch >= 1024
    low, high, table, lens = make_batch(batch, kv_heads, cols, 900, dtype, seed=rows + group + cols)
    query = make_rows(batch * rows, group * kv_heads, dtype, 3)
    for count, sink, recent in ((16, 1, 1), (9, 3, 4)):
        want = ranked(query, low, high, table, lens, count, sink, recent)
        got = TP.select_pages(query.to(gpu), low.to(gpu), high.to(gpu), table.to(gpu), lens.to(gpu), count,
                              sink_pages=sink, recent_pages=recent).cpu()
        assert torch.equal(got, want), f"{int((got != want).any(dim=-1).sum())} of {got[..., 0].numel()} selections differ"


def test_ranking_equals_the_oracle():
    """The ranking above, on a small case, against the oracle's own loop."""
    low, high, table, lens = make_batch(4, 2, 20, 30, BF16, seed=1)
    for rows in (1, 5, 40):
        query = make_rows(4 * rows, 6, BF16, 2)
        assert torch.equal(ranked(query, low, high, table, lens, 6, 1, 2),
                           OP.select_pages(query, low, high, table, lens, 6, 1, 2))


@pytest.mark.gpu
@pytest.mark.parametrize("batch,rows,heads,kv_heads", [
    (64, 1, 8, 8),     # 40 requests, then 24
    (24, 40, 16, 8),   # pooled rows: 19 requests of two blocks, then 5
    (2, 1607, 16, 8),  # one request's 51 blocks: 39, then 12, with seven rows in the last one; then the other request's
])
def test_calls_of_several_slabs(gpu, batch, rows, heads, kv_heads):
    """Scores past the workspace's 40 MiB: several launches over it, each with its part of the requests and blocks."""
    from trianglemix import cabi

    print(f"select slabs {batch} {rows} {heads} {kv_heads}", flush=True)
    cols, blocks = 16384, -(-rows // 32)
    each = kv_heads * cols * 8 + (heads * 128 * 8 if rows > 1 else 0)
    assert batch * blocks * each > 40 << 20
    assert cabi.load_hip_library().tm_select_pages_workspace_size(batch, rows, heads, kv_heads, cols) <= 40 << 20
    low, high, table, _ = make_batch(batch, kv_heads, cols, 900, BF16, seed=rows)
    g = torch.Generator().manual_seed(rows)
    lens = torch.randint(1, 60 * 128, (batch,), generator=g).to(torch.int32)
    lens[-1] = 130 * 128 + 77
    query = make_rows(batch * rows, heads, BF16, 4)
    want = ranked(query, low, high, table, lens, 12, 1, 1)
    out = torch.full_like(want, 7, device=gpu)
    TP.select_pages(query.to(gpu), low.to(gpu), high.to(gpu), table.to(gpu), lens.to(gpu), 12, out=out)
    assert torch.equal(out.cpu(), want)
    assert all(not torch.equal(want[0], want[b]) for b in range(1, batch))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("rows,group", [(1, 1), (1, 3), (33, 2), (70, 8), (1, 32)])
def test_equal_pages_beside_odd_bounds(gpu, dtype, rows, group):
    """Two logical pages with the same bounds have the same score, also where sums round and a neighbour is infinite."""
    print(f"select equal pages {rows} {group} {dtype}", flush=True)
    batch, kv, cols, pages = 32, 8, 64, 8
    g = torch.Generator().manual_seed(rows + group)

    def wide(*shape, bits):  # values of many magnitudes: their products' sum takes more than 53 bits
        return torch.randn(*shape, generator=g) * 2.0 ** torch.randint(-bits, bits + 1, shape, generator=g)

    bits = 7 if dtype == FP16 else 25
    low, high = wide(pages, kv, 128, bits=bits), wide(pages, kv, 128, bits=bits)
    low, high = torch.minimum(low, high).to(dtype), torch.maximum(low, high).to(dtype)
    low[1:], high[1:] = 0, 0
    low[0] -= 1
    high[0] += 1
    high[2, :, 5] = float("inf")
    query = wide(batch * rows, group * kv, 128, bits=bits).to(dtype)
    query[..., 5] = -query[..., 5].abs() - 0.25  # takes the lower bound there, which is zero
    table = torch.ones(batch, cols, dtype=torch.int32)
    table[:, 3] = table[:, 40] = 0
    table[:, 41] = 2
    lens = torch.full((batch,), cols * 128, dtype=torch.int32)
    got = TP.select_pages(query.to(gpu), low.to(gpu), high.to(gpu), table.to(gpu), lens.to(gpu), 1 if rows == 1 else 3,
                          sink_pages=0, recent_pages=0).cpu()
    # where the sum of page 0's terms is negative, the pages without bounds of their own come first: 0, 1, 2
    first = (got == 3).any(dim=-1)
    assert first.float().mean() > 0.8
    assert not ((got == 40).any(dim=-1) & ~first).any()
    one = TP.select_pages(query.to(gpu), low.to(gpu), high.to(gpu), table.to(gpu), lens.to(gpu), 1, sink_pages=0,
                          recent_pages=0).cpu()[..., 0]
    assert not (one == 40).any(), f"page 40 before page 3 in {int((one == 40).sum())} of {one.numel()} selections"
