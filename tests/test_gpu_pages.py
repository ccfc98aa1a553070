"""Page bounds, page selection and attention over selected pages against the 64-bit oracle.

Bounds and selections are compared exactly, attention within the rounding of its type (``pages_cases.tolerance``).
"""

from __future__ import annotations

import pytest
import torch

from oracle import pages as OP
from pages_cases import SCALE, make_cache, make_rows, to_gpu, tolerance
from trianglemix import pages as TP

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def ints(x, device="cpu"):
    return torch.tensor(x, dtype=torch.int32, device=device)


def same(a, b):
    """Equal as floating values, NaNs alike."""
    return torch.equal(a.float().nan_to_num(nan=12345.0), b.float().nan_to_num(nan=12345.0))


# ---- bounds ----

@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("lens,num_tokens,kv_heads", [
    ([1], 1, 8), ([128, 129, 127, 0], 1, 8), ([300, 5, 640], 2, 4), ([777], 300, 3), ([1000], 2000, 1),
    ([130, 512, 256, 257], 130, 2)])
def test_bounds(gpu, dtype, lens, num_tokens, kv_heads):
    print(f"bounds {lens} {num_tokens} {kv_heads} {dtype}", flush=True)
    keys, _, table = make_cache(lens, kv_heads, dtype, seed=len(lens) * 7 + num_tokens)
    low, high = make_rows(keys.shape[0], kv_heads, dtype, 1), make_rows(keys.shape[0], kv_heads, dtype, 2)
    want = OP.page_bounds(keys, table, ints(lens), num_tokens, low, high)
    low_d, high_d = low.to(gpu), high.to(gpu)
    TP.update_page_bounds(keys.to(gpu), table.to(gpu), ints(lens, gpu), num_tokens, low_d, high_d)
    assert same(low_d.cpu(), want[0]) and same(high_d.cpu(), want[1])


def test_bounds_of_odd_values_and_bad_pages(gpu):
    lens = [300, 400, 260]
    keys, _, table = make_cache(lens, 2, BF16, seed=5, stride_pages=True)
    keys[table[0, 1].item(), 7, 0, 3] = float("nan")
    keys[table[0, 1].item(), 9, 1, 4] = -float("nan")
    keys[table[0, 2].item(), 43, 0, 5] = float("inf")
    keys[table[0, 2].item(), 42, 0, 6] = -float("inf")
    keys[table[0, 2].item(), 44:] = float("nan")  # behind the request's last token
    table[1, 1] = -3
    table[1, 2] = keys.shape[0]
    lens[2] = 5000  # past the table: only its pages exist
    low, high = TP.page_bounds_like(keys.contiguous())
    want = OP.page_bounds(keys, table, ints(lens), 300, low, high)
    low_d, high_d = low.to(gpu), high.to(gpu)
    TP.update_page_bounds(to_gpu(keys, gpu), table.to(gpu), ints(lens, gpu), 300, low_d, high_d)
    assert same(low_d.cpu(), want[0]) and same(high_d.cpu(), want[1])
    assert torch.isnan(want[0]).sum() == 2


# ---- selection ----

def bounds_of(keys, table, lens):
    low, high = TP.page_bounds_like(keys)
    return OP.page_bounds(keys, table, ints(lens), 1 << 20, low, high)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("lens,rows,heads,kv_heads,count,sink,recent", [
    ([1], 1, 4, 1, 4, 1, 1),
    ([3000, 1, 0, 1500, 128], 1, 8, 2, 5, 1, 1),
    ([3000, 1, 0, 1500, 129], 1, 8, 2, 6, 0, 0),
    ([2900, 700], 5, 14, 2, 7, 2, 2),
    ([3333], 32, 4, 4, 4, 1, 2),
    ([3333], 33, 8, 1, 9, 1, 1),
    ([140], 140, 8, 2, 3, 1, 1),
    ([70, 20], 100, 4, 2, 3, 0, 1),   # more rows than tokens: the first ones are none
    ([4000], 200, 8, 2, 64, 1, 1),    # fewer pages than wanted
    ([40000], 64, 4, 1, 40, 2, 3),
])
def test_select(gpu, dtype, lens, rows, heads, kv_heads, count, sink, recent):
    print(f"select {lens} {rows} {heads}/{kv_heads} {count} {sink} {recent} {dtype}", flush=True)
    keys, _, table = make_cache(lens, kv_heads, dtype, seed=rows + count)
    low, high = bounds_of(keys, table, lens)
    query = make_rows(len(lens) * rows, heads, dtype, 3)
    want = OP.select_pages(query, low, high, table, ints(lens), count, sink, recent)
    got = TP.select_pages(query.to(gpu), low.to(gpu), high.to(gpu), table.to(gpu), ints(lens, gpu), count,
                          sink_pages=sink, recent_pages=recent)
    assert torch.equal(got.cpu(), want)


def test_select_ties_bad_pages_and_odd_bounds(gpu):
    lens = [128 * 40, 128 * 40]
    keys, _, table = make_cache(lens, 2, BF16, seed=9)
    low, high = bounds_of(keys, table, lens)
    # equal pages: pages 5 .. 24 of request 0 all have the bounds of page 5
    same_as = table[0, 5].item()
    for j in range(6, 25):
        low[table[0, j].item()], high[table[0, j].item()] = low[same_as], high[same_as]
    high[table[0, 30].item(), :, 1] = float("nan")
    high[table[0, 31].item(), :, 2] = float("inf")
    low[table[0, 31].item(), :, 2] = -float("inf")
    table[1, 3], table[1, 4], table[1, 39] = -1, keys.shape[0], -7
    wide = torch.zeros(2, 12, 128, dtype=BF16)
    wide[:, 2:10] = make_rows(2, 8, BF16, 4)
    query = wide[:, 2:10]  # a slice of a fused buffer
    table_wide = torch.full((2, 2 * table.shape[1]), 99999, dtype=torch.int32)
    table_wide[:, :table.shape[1]] = table
    query_d = wide.to(gpu)[:, 2:10]
    table_d = table_wide.to(gpu)[:, :table.shape[1]]
    for count in (1, 4, 16, 22, 38, 40, 60):
        want = OP.select_pages(query, low, high, table, ints(lens), count, 0, 0)
        got = torch.full_like(want, 7).to(gpu)
        TP.select_pages(query_d, low.to(gpu), high.to(gpu), table_d, ints(lens, gpu), count, sink_pages=0,
                        recent_pages=0, out=got)
        assert torch.equal(got.cpu(), want), count


@pytest.mark.parametrize("cols", [1024, 1025, 4096, 4097, 16384])
def test_select_wide_tables(gpu, cols):
    """Tables on either side of the sizes at which the kernels change, with few tokens and with all of them."""
    print(f"select wide {cols}", flush=True)
    g = torch.Generator().manual_seed(cols)
    pages = 600
    low = torch.randn(pages, 1, 128, generator=g).to(BF16)
    high = (low.float() + 1 + torch.rand(pages, 1, 128, generator=g)).to(BF16)
    table = torch.randint(0, pages, (2, cols), generator=g).to(torch.int32)  # pages shared: many equal scores
    lens = ints([cols * 128, 5 * 128 + 3])
    query = make_rows(2, 4, BF16, 8)
    # the oracle's loop over all pages takes too long: rank the pages here
    got = TP.select_pages(query.to(gpu), low.to(gpu), high.to(gpu), table.to(gpu), lens.to(gpu), 48, sink_pages=1,
                          recent_pages=2).cpu()
    small = OP.select_pages(query[1:], low, high, table[1:], lens[1:], 48, 1, 2)
    assert torch.equal(got[1:], small)
    q = query[0].double()
    per_page = torch.stack([torch.where(q[h] >= 0, q[h] * high[:, 0].double(), q[h] * low[:, 0].double()).sum(dim=1)
                            for h in range(4)]).amax(dim=0)
    score = per_page[table[0].long()]
    score[:1] = score[-2:] = float("inf")
    want = score.sort(descending=True, stable=True).indices[:48].sort().values
    assert torch.equal(got[0, 0, 0], want.to(torch.int32))


# ---- attention ----

def random_lists(lens, rows, kv_heads, count, seed, shuffle=False):
    g = torch.Generator().manual_seed(seed)
    blocks = -(-rows // 32)
    out = torch.full((len(lens), blocks, kv_heads, count), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        for i in range(blocks):
            first, last = OP.block_rows(n, rows, i)
            if last < first:
                continue
            for h in range(kv_heads):
                own = list(range(first // 128, last // 128 + 1))
                others = torch.randperm(last // 128 + 1, generator=g).tolist()
                chosen = (own + [j for j in others if j not in own])[:count]
                chosen = chosen if shuffle else sorted(chosen)
                out[b, i, h, :len(chosen)] = torch.tensor(chosen, dtype=torch.int32)
    return out


def check_attention(gpu, query, keys, values, table, lens, pages, query_d=None):
    dtype = query.dtype
    out = make_rows(query.shape[0], query.shape[1], dtype, 77)
    want, size, written = OP.selected_attention(query, keys, values, table, ints(lens), pages, SCALE, out)
    out_d = out.to(gpu)
    TP.selected_page_attention(query.to(gpu) if query_d is None else query_d, to_gpu(keys, gpu), to_gpu(values, gpu),
                               table.to(gpu), ints(lens, gpu), pages.to(gpu), SCALE, out=out_d)
    got = out_d.cpu()
    assert torch.equal(got[~written], out[~written])  # what is no row is left as it was
    real = values[values.isfinite()]
    tol = tolerance(want, size, real, pages.shape[-1] * 128, dtype)
    off = (got.double() - want).abs()[written]
    assert bool((off <= tol[written]).all()), f"off by {(off / tol[written].clamp(min=1e-30)).max():.2f} of the tolerance"
    return got


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("lens,rows,heads,kv_heads,count", [
    ([1], 1, 4, 1, 1),
    ([1, 128, 129, 0, 777], 1, 8, 2, 3),
    ([900, 1300], 1, 32, 8, 7),
    ([5000], 1, 7, 1, 30),             # seven heads a group
    ([700, 701, 702], 2, 16, 2, 4),    # 16 rows
    ([600], 5, 8, 2, 4),               # 20 rows of 32
    ([650], 15, 4, 1, 5),              # 60 rows of 64
    ([1000], 29, 4, 1, 8),             # 116 rows of 128
    ([1000], 31, 16, 2, 6),            # 248 rows of 256
    ([700], 32, 16, 1, 4),             # 512 rows: two row parts
    ([900], 40, 20, 1, 4),             # 640 and 160 rows: three row parts, the last block has two
    ([530], 100, 4, 4, 3),             # one head a group
    ([1111], 70, 4, 2, 6),
    ([300], 300, 4, 1, 3),             # a whole prompt
    ([50, 10, 0], 64, 4, 1, 2),        # more rows than tokens
    ([900], 260, 32, 8, 64),           # 128 rows, lists longer than the table
    ([700, 3, 1025, 40], 64, 24, 8, 64),  # 96 rows of 128
    ([8300], 40, 8, 4, 1024),          # 64 rows, lists of 65 pages
    ([700], 260, 128, 64, 5),          # 576 groups: two workgroups a CU, split groups
    ([400, 3], 130, 128, 64, 3),       # 640 groups in one piece each, the second request's mostly without rows
])
def test_attention(gpu, dtype, lens, rows, heads, kv_heads, count):
    print(f"attend {lens} {rows} {heads}/{kv_heads} {count} {dtype}", flush=True)
    keys, values, table = make_cache(lens, kv_heads, dtype, seed=rows * 3 + count)
    query = make_rows(len(lens) * rows, heads, dtype, 5)
    check_attention(gpu, query, keys, values, table, lens, random_lists(lens, rows, kv_heads, count, seed=rows))


def test_lists_in_any_form(gpu):
    """Shuffled, repeated, negative, too large and empty lists; strided pages, query rows and table rows."""
    lens, rows, kv_heads = [1500, 900, 640], 3, 2
    keys, values, table = make_cache(lens, kv_heads, BF16, seed=11, stride_pages=True)
    wide = torch.zeros(9, 12, 128, dtype=BF16)
    wide[:, :8] = make_rows(9, 8, BF16, 6)
    query = wide[:, :8]
    pages = random_lists(lens, rows, kv_heads, 9, seed=12, shuffle=True)
    pages[0, 0, 0] = ints([3, 3, 11, -1, 0, 11, 3, 700, -2147483648])
    pages[0, 0, 1] = ints([11, 2147483647, 12, 5, -5, 4, 4, 4, 16384])
    pages[1, 0, 0] = -1           # nothing: zeros
    pages[1, 0, 1] = ints([1, 2, 3, 5, 7, -1, 6, 200, 6])  # ascending at first only
    pages[2, 0, 0] = ints([0, 1, 2, 5, 6, 7, 8, 9, 10])    # ascending, what is no page behind
    pages[2, 0, 1] = ints([7, 6, 5, 5, 5, 5, 5, 5, 5])     # the block's own page is not among them
    got = check_attention(gpu, query, keys, values, table, lens, pages, query_d=wide.to(gpu)[:, :8])
    assert (got[3:6, :4] == 0).all()


@pytest.mark.parametrize("count,rows", [(64, 1), (65, 1), (200, 1), (1024, 2), (130, 40)])
def test_long_lists(gpu, count, rows):
    print(f"attend long lists {count} {rows}", flush=True)
    lens = [128 * 140 - 5]
    keys, values, table = make_cache(lens, 1, BF16, seed=count)
    query = make_rows(rows, 4, BF16, 7)
    pages = random_lists(lens, rows, 1, count, seed=count)
    check_attention(gpu, query, keys, values, table, lens, pages)
    shuffled = pages[..., torch.randperm(count, generator=torch.Generator().manual_seed(1))].contiguous()
    check_attention(gpu, query, keys, values, table, lens, shuffled)


@pytest.mark.parametrize("rows,count,heads,kv", [(20, 4, 4, 1), (64, 1024, 4, 1), (160, 4, 128, 64), (32, 4, 8, 1)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_bad_pages_and_values_nobody_attends(gpu, dtype, rows, count, heads, kv):
    """Pages that are none, pages not chosen full of NaN, NaN and infinities at positions a row does not attend."""
    print(f"attend bad pages {rows} {count} {heads}/{kv} {dtype}", flush=True)
    lens = [700, 450]
    keys, values, table = make_cache(lens, kv, dtype, seed=21)
    pages = random_lists(lens, rows, kv, 4, seed=22)
    pages = torch.cat([pages, torch.full((*pages.shape[:-1], count - 4), -1, dtype=torch.int32)], dim=-1)
    for b in range(2):
        for j in range(table.shape[1]):
            if j not in pages[b].flatten().tolist() and table[b, j] >= 0:
                keys[table[b, j].item()] = values[table[b, j].item()] = float("nan")
    # position 695: attended by the rows from 695 on alone
    page, slot = table[0, 695 // 128].item(), 695 % 128
    values[page, slot, 0, 5], values[page, slot, 0, 6] = float("nan"), float("inf")
    values[page, slot, 0, 7], keys[page, slot - 4, 0, 0] = -float("inf"), 100.0
    values[page, 700 % 128:] = float("nan")  # behind the last token
    keys[page, 700 % 128:] = float("nan")
    table[1, pages[1, 0, 0, 0].item()] = -1
    table[1, pages[1, 0, 0, 1].item()] = keys.shape[0] + 3
    query = make_rows(2 * rows, heads, dtype, 23)
    out = torch.zeros_like(query)
    want, size, _ = OP.selected_attention(query, keys, values, table, ints(lens), pages, SCALE, out)
    got = TP.selected_page_attention(query.to(gpu), keys.to(gpu), values.to(gpu), table.to(gpu), ints(lens, gpu),
                                     pages.to(gpu), SCALE).cpu().double()
    finite = want.isfinite()
    assert torch.equal(got.isfinite(), finite)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
    assert (~finite).any() and finite[:rows - 5].all()
    tol = tolerance(want, size, values[values.isfinite()], 512, dtype)
    assert bool(((got - want).abs() <= tol)[finite].all())


@pytest.mark.parametrize("length,rows,heads,kv", [(1, 1, 4, 1), (300, 1, 32, 1), (300, 20, 4, 1), (300, 33, 16, 1),
                                                  (300, 256, 128, 64)])
def test_queries_and_keys_that_are_no_numbers(gpu, length, rows, heads, kv):
    """A NaN among a row's queries or attended keys makes the row NaN, not one without keys, and no other row."""
    print(f"attend NaN {length} {rows} {heads}/{kv}", flush=True)
    keys, values, table = make_cache([length], kv, BF16, seed=81)
    query = make_rows(rows, heads, BF16, 82)
    query[0, 1, 7] = query[-1, -1, 0] = float("nan")
    keys[table[0, 0].item(), 0, 0, 3] = float("nan")  # the first KV head's first key
    pages = random_lists([length], rows, kv, 3, seed=83)
    want, size, _ = OP.selected_attention(query, keys, values, table, ints([length]), pages, SCALE, torch.zeros_like(query))
    got = TP.selected_page_attention(query.to(gpu), keys.to(gpu), values.to(gpu), table.to(gpu), ints([length], gpu),
                                     pages.to(gpu), SCALE).cpu().double()
    assert torch.equal(got.isnan(), want.isnan()) and want[0, 1].isnan().all() and want[-1, -1].isnan().all()
    real = ~want.isnan()
    assert bool(((got - want).abs() <= tolerance(want, size, values, 384, BF16))[real].all())


def test_attention_equals_the_dense_companion_over_all_pages(gpu):
    """Write a chunk's K/V, bounds, selection of every page, attention: as dense causal attention."""
    from trianglemix import cache, kernel

    print("pages pipeline", flush=True)
    seq, rows, heads, kv = 1000, 333, 32, 8
    keys, values, table = make_cache([seq], kv, BF16, seed=31)
    keys, values, table = keys.to(gpu), values.to(gpu), table.to(gpu)
    qkv = make_rows(rows, heads + 2 * kv, BF16, 32).to(gpu)
    start, lens = seq - rows, ints([seq], gpu)
    cache.write_chunk_kv(qkv[:, heads:heads + kv], qkv[:, heads + kv:], keys, values, table, start)
    low, high = TP.page_bounds_like(keys)
    TP.update_page_bounds(keys, table, lens, start, low, high)
    TP.update_page_bounds(keys, table, lens, rows, low, high)
    TP.update_page_bounds(keys, table, lens, seq, low, high)
    query = qkv[:, :heads]
    pages = TP.select_pages(query, low, high, table, lens, 8)
    assert (pages[0, -1] == torch.arange(8, device=gpu)).all()
    got = TP.selected_page_attention(query, keys, values, table, lens, pages, SCALE)
    dense = torch.empty(rows, heads, 128, dtype=BF16, device=gpu)
    kernel.dense_paged_causal_attention(query=query.contiguous(), key_cache=keys, value_cache=values,
                                        block_table=table, seq_len=seq, output=dense, softmax_scale=SCALE)
    # both round the weights to bf16 and the result once: 4 half steps of values of up to 4 in all
    assert (got.float() - dense.float()).abs().max() <= 4 * 2.0 ** -8 * 4
    # fewer pages: the oracle's choice and the oracle's attention
    few = TP.select_pages(query, low, high, table, lens, 4)
    cpu = [t.cpu() for t in (query, low, high, table, lens)]
    assert torch.equal(few.cpu(), OP.select_pages(*cpu, 4, 1, 1))


def test_captured_and_replayed_with_other_lengths(gpu):
    """One graph of all three operators on a batch that decodes; every replay with its own lengths and eager work."""
    print("pages graph", flush=True)
    kv, heads, batch = 2, 8, 3
    all_lens = [[700, 129, 1], [701, 130, 2], [1400, 0, 128], [5, 1300, 900]]
    keys, values, table = make_cache([1400, 1300, 900], kv, BF16, seed=41)
    keys, values, table = keys.to(gpu), values.to(gpu), table.to(gpu)
    query = make_rows(batch, heads, BF16, 42).to(gpu)
    lens = ints(all_lens[0], gpu)

    def step(low, high, out):
        TP.update_page_bounds(keys, table, lens, 1400, low, high)
        pages = TP.select_pages(query, low, high, table, lens, 4)
        TP.selected_page_attention(query, keys, values, table, lens, pages, SCALE, out=out)
        return pages

    bounds = TP.page_bounds_like(keys)
    out = torch.zeros_like(query)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*bounds, out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pages = step(*bounds, out)
    for one in all_lens + all_lens[:2]:
        lens.copy_(ints(one))
        out.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        eager_bounds, eager = TP.page_bounds_like(keys), torch.full_like(query, 3.0)
        eager_pages = step(*eager_bounds, eager)
        torch.cuda.synchronize()
        assert torch.equal(pages, eager_pages) and torch.equal(out, eager), one
        assert (out[[i for i, n in enumerate(one) if n == 0]] == 3.0).all()


@pytest.mark.parametrize("length", [10000, 2 ** 31 - 100, 2 ** 31 - 1])
@pytest.mark.parametrize("rows,heads", [(1, 8), (1, 32), (3, 2), (33, 32)])
def test_lengths_past_the_table(gpu, length, rows, heads):
    """Positions behind every page: the table's pages whole, whatever the distance."""
    print(f"pages past the table {length} {rows} {heads}", flush=True)
    keys, values, table = make_cache([500, 128], 1, BF16, seed=61)
    lens = ints([length, length - 7])
    low, high = bounds_of(keys, table, [500, 128])
    query = make_rows(2 * rows, heads, BF16, 62)
    want = OP.select_pages(query, low, high, table, lens, 3, 1, 1)
    got = TP.select_pages(query.to(gpu), low.to(gpu), high.to(gpu), table.to(gpu), lens.to(gpu), 3).cpu()
    assert torch.equal(got, want) and (want[0] >= 0).all()
    check_attention(gpu, query, keys, values, table, lens.tolist(), want)


def test_calls_on_two_streams_at_once(gpu):
    print("pages two streams", flush=True)
    lens = [128 * 60]
    keys, values, table = make_cache(lens, 2, BF16, seed=51)
    keys, values, table, lens_d = keys.to(gpu), values.to(gpu), table.to(gpu), ints(lens, gpu)
    pages = random_lists(lens, 1, 2, 50, seed=52).to(gpu)
    queries = [make_rows(1, 8, BF16, 53 + i).to(gpu) for i in range(2)]
    alone = [TP.selected_page_attention(q, keys, values, table, lens_d, pages, SCALE) for q in queries]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(TP.selected_page_attention(queries[i], keys, values, table, lens_d, pages, SCALE))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, alone[i]) for o in outs[i])


def test_two_graphs_replayed_at_once(gpu):
    """Two captured calls, each with its own workspace, replayed side by side with eager calls on the capture stream."""
    print("pages two graphs", flush=True)
    lens = [128 * 60]
    keys, values, table = make_cache(lens, 2, BF16, seed=71)
    keys, values, table, lens = keys.to(gpu), values.to(gpu), table.to(gpu), ints(lens, gpu)
    low, high = TP.page_bounds_like(keys)
    TP.update_page_bounds(keys, table, lens, 128 * 60, low, high)
    queries = [make_rows(rows, 8, BF16, 72 + rows).to(gpu) for rows in (1, 70)]

    def step(query, out):
        pages = TP.select_pages(query, low, high, table, lens, 40)
        return TP.selected_page_attention(query, keys, values, table, lens, pages, SCALE, out=out)

    want = [step(q, torch.zeros_like(q)) for q in queries]
    outs = [torch.zeros_like(q) for q in queries]
    graphs = []
    for q, out in zip(queries, outs):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            step(q, out)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for out in outs:
            out.fill_(9.0)
        torch.cuda.synchronize()
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                for _ in range(20):
                    graph.replay()
        eager = step(queries[1], torch.zeros_like(queries[1]))
        torch.cuda.synchronize()
        assert torch.equal(eager, want[1])
        assert all(torch.equal(out, w) for out, w in zip(outs, want))
