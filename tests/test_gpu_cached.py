"""Attention over 8-bit and 16-bit paged caches against the 64-bit oracle."""

from __future__ import annotations

import threading

import pytest
import torch

from cached_cases import (attention_tolerance, bits, e4m3_tolerance, make_any_cache, make_scales, quantised,
                          rotation_tolerance, side_by_side, turn_error)
from oracle import cached as OC
from pages_cases import SCALE, make_rows
from trianglemix import cabi, cached, rotary
from trianglemix.kernel import dense_paged_causal_attention

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def ints(x, device="cpu"):
    return torch.tensor(x, dtype=torch.int32, device=device)


def gpu_scales(ks, vs, gpu):
    return {} if ks is None else {"key_scale": ks.to(gpu), "value_scale": vs.to(gpu)}


def check(got, want, size, values, vs, keys: int, lens, rows: int, before):
    """Rows that are some within the tolerance, the others as they were."""
    t = torch.arange(got.shape[0]) % rows if rows else torch.zeros(0)
    held = torch.tensor(lens).clamp(min=0).repeat_interleave(rows) - rows + t >= 0
    tol = attention_tolerance(want, size, values, vs, keys, got.dtype)
    off = ((got.double() - want).abs() - tol)[held]
    assert off.numel() == 0 or off.max() <= 0, off.max()
    assert torch.equal(got[~held], before[~held])


CASES = [
    # lens, rows, heads, kv_heads, window, sinks
    ([1], 1, 4, 1, -1, 0),
    ([128, 129, 127, 0, 31, 33, -5], 1, 8, 2, -1, 0),
    ([8111], 1, 8, 2, -1, 0),             # one request over many workgroups
    ([3000, 1, 0, 1500, 700], 1, 32, 8, -1, 0),
    ([500, 77, 1300], 1, 12, 4, -1, 0),
    ([2000, 300], 1, 32, 1, -1, 0),       # 32 query heads a KV head
    ([260, 130], 1, 8, 8, -1, 0),         # one
    ([900, 4, 1100, 130], 5, 32, 8, -1, 0),  # drafted tokens; a request with fewer tokens than rows
    ([300], 16, 16, 4, -1, 0),
    ([640, 900], 17, 8, 2, -1, 0),        # more rows than a workgroup holds
    ([70, 20], 100, 4, 2, -1, 0),
    ([333], 333, 6, 2, -1, 0),            # a whole prompt
    ([1000], 130, 32, 8, -1, 0),
    ([5000, 100, 513, 522], 1, 8, 2, 512, 8),
    ([3000, 40], 1, 8, 2, 0, 0),          # itself alone
    ([3000, 700], 1, 8, 2, 1, 130),       # sinks over more than a page
    ([1500, 2], 9, 12, 4, 100, 4),
    ([900], 300, 8, 2, 64, 1),
    ([400], 1, 4, 1, 1 << 40, 1 << 40),
    ([700], 40, 4, 1, 200, 1000),         # sinks past the window's first key
    ([7200] + [(53 * i) % 400 for i in range(39)], 1, 32, 8, -1, 0),  # eight KV heads a workgroup
    ([(211 * i) % 3001 for i in range(70)], 1, 8, 4, -1, 0),          # more requests than a wave has lanes
    ([20000, 700], 12, 16, 4, -1, 0),     # more shares than are merged at once
    # chunks: more rows of a KV head than the waves of a workgroup hold
    ([900, 64, 0, 1300], 64, 32, 8, -1, 0),
    ([3000], 200, 8, 2, -1, 0),           # shared out over the keys
    ([2500, 100], 150, 12, 4, 300, 5),
    ([700, 50], 40, 32, 1, -1, 0),        # four tokens a workgroup
    ([260, 1], 33, 4, 1, -1, 0),          # a part and four rows
    ([900, 30], 13, 5, 1, -1, 0),         # 65 rows: one more than fits
    ([600, 900], 11, 18, 3, -1, 0),       # 66 rows
    ([640, 300], 7, 18, 2, 100, 3),       # 63 rows, nine heads a KV head
    ([900, 30, 2000], 11, 9, 3, -1, 0),   # 33 rows
    ([1100, 8, 700], 8, 8, 2, -1, 0),     # 32 rows
    ([5000], 129, 8, 8, 700, 0),
]


@pytest.mark.parametrize("cache", ["e4m3", "same"])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("lens,rows,heads,kv_heads,window,sinks", CASES)
def test_attention(gpu, dtype, cache, lens, rows, heads, kv_heads, window, sinks):
    print(f"cached {lens} {rows} {heads}/{kv_heads} {window} {sinks} {dtype} {cache}", flush=True)
    keys, values, table, ks, vs = make_any_cache(lens, kv_heads, dtype, cache, seed=rows + heads)
    query = make_rows(len(lens) * rows, heads, dtype, 3)
    want, size = OC.attention(query, keys, values, table, ints(lens), SCALE, window, sinks, ks, vs)
    before = make_rows(len(lens) * rows, heads, dtype, 4)
    out = before.to(gpu)
    args = (query.to(gpu), keys.to(gpu), values.to(gpu), table.to(gpu), ints(lens, gpu))
    scales = gpu_scales(ks, vs, gpu)
    got = cached.cached_attention(*args, SCALE, window=window, sinks=sinks, out=out, **scales)
    assert got is out
    check(got.cpu(), want, size, values, vs, max(max(lens), 1), lens, rows, before)
    again = before.to(gpu)
    cabi.cached_attention(*args, again, scale=SCALE, window=window, sinks=sinks, **scales)
    assert torch.equal(again, out)  # the same bits, whichever workgroup merges
    fresh = cached.cached_attention(*args, SCALE, window=window, sinks=sinks, **scales).cpu()
    t = torch.arange(fresh.shape[0]) % rows
    held = ints(lens).long().clamp(min=0).repeat_interleave(rows) - rows + t >= 0
    assert torch.equal(fresh[held], out.cpu()[held]) and not fresh[~held].any()


@pytest.mark.parametrize("cache", ["e4m3", "same"])
def test_strides_bad_pages_and_lengths_past_the_table(gpu, cache):
    """K and V pages side by side, Q in a fused buffer, a table with wide rows and pages that are none."""
    lens = [1000, 700, 300, 2 ** 31 - 1]
    keys, values, table, ks, vs = make_any_cache([1000, 700, 300, 400], 2, BF16, cache, seed=11)
    pages = keys.shape[0]
    both = side_by_side(keys, values)
    table[0, 2], table[0, 5], table[1, 0], table[2, :] = -1, pages, -(1 << 31), 1 << 30
    wide_table = torch.full((4, 2 * table.shape[1] + 3), 77777, dtype=torch.int32)
    wide_table[:, :table.shape[1]] = table
    view = wide_table[:, :table.shape[1]]
    wide = make_rows(4 * 3, 14, BF16, 12)
    query = wide[:, 3:11]
    want, size = OC.attention(query, keys, values, view, ints(lens), SCALE, -1, 0, ks, vs)
    assert not want[6:9].any()  # a request without a page: zeros
    b, w = both.to(gpu), wide.to(gpu)
    out = torch.full((12, 8, 128), 7.0, dtype=BF16, device=gpu)
    cached.cached_attention(w[:, 3:11], b[:, 0], b[:, 1], wide_table.to(gpu)[:, :table.shape[1]], ints(lens, gpu), SCALE,
                            out=out, **gpu_scales(ks, vs, gpu))
    check(out.cpu(), want, size, values, vs, 1500, lens, 3, out.cpu())
    # a window of the longest length holds no key of the table: zeros again
    cached.cached_attention(w[:, 3:11], b[:, 0], b[:, 1], wide_table.to(gpu)[:, :table.shape[1]], ints(lens, gpu), SCALE,
                            window=5, out=out, **gpu_scales(ks, vs, gpu))
    want, size = OC.attention(query, keys, values, view, ints(lens), SCALE, 5, 0, ks, vs)
    check(out.cpu(), want, size, values, vs, 1500, lens, 3, out.cpu())
    assert not out[9:].any()


@pytest.mark.parametrize("cache", ["e4m3", "same"])
@pytest.mark.parametrize("rows,heads,window,sinks", [(1, 8, -1, 0), (1, 8, 100, 4), (9, 8, -1, 0), (9, 8, 100, 4), (40, 12, 30, 4),
                                                    (130, 8, -1, 0)])
def test_what_a_row_does_not_attend_cannot_reach_it(gpu, cache, rows, heads, window, sinks):
    """NaN behind the last token, in front of the window and at drafted tokens after a row's own position."""
    lens, kv = [700, 300], 2
    keys, values, table, ks, vs = make_any_cache(lens, kv, BF16, cache, seed=21)
    query = make_rows(2 * rows, heads, BF16, 22)
    poisoned = [keys.clone(), values.clone()]
    nan = torch.tensor(float("nan")).to(keys.dtype)
    hidden = []
    for b, n in enumerate(lens):
        first = max(0, n - rows - window) if window >= 0 else 0
        for k in list(range(n, -(-n // 128) * 128)) + list(range(sinks, first)):
            hidden.append((int(table[b, k // 128]), k % 128))
    for page, slot in hidden:
        for t in poisoned:
            bits(t)[page, slot] = bits(nan)
    args = (table.to(gpu), ints(lens, gpu), SCALE)
    more = dict(window=window, sinks=sinks, **gpu_scales(ks, vs, gpu))
    clean = cached.cached_attention(query.to(gpu), keys.to(gpu), values.to(gpu), *args, **more)
    got = cached.cached_attention(query.to(gpu), poisoned[0].to(gpu), poisoned[1].to(gpu), *args, **more)
    assert torch.equal(got, clean) and clean.isfinite().all()


@pytest.mark.parametrize("cache,odd", [("e4m3", "nan"), ("same", "nan"), ("same", "inf"), ("same", "-inf"), ("same", "both")])
@pytest.mark.parametrize("rows,window,sinks", [(1, -1, 0), (7, -1, 0), (7, 20, 3), (20, -1, 0), (40, -1, 0), (70, 20, 3)])
def test_odd_values_reach_their_rows_and_dims(gpu, cache, odd, rows, window, sinks):
    """A value that is no finite number reaches the rows that attend its key, in its dim and KV head alone."""
    lens, kv, heads = [300, 170], 2, 8
    keys, values, table, ks, vs = make_any_cache(lens, kv, BF16, cache, seed=31)
    keys = (keys.float() * 0.1).to(keys.dtype)  # weights of a kind: an infinity's does not round to zero
    query = make_rows(2 * rows, heads, BF16, 32)
    v = values.float()
    places = [(0, 299, 0, 5), (0, 296, 1, 77), (0, 290, 0, 127), (1, 169, 1, 0), (1, 164, 0, 64), (1, 1, 1, 30)]
    for i, (b, k, h, d) in enumerate(places):
        x = {"nan": float("nan"), "inf": float("inf"), "-inf": -float("inf"), "both": (-1) ** i * float("inf")}[odd]
        v[int(table[b, k // 128]), k % 128, h, d] = x
    if odd == "both":  # opposite infinities in one dim: NaN where both are attended
        v[int(table[0, 2]), 298 - 256, 0, 5] = -float("inf")
    values = v.to(values.dtype)
    want, size = OC.attention(query, keys, values, table, ints(lens), SCALE, window, sinks, ks, vs)
    got = cached.cached_attention(query.to(gpu), keys.to(gpu), values.to(gpu), table.to(gpu), ints(lens, gpu), SCALE,
                                  window=window, sinks=sinks, **gpu_scales(ks, vs, gpu)).cpu()
    assert torch.equal(got.isnan(), want.isnan()) and not want.isfinite().all()
    assert torch.equal(got.isinf() * got.sign().nan_to_num(), (want.isinf() * want.sign().nan_to_num()).to(BF16))
    fine = want.isfinite()
    tol = attention_tolerance(want, size, values, vs, 300, BF16)
    assert ((got.double() - want).abs() <= tol)[fine].all()


@pytest.mark.parametrize("rows", [6, 40, 100])
def test_nan_in_queries_and_keys(gpu, rows):
    lens, kv, heads = [400], 2, 8
    keys, values, table, ks, vs = make_any_cache(lens, kv, BF16, "e4m3", seed=41)
    query = make_rows(rows, heads, BF16, 42)
    query[2, 5, 9] = float("nan")
    bits(keys)[int(table[0, 3]), 397 - 384, 0, 3] = 0x7f  # key 397: the last three rows attend it
    got = cached.cached_attention(query.to(gpu), keys.to(gpu), values.to(gpu), table.to(gpu), ints(lens, gpu), SCALE,
                                  **gpu_scales(ks, vs, gpu)).cpu()
    want = torch.zeros(rows, heads, dtype=torch.bool)
    want[2, 5] = True
    want[-3:, :4] = True
    assert torch.equal(got.isnan().all(dim=-1), want) and torch.equal(got.isnan().any(dim=-1), want)


def test_scores_of_minus_infinity_and_of_one_size(gpu):
    """Keys at -infinity have no weight, rows of them alone give zeros; equal scores give the mean."""
    lens, kv = [200, 150], 1
    keys, values, table, _, _ = make_any_cache(lens, kv, BF16, "same", seed=51)
    keys.zero_()
    for k in range(150):
        keys[int(table[1, k // 128]), k % 128, 0, 0] = -float("inf")
    keys[int(table[0, 0]), 7, 0, 0] = -float("inf")
    query = torch.zeros(2, 4, 128, dtype=BF16)
    query[..., 0] = 1.0
    got = cached.cached_attention(query.to(gpu), keys.to(gpu), values.to(gpu), table.to(gpu), ints(lens, gpu), SCALE).cpu()
    assert not got[1].any()
    rows = values[table[0, :2].long()].double().flatten(0, 1)[:200, 0]
    mean = torch.cat([rows[:7], rows[8:]]).mean(dim=0)
    size = torch.cat([rows[:7], rows[8:]]).abs().mean(dim=0)
    assert ((got[0].double() - mean).abs() <= attention_tolerance(mean, size, values, None, 200, BF16)).all()


def test_many_small_weights_are_not_lost(gpu):
    """One large weight beside 65535 of 2^-26 of it each: their sum is 2^-10 of it, and fp16 alone would drop them."""
    n, kv = 65536, 1
    table = torch.arange(512, dtype=torch.int32).view(1, 512)
    keys, values = cached.new_cache(512, kv)
    keys, values = keys.float(), values.float()
    values[...] = 256.0
    values[0, 0] = 0.0
    query = torch.zeros(1, 4, 128, dtype=FP16)
    query[..., 0] = 1.0
    keys[0, 0, 0, 0] = 26.0  # times ln 2 below: 2^26 times the others' weight
    keys, values = keys.to(torch.float8_e4m3fn), values.to(torch.float8_e4m3fn)
    one = torch.ones(1)
    scale = 0.6931471805599453
    want, size = OC.attention(query, keys, values, table, ints([n]), scale, -1, 0, one, one)
    assert 0.2 < want.mean() < 0.3  # 256 * 2^-10
    got = cached.cached_attention(query.to(gpu), keys.to(gpu), values.to(gpu), table.to(gpu), ints([n], gpu), scale,
                                  **gpu_scales(one, one, gpu)).cpu()
    assert ((got.double() - want).abs() <= attention_tolerance(want, size, values, one, n, FP16)).all()


def test_a_cache_behind_2_31_bytes(gpu):
    """Pages far behind 2^31 bytes and numbers of the cache, and contexts of two million tokens."""
    print("far cache", flush=True)
    pages, kv, heads = 36000, 8, 32
    keys, values = cached.new_cache(pages, kv, device=gpu)
    used = [35999, 17001, 33000, 5, 20000]
    lens = [5 * 128 - 3]
    k, v, _, ks, vs = make_any_cache([640], kv, BF16, "e4m3", seed=61, spare=0)
    at = torch.tensor(used, device=gpu)
    bits(keys)[at], bits(values)[at] = bits(k).to(gpu), bits(v).to(gpu)
    query = make_rows(1, heads, BF16, 62)
    want, size = OC.attention(query, k, v, torch.arange(5, dtype=torch.int32)[None], ints(lens), SCALE, -1, 0, ks, vs)
    got = cached.cached_attention(query.to(gpu), keys, values, ints([used], gpu), ints(lens, gpu), SCALE,
                                  **gpu_scales(ks, vs, gpu)).cpu()
    assert ((got.double() - want).abs() <= attention_tolerance(want, size, v, vs, 640, BF16)).all()
    many = make_rows(100, heads, BF16, 63)  # a chunk
    want, size = OC.attention(many, k, v, torch.arange(5, dtype=torch.int32)[None], ints(lens), SCALE, -1, 0, ks, vs)
    got = cached.cached_attention(many.to(gpu), keys, values, ints([used], gpu), ints(lens, gpu), SCALE,
                                  **gpu_scales(ks, vs, gpu)).cpu()
    assert ((got.double() - want).abs() - attention_tolerance(want, size, v, vs, 640, BF16)).max() <= 0
    # 16384 columns that repeat these pages: every key 3276 or 3277 times
    cols = 16384
    long = at.to(torch.int32).repeat(cols // 5 + 1)[:cols].view(1, cols).contiguous()
    got = cached.cached_attention(query.to(gpu), keys, values, long, ints([cols * 128], gpu), SCALE,
                                  **gpu_scales(ks, vs, gpu)).cpu()
    order = (torch.arange(cols) % 5).to(torch.int32)[None]
    want, size = OC.attention(query, k, v, order, ints([cols * 128]), SCALE, -1, 0, ks, vs)
    assert ((got.double() - want).abs() <= attention_tolerance(want, size, v, vs, cols * 128, BF16)).all()


@pytest.mark.parametrize("cache", ["e4m3", "same"])
@pytest.mark.parametrize("lens,rows,window,sinks", [([300], 128, -1, 0), ([40, 700, 0], 33, -1, 0), ([500, 90], 9, -1, 0), ([700, 70], 50, 200, 3),
                                                    ([900, 3], 1, -1, 0)])
def test_tables_far_wider_than_the_requests(gpu, cache, lens, rows, window, sinks):
    """A table for two million tokens, as a captured call has it: nothing but the lengths bounds what is read."""
    heads, kv = 8, 2
    keys, values, table, ks, vs = make_any_cache(lens, kv, BF16, cache, seed=131)
    query, before = make_rows(len(lens) * rows, heads, BF16, 132), make_rows(len(lens) * rows, heads, BF16, 133)
    want, size = OC.attention(query, keys, values, table, ints(lens), SCALE, window, sinks, ks, vs)
    wide = torch.full((len(lens), 16384), 1 << 30, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    out = before.to(gpu)
    cached.cached_attention(query.to(gpu), keys.to(gpu), values.to(gpu), wide.to(gpu), ints(lens, gpu), SCALE, window=window,
                            sinks=sinks, out=out, **gpu_scales(ks, vs, gpu))
    check(out.cpu(), want, size, values, vs, max(lens), lens, rows, before)


def test_many_requests(gpu):
    """1024 requests of 0 to 300 tokens: more than a wave's lanes hold lengths of."""
    lens = [(i * 37) % 301 for i in range(1024)]
    keys, values, table, ks, vs = make_any_cache(lens, 1, BF16, "e4m3", seed=71)
    query = make_rows(1024, 2, BF16, 72)
    want, size = OC.attention(query, keys, values, table, ints(lens), SCALE, -1, 0, ks, vs)
    before = torch.full((1024, 2, 128), 3.0, dtype=BF16)
    out = before.to(gpu)
    cached.cached_attention(query.to(gpu), keys.to(gpu), values.to(gpu), table.to(gpu), ints(lens, gpu), SCALE, out=out,
                            **gpu_scales(ks, vs, gpu))
    check(out.cpu(), want, size, values, vs, 300, lens, 1, before)


@pytest.mark.parametrize("rows", [1, 6, 60])
def test_graph_replays_with_other_lengths(gpu, rows):
    """Two graphs of steps from one pool, replayed in turn with lengths of their own and eager calls between."""
    heads, kv, batch = 8, 2, 5
    keys, values, table, ks, vs = make_any_cache([2500, 1800, 2000, 900, 700], kv, BF16, "e4m3", seed=81)
    keys, values, table = keys.to(gpu), values.to(gpu), table.to(gpu)
    scales = gpu_scales(ks, vs, gpu)
    query = make_rows(batch * rows, heads, BF16, 82).to(gpu)
    lens = [ints([1] * batch, gpu) for _ in range(2)]
    outs = [torch.zeros_like(query) for _ in range(2)]
    cached.cached_attention(query, keys, values, table, lens[0], SCALE, out=outs[0], **scales)
    pool = torch.cuda.graph_pool_handle()
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    for i, graph in enumerate(graphs):
        with torch.cuda.graph(graph, pool=pool):
            cached.cached_attention(query, keys, values, table, lens[i], SCALE, window=-1 if i else 300, out=outs[i], **scales)
    for turn in range(4):
        now = [[2500 - 300 * turn, 1800, 17 * turn, 900 - turn, 128 * turn], [turn, 5, 2000, 1, 700]]
        for i, graph in enumerate(graphs):
            lens[i].copy_(ints(now[i]))
            outs[i].zero_()
            graph.replay()
        torch.cuda.synchronize()
        for i in range(2):
            eager = torch.zeros_like(query)
            cached.cached_attention(query, keys, values, table, lens[i], SCALE, window=-1 if i else 300, out=eager, **scales)
            assert torch.equal(eager, outs[i]), (turn, i)


@pytest.mark.parametrize("binding", ["torch", "ctypes"])
def test_threads_and_streams(gpu, binding):
    """Three host threads, two of them on one stream, the third on another: every call's result as if it were alone."""
    lens = [9000, 128 * 40 - 3, 700]
    keys, values, table, ks, vs = make_any_cache(lens, 2, BF16, "e4m3", seed=91)
    args = (keys.to(gpu), values.to(gpu), table.to(gpu), ints(lens, gpu))
    scales = gpu_scales(ks, vs, gpu)
    queries = [make_rows(3 * r, 8, BF16, 92 + r).to(gpu) for r in (1, 5, 60)]

    def call(i):
        out = torch.zeros_like(queries[i])
        if binding == "torch":
            return cached.cached_attention(queries[i], *args, SCALE, out=out, **scales)
        cabi.cached_attention(queries[i], *args, out, scale=SCALE, **scales)
        return out

    alone = [call(i) for i in range(3)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    streams = [torch.cuda.current_stream(), torch.cuda.current_stream(), side]
    wrong = []

    def work(i):
        with torch.cuda.stream(streams[i]):
            results = [call(i) for _ in range(30)]
        torch.cuda.synchronize()
        wrong.extend(i for r in results if not torch.equal(r, alone[i]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("cache", ["e4m3", "same"])
def test_a_request_from_prompt_to_tokens(gpu, cache):
    """A prompt in two chunks, then tokens one by one: rotated writes, and attention over what they wrote."""
    heads, kv, chunks = 32, 8, [(0, 300), (300, 77)] + [(377 + i, 1) for i in range(4)]
    total = 381
    f = rotary.frequencies(128, 500000.0)
    qkv = make_rows(total, heads + 2 * kv, BF16, 101)
    ks, vs = (make_scales(kv, 1), make_scales(kv, 2)) if cache == "e4m3" else (None, None)
    table = ints([[4, 0, 2]])
    keys, values = cached.new_cache(5, kv, None if cache == "e4m3" else BF16, device=gpu)
    scales = gpu_scales(ks, vs, gpu)
    slot_of = lambda t: int(table[0, t // 128]) * 128 + t % 128  # noqa: E731
    outs, queries = [], []
    for first, n in chunks:
        part = qkv[first:first + n].to(gpu)
        pos = torch.arange(first, first + n, device=gpu)
        slots = torch.tensor([slot_of(t) for t in range(first, first + n)], device=gpu)
        q = torch.empty(n, heads, 128, dtype=BF16, device=gpu)
        rotary.rotate_and_cache(part[:, :heads], part[:, heads:heads + kv], part[:, heads + kv:], pos, slots, f.to(gpu), keys,
                                values, query_out=q, **scales)
        lens = ints([first + n], gpu)
        out = cached.cached_attention(q, keys, values, table.to(gpu), lens, SCALE, **scales)
        if cache == "same" and n > 1:  # the dense prefill kernel over the same pages
            dense = torch.empty_like(q)
            dense_paged_causal_attention(query=q, key_cache=keys, value_cache=values, block_table=table.to(gpu),
                                         seq_len=first + n, output=dense, softmax_scale=SCALE)
            assert (dense.float() - out.float()).abs().max() < 2e-2
        outs.append(out.cpu())
        queries.append(q.cpu())
    # from the definitions, with the stored numbers that the definitions give
    at = torch.arange(total)
    k = OC.rotate(qkv[:, heads:heads + kv], at, f, False, 1.0)
    v = qkv[:, heads + kv:]
    slots = torch.tensor([slot_of(t) for t in range(total)])
    got_k = keys.cpu().double().view(-1, kv, 128)[slots]
    got_v = bits(values.cpu()).view(-1, kv, 128)[slots].view(values.dtype)
    if cache == "e4m3":
        want = OC.quotient(k, ks)
        error = turn_error(qkv[:, heads:heads + kv], 64, False, 1.0) / ks.double()[:, None]
        assert ((got_k - want).abs() - e4m3_tolerance(want, error)).max() <= 0
        assert torch.equal(bits(got_v), bits(quantised(v, vs)))
    else:
        tol = rotation_tolerance(qkv[:, heads:heads + kv], k, 64, False, 1.0, BF16)
        assert ((got_k - k).abs() - tol).max() <= 0 and torch.equal(got_v, v)
    for (first, n), q, out in zip(chunks, queries, outs):
        want, size = OC.attention(q, keys.cpu(), values.cpu(), table, ints([first + n]), SCALE, -1, 0, ks, vs)
        assert ((out.double() - want).abs() - attention_tolerance(want, size, values.cpu(), vs, total, BF16)).max() <= 0
