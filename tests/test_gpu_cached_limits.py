"""Attention over caches where its numbers or its sizes end, against the definitions in 64 bits."""

from __future__ import annotations

import pytest
import torch

from cached_cases import attention_tolerance, bits, half_step, make_any_cache
from pages_cases import SCALE, make_rows
from trianglemix import cached
from trianglemix.native import load_hip_library

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def ints(x, device="cpu"):
    return torch.tensor(x, dtype=torch.int32, device=device)


def gpu_scales(ks, vs, gpu):
    return {} if ks is None else {"key_scale": ks.to(gpu), "value_scale": vs.to(gpu)}


def seen_keys(n: int, rows: int, window: int, sinks: int):
    """[rows, n]: the keys that each row of a request of n tokens attends."""
    p, k = torch.arange(n - rows, n)[:, None], torch.arange(n)
    seen = k <= p
    return seen if window < 0 else seen & ((k >= p - window) | (k < sinks))


def definition(query, keys, values, table, lens, rows: int, window: int, sinks: int, ks, vs):
    """(out, size) as the oracle gives them, the heads of a request together."""
    batch, kv, heads = len(lens), keys.shape[2], query.shape[1]
    out = torch.zeros(batch * rows, heads, 128, dtype=torch.float64)
    size = torch.zeros_like(out)
    for b, n in enumerate(lens):
        if n == 0:
            continue
        held = min(rows, n)
        pages = table[b, :-(-n // 128)].long()
        k = bits(keys)[pages].view(keys.dtype).double().flatten(0, 1)[:n].transpose(0, 1)
        v = bits(values)[pages].view(values.dtype).double().flatten(0, 1)[:n].transpose(0, 1)
        if ks is not None:
            k, v = k * ks.double()[:, None, None], v * vs.double()[:, None, None]
        at = slice((b + 1) * rows - held, (b + 1) * rows)
        q = query[at].double().view(held, kv, heads // kv, 128).permute(1, 2, 0, 3).reshape(kv, -1, 128)
        score = (q @ k.transpose(1, 2) * SCALE).view(kv, heads // kv, held, n)
        weight = score.masked_fill(~seen_keys(n, held, window, sinks), -float("inf")).softmax(dim=-1).view(kv, -1, n)
        for to, x in ((out, weight @ v), (size, weight @ v.abs())):
            to[at] = x.view(kv, heads // kv, held, 128).permute(2, 0, 1, 3).reshape(held, heads, 128)
    return out, size


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("requests,rows,heads,kv", [(2, 1, 8, 2), (2, 5, 8, 2), (2, 8, 8, 2), (2, 30, 2, 1), (2, 40, 8, 2), (32, 64, 32, 8)])
def test_odd_values_at_keys_of_no_weight(gpu, dtype, requests, rows, heads, kv):
    """NaN in V reaches the rows whose scores there, or everywhere, are -infinity."""
    lens = [700] * requests
    keys, values, table, _, _ = make_any_cache(lens, kv, dtype, "same", seed=33)
    keys.zero_()
    query = torch.zeros(requests * rows, heads, 128, dtype=dtype)
    query[..., 0] = 1.0
    # request 0: its keys have no weight; the others: the first 640
    for b in range(requests):
        for k in range(700 if b == 0 else 640):
            keys[int(table[b, k // 128]), k % 128, :, 0] = -float("inf")
        for k, d in ((5, 3), (37, 64), (333, 127)):  # long before the step, in tiles that no row masks
            values[int(table[b, k // 128]), k % 128, :, d] = float("nan")
    got = cached.cached_attention(query.to(gpu), keys.to(gpu), values.to(gpu), table.to(gpu), ints(lens, gpu), SCALE).cpu()
    want = torch.zeros(128, dtype=torch.bool)
    want[[3, 64, 127]] = True
    assert torch.equal(got.isnan(), want.expand_as(got))
    assert not got[:rows, :, ~want].any() and got[rows:, :, ~want].isfinite().all() and got[rows:, :, ~want].any()


@pytest.mark.parametrize("n,rows,heads", [(60, 1, 8), (100000, 1, 8), (100000, 8, 8), (100000, 20, 8), (20000, 300, 16)])
def test_value_scales_of_any_size(gpu, n, rows, heads):
    """From 2^-126 to 2^118, over sums of many weights: equal keys, so that a row is the mean of one number.

    The weights are equal and exact; what is summed and multiplied in 32 bits stays below 2^-12, the rounding is half a step.
    """
    kv, pages = 4, -(-n // 128)
    vs = torch.tensor([2.0 ** -126, 1.7 * 2.0 ** -126, 1.3 * 2.0 ** -118, 2.0 ** 118])
    table = torch.arange(pages, dtype=torch.int32).view(1, -1)
    keys, values = cached.new_cache(pages, kv)
    values = torch.full(values.shape, 448.0).to(values.dtype)
    query = make_rows(rows, heads, BF16, 5)
    got = cached.cached_attention(query.to(gpu), keys.to(gpu), values.to(gpu), table.to(gpu), ints([n], gpu), SCALE,
                                  **gpu_scales(torch.ones(kv), vs, gpu)).cpu()
    want = (448.0 * vs.double()).repeat_interleave(heads // kv)[:, None].expand(rows, heads, 128)
    assert ((got.double() - want).abs() <= (2.0 ** -12 + half_step(BF16)) * want).all()


# requests, rows, heads, KV heads, window, first keys, columns of the table: four and eight waves of 16 rows, 32 rows with
# one and two row tiles a workgroup, chunks of 128 and of 256 rows
SHAPES = [(2, 4, 8, 2, -1, 0, 0), (2, 4, 8, 2, 40, 3, 0), (32, 2, 16, 8, -1, 0, 64), (32, 2, 16, 8, 40, 3, 300), (2, 8, 8, 2, -1, 0, 0),
          (2, 8, 8, 2, 40, 3, 0), (2, 16, 8, 2, 40, 3, 0), (2, 50, 8, 2, -1, 0, 0), (2, 50, 8, 2, 40, 3, 0), (2, 150, 6, 2, 70, 130, 0),
          (32, 64, 32, 8, -1, 0, 0), (32, 64, 32, 8, 40, 3, 0)]


@pytest.mark.parametrize("cache,dtype", [("e4m3", BF16), ("same", BF16), ("same", FP16)])
@pytest.mark.parametrize("requests,rows,heads,kv,window,sinks,cols", SHAPES)
def test_rows_of_a_step_are_apart(gpu, cache, dtype, requests, rows, heads, kv, window, sinks, cols):
    """NaN at a key that the step's later tokens alone attend, or the earlier ones' windows alone: these rows' results are
    NaN, the others as without it."""
    print(f"apart {requests} {rows} {heads}/{kv} {window} {sinks} {cols} {cache} {dtype}", flush=True)
    lens = [700 if b % 2 == 0 else 300 for b in range(requests)]
    keys, values, table, ks, vs = make_any_cache(lens, kv, dtype, cache, seed=rows + requests)
    if cols:  # as a captured call's
        wide = torch.full((requests, cols), -1, dtype=torch.int32)
        wide[:, :table.shape[1]] = table
        table = wide
    query = make_rows(requests * rows, heads, dtype, 22)
    want, size = definition(query, keys, values, table, lens, rows, window, sinks, ks, vs)
    tol = attention_tolerance(want, size, values, vs, 700, dtype)
    nan = bits(torch.tensor(float("nan")).to(keys.dtype))
    # behind the step's middle; before it, at the first key that the first row's window holds
    places = [(lambda n: n - rows // 2)] + ([lambda n: n - rows - window] if window >= 0 else [])
    for place in places:
        for poisoned in range(2):
            both = [keys.clone(), values.clone()]
            attends = torch.zeros(requests * rows, dtype=torch.bool)
            for b, n in enumerate(lens):
                k = place(n)
                bits(both[poisoned])[int(table[b, k // 128]), k % 128] = nan
                attends[b * rows:(b + 1) * rows] = seen_keys(n, rows, window, sinks)[:, k]
            assert attends.any() and not attends.all()
            got = cached.cached_attention(query.to(gpu), both[0].to(gpu), both[1].to(gpu), table.to(gpu), ints(lens, gpu),
                                          SCALE, window=window, sinks=sinks, **gpu_scales(ks, vs, gpu)).cpu()
            assert got[attends].isnan().all()
            assert ((got.double() - want).abs() <= tol)[~attends].all()


@pytest.mark.parametrize("cache", ["e4m3", "same"])
@pytest.mark.parametrize("requests,rows,heads,kv,window,sinks", [
    (1024, 1, 64, 64, -1, 0), (1024, 1, 64, 64, 100, 4), (256, 16, 32, 8, -1, 0), (1024, 5, 32, 8, -1, 0), (900, 5, 32, 8, 33, 2)])
def test_batches_whose_groups_are_too_many_to_share(gpu, cache, requests, rows, heads, kv, window, sinks):
    """As many groups as leave no memory for records: each is one workgroup's, of any length."""
    print(f"unshared {requests} {rows} {heads}/{kv} {window} {cache}", flush=True)
    lens = [(i * 37) % 301 for i in range(requests)]
    keys, values, table, ks, vs = make_any_cache([300] * 40, kv, BF16, cache, seed=71)
    table = table[torch.arange(requests) % 40].contiguous()  # requests that share pages
    if cache == "e4m3" or rows * heads // kv <= 32:  # more rows over a 16-bit cache are a chunk's
        size_of = load_hip_library().tm_cached_attention_workspace_size
        assert size_of(requests, rows, heads, kv, table.shape[1], window, sinks) == 0
    query = make_rows(requests * rows, heads, BF16, 72)
    want, size = definition(query, keys, values, table, lens, rows, window, sinks, ks, vs)
    before = torch.full(query.shape, 3.0, dtype=BF16)
    out = before.to(gpu)
    cached.cached_attention(query.to(gpu), keys.to(gpu), values.to(gpu), table.to(gpu), ints(lens, gpu), SCALE, window=window,
                            sinks=sinks, out=out, **gpu_scales(ks, vs, gpu))
    got = out.cpu()
    held = ints(lens).repeat_interleave(rows) - rows + torch.arange(requests * rows) % rows >= 0
    assert ((got.double() - want).abs() <= attention_tolerance(want, size, values, vs, 300, BF16))[held].all()
    assert torch.equal(got[~held], before[~held])


@pytest.mark.parametrize("cache", ["e4m3", "same"])
@pytest.mark.parametrize("lens,rows,heads,kv,window,sinks", [
    ([1100, 2000, 700], 1024, 15, 3, -1, 0), ([2100, 900], 1500, 20, 5, -1, 0), ([2048], 2048, 28, 7, 300, 5),
    ([700, 1200], 700, 9, 9, -1, 0)])
def test_chunks_of_odd_kv_heads(gpu, cache, lens, rows, heads, kv, window, sinks):
    """KV heads that divide no round of the GPU, groups that divide no workgroup's rows."""
    keys, values, table, ks, vs = make_any_cache(lens, kv, BF16, cache, seed=81)
    query = make_rows(len(lens) * rows, heads, BF16, 82)
    want, size = definition(query, keys, values, table, lens, rows, window, sinks, ks, vs)
    before = torch.full(query.shape, 3.0, dtype=BF16)
    out = before.to(gpu)
    cached.cached_attention(query.to(gpu), keys.to(gpu), values.to(gpu), table.to(gpu), ints(lens, gpu), SCALE, window=window,
                            sinks=sinks, out=out, **gpu_scales(ks, vs, gpu))
    got = out.cpu()
    held = ints(lens).repeat_interleave(rows) - rows + torch.arange(len(lens) * rows) % rows >= 0
    assert ((got.double() - want).abs() <= attention_tolerance(want, size, values, vs, 2100, BF16))[held].all()
    assert torch.equal(got[~held], before[~held])
