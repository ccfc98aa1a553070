"""Attention over caches where its numbers or its sizes end, against the definitions in 64 bits."""

from __future__ import annotations

import pytest
import torch

from cached_cases import attention_tolerance, bits, half_step, make_any_cache
from pages_cases import SCALE, make_rows
from trianglemix import cached

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
