"""Seeded inputs of the paged serving operators' tests, on the CPU."""

from __future__ import annotations

import torch

SCALE = 128 ** -0.5


def make_cache(lens, kv_heads: int, dtype, seed: int, spare: int = 3, stride_pages: bool = False):
    """(keys, values, table): random pages of requests with these lengths, scattered over the cache.

    ``stride_pages`` interleaves K and V pages in one tensor, as ``[pages, 2, 128, kv_heads, 128]`` caches do.
    """
    g = torch.Generator().manual_seed(seed)
    used = [-(-max(n, 0) // 128) for n in lens]
    pages = sum(used) + spare
    order = torch.randperm(pages, generator=g)
    cols = max(max(used), 1) + 1
    table = torch.full((len(lens), cols), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n].to(torch.int32)
        at += n
    kv = torch.randn(pages, 2, 128, kv_heads, 128, generator=g)
    kv[:, 0] += 0.7 * torch.randn(pages, 1, kv_heads, 128, generator=g)
    kv = kv.to(dtype)
    keys, values = kv[:, 0], kv[:, 1]
    if not stride_pages:
        keys, values = keys.contiguous(), values.contiguous()
    return keys, values, table


def make_rows(n: int, heads: int, dtype, seed: int):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, heads, 128, generator=g) + 0.5 * torch.randn(1, heads, 128, generator=g)).to(dtype)


def to_gpu(t, gpu):
    """The tensor on the GPU, a page- or row-strided view as such."""
    if t.is_contiguous() or t.numel() == 0:
        return t.to(gpu)
    base = t._base if t._base is not None else t
    return base.to(gpu).as_strided(t.size(), t.stride(), t.storage_offset())


def tolerance(out, size, values, keys: int, dtype):
    """Largest error of an attention output of this type, from the arithmetic.

    ``size`` is sum(weight * |value|).  The weights enter the value product rounded to the type, off by at most half a
    step u each: u * size; the result is rounded once: u * |out|.  fp16 weights below its normal range are off by up
    to 2^-25 of the row's largest (at least 1, the sum too): keys * 2^-25 * max |value|.  What is summed in 32 bits
    (128 products of a score, `keys` weights) and the hardware's exp2 (2^-22 relative for scores below 64) stay
    below 2^-12 of size.
    """
    u = torch.finfo(dtype).eps / 2
    tol = u * (size + out.abs()) + 2.0 ** -12 * size
    if dtype == torch.float16:
        tol = tol + keys * 2.0 ** -25 * float(values.abs().max())
    return tol
