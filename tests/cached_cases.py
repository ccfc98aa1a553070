"""Seeded inputs and tolerances of the cached-attention operators' tests, on the CPU."""

from __future__ import annotations

import torch
from pages_cases import make_cache

E4M3, E4M3_MAX = torch.float8_e4m3fn, 448.0


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def quantised(x, scale):
    """e4m3 numbers of ``x [..., heads, 128]`` by the heads' scales, as an 8-bit cache takes them."""
    return (x.float() / scale[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(E4M3)


def make_scales(kv_heads: int, seed: int):
    g = torch.Generator().manual_seed(seed)
    return (3.0 + 3.0 * torch.rand(kv_heads, generator=g)) / E4M3_MAX


def make_any_cache(lens, kv_heads: int, dtype, cache: str, seed: int, **more):
    """(keys, values, table, key_scale, value_scale): a 16-bit cache, or its 8-bit numbers and their scales."""
    keys, values, table = make_cache(lens, kv_heads, dtype, seed, **more)
    if cache == "same":
        return keys, values, table, None, None
    ks, vs = make_scales(kv_heads, seed + 1), make_scales(kv_heads, seed + 2)
    return quantised(keys, ks), quantised(values, vs), table, ks, vs


def bits(x):
    """The numbers' bits as integers: indexing, stacking and comparison know no 8-bit floats."""
    return x.view(torch.uint8 if x.dtype == E4M3 else torch.int16)


def side_by_side(keys, values):
    """K and V pages in one tensor, as ``[pages, 2, 128, kv_heads, 128]`` caches have them."""
    return torch.stack([bits(keys), bits(values)], dim=1).view(keys.dtype)


def pair_sum(x, pairs: int, interleaved: bool):
    """|a| + |b| of each dim's pair, zeros for the dims that do not turn."""
    size = x.double().abs()
    out = torch.zeros_like(size)
    if interleaved:
        both = size[..., 0:2 * pairs:2] + size[..., 1:2 * pairs:2]
        out[..., 0:2 * pairs:2], out[..., 1:2 * pairs:2] = both, both
    else:
        both = size[..., :pairs] + size[..., pairs:2 * pairs]
        out[..., :pairs], out[..., pairs:2 * pairs] = both, both
    return out


def turn_error(x, pairs: int, interleaved: bool, magnitude: float):
    """Largest error of a rotated number before its rounding.

    The angle is left with 2^-24 of half a turn after its reduction (less than 2^-22 radians), sine and cosine of it are
    off by up to 2^-22 more, their product with the magnitude and the two products with a and b by 2^-24 each: below
    2^-20 of |a| + |b| together.
    """
    return 2.0 ** -20 * abs(magnitude) * pair_sum(x, pairs, interleaved)


def rotation_tolerance(x, want, pairs: int, interleaved: bool, magnitude: float, dtype):
    """The error above and one rounding: half a step, for fp16 numbers below its normal range 2^-25."""
    return turn_error(x, pairs, interleaved, magnitude) + half_step(dtype) * 1.001 * want.abs() + (
        2.0 ** -25 if dtype == torch.float16 else 0.0)


def e4m3_tolerance(quotient, error):
    """Of a stored e4m3 number: its quotient's error, that of the division and one rounding (half a step is 2^-4 of the
    number, below the normal range 2^-10)."""
    return error + quotient.abs() * (2.0 ** -22 + 1.001 * 2.0 ** -4) + 2.0 ** -10


def attention_tolerance(out, size, values, value_scale, keys: int, dtype):
    """Largest error of an attention output, from the arithmetic; ``size`` is sum(weight * |value|).

    The weights enter the value product rounded to fp16 over an 8-bit cache, else to the type, off by at most half a step
    u: u * size; the result is rounded once.  fp16 weights stand 2^7 times larger than themselves, so those below its
    normal range are off by up to 2^-32 of the row's largest (at least 1, the sum too).  What is summed in 32 bits (128
    products of a score, the weights) and the hardware's exp2 (2^-22 relative for scores below 64) stay below 2^-12 of
    size.
    """
    weight = torch.float16 if value_scale is not None else dtype
    tol = half_step(weight) * size + half_step(dtype) * out.abs() + 2.0 ** -12 * size
    if weight == torch.float16:
        largest = values.float().nan_to_num(0.0, 0.0, 0.0).abs().max() * (1.0 if value_scale is None else value_scale.max())
        tol = tol + keys * 2.0 ** -32 * float(largest)
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25
    return tol
