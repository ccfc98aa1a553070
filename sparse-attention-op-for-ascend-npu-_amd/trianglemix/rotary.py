"""Position rotation of query and key rows, alone or with the write of a step's keys and values into the cache.

``frequencies`` gives the radians a position of each pair of dims, ``rotate`` turns rows that stay outside the cache
(drafted tokens, ``tree.tree_attention``), ``rotate_and_cache`` turns a step's queries and keys and stores keys and
values in one launch, into a cache of the rows' own type or of 8-bit numbers (``cached.new_cache``).  Positions, slots
and scales are read on the device: a captured call can be replayed with others.  The operators are
``torch.ops.trianglemix`` ones; ``include/trianglemix_cached.h`` is their C ABI and states every rule.
"""

from __future__ import annotations

import math


def frequencies(rotary_dim: int, base: float = 10000.0, *, stretch: float = 1.0, method: str = "parts",
                trained_length: int | None = None, fast_turns: float = 32.0, slow_turns: float = 1.0, device=None):
    """float64 ``[rotary_dim / 2]``: ``base ** (-2 i / rotary_dim)``, changed for contexts ``stretch`` times as long.

    ``method`` says how: ``"positions"`` divides every frequency by ``stretch``; ``"base"`` enlarges the base so that the
    slowest pair is divided by it and the fastest is left alone; ``"parts"`` leaves alone the pairs that turn at least
    ``fast_turns`` times over ``trained_length`` positions, divides those of at most ``slow_turns``, and mixes linearly
    in between (``magnitude`` belongs to it).  Linearly in the turns: a model trained with a mix that is linear in the
    pair's index has frequencies of its own, which the operators take as they are.
    """
    import torch

    if rotary_dim < 16 or rotary_dim > 128 or rotary_dim % 16:
        raise ValueError("rotary_dim must be a multiple of 16 from 16 to 128")
    if not (math.isfinite(base) and base > 1.0 and math.isfinite(stretch) and stretch >= 1.0):
        raise ValueError("base must be finite and above 1, stretch finite and at least 1")
    if method not in ("positions", "base", "parts"):
        raise ValueError("method must be 'positions', 'base' or 'parts'")
    if method == "base":
        base = base * stretch ** (rotary_dim / (rotary_dim - 2))
    i = torch.arange(rotary_dim // 2, dtype=torch.float64)
    f = base ** (-2.0 * i / rotary_dim)
    if stretch > 1.0 and method == "positions":
        f = f / stretch
    if stretch > 1.0 and method == "parts":
        if trained_length is None or trained_length <= 0 or not fast_turns > slow_turns:
            raise ValueError("method 'parts' needs the trained_length, and fast_turns above slow_turns")
        turns = trained_length * f / (2.0 * math.pi)
        keep = ((turns - slow_turns) / (fast_turns - slow_turns)).clamp(0.0, 1.0)
        f = f * keep + f / stretch * (1.0 - keep)
    return f.to(device) if device is not None else f


def magnitude(stretch: float) -> float:
    """The factor on rotated rows that goes with frequencies stretched by parts."""
    return 0.1 * math.log(stretch) + 1.0


def rotate(x, positions, freqs, *, interleaved: bool = False, magnitude: float = 1.0, out=None):
    """Rows ``x [rows, heads, 128]`` turned by ``positions`` (int64; a negative one is no row).

    ``interleaved`` pairs dims (2 i, 2 i + 1), otherwise (i, i + rotary_dim / 2).  ``out`` may be ``x`` itself; its rows at
    negative positions keep what they hold (zeros without ``out``).
    """
    import torch

    from .native import require_adapter

    require_adapter()  # no CPU fallback: fails loudly without the native library
    op = torch.ops.trianglemix.rotate_positions
    if out is None:
        return op(x, positions, freqs, interleaved, magnitude)
    return op.out(x, positions, freqs, interleaved, magnitude, out=out)


def rotate_and_cache(query, key, value, positions, slot_mapping, freqs, key_cache, value_cache, *,
                     interleaved: bool = False, magnitude: float = 1.0, key_scale=None, value_scale=None,
                     query_out=None):
    """Turn a step's queries and keys, store keys and values in their slots; returns ``query_out`` (default: in place).

    ``query``, ``key`` and ``value`` may be slices of one fused buffer.  ``slot_mapping`` is int64 as that of
    ``cache.reshape_and_cache`` (negative: not stored); 8-bit caches take ``key_scale`` and ``value_scale``.
    """
    import torch

    from .native import require_adapter

    require_adapter()
    if query_out is None:
        query_out = query
    torch.ops.trianglemix.rotate_and_cache(query, key, value, positions, slot_mapping, freqs, interleaved, magnitude,
                                           query_out, key_cache, value_cache, key_scale, value_scale)
    return query_out
