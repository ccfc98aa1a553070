"""The rotated write into an 8-bit cache at the ends of its scales' range."""

from __future__ import annotations

import pytest
import torch

from cached_cases import E4M3, E4M3_MAX, bits
from trianglemix import cached, rotary

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def test_8_bit_numbers_of_tiny_and_large_scales(gpu):
    """Every 16-bit number by scales at the ends of their range: the quotient's nearest, ties to even, as elsewhere."""
    value = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(BF16).view(512, 1, 128)
    slots = torch.arange(512, device=gpu)
    f = rotary.frequencies(128).to(gpu)
    for scale in (2.0 ** -126, 1.5 * 2.0 ** -126, 1.75 * 2.0 ** -121, 1.875 * 2.0 ** -120, 1.5625 * 2.0 ** -110, 1.3 * 2.0 ** -90,
                  1.75 * 2.0 ** -64, 1.9 * 2.0 ** 100, 2.0 ** 126):
        s = torch.tensor([scale])
        keys, values = cached.new_cache(4, 1, device=gpu)
        rotary.rotate_and_cache(value.to(gpu), value.to(gpu), value.to(gpu), torch.zeros_like(slots), slots, f, keys, values,
                                key_scale=s.to(gpu), value_scale=s.to(gpu), query_out=torch.empty_like(value, device=gpu))
        got = values.view(-1, 1, 128).cpu()
        want = (value.float() / s).clamp(-E4M3_MAX, E4M3_MAX).to(E4M3)
        nan = value.isnan()
        assert torch.equal(got.float().isnan(), nan)
        assert torch.equal(bits(got)[~nan], bits(want)[~nan]), scale
        k = keys.view(-1, 1, 128).cpu()  # position 0 turns nothing, but 0 * infinity is NaN: finite pairs alone
        fine = value.float().isfinite() & value.float().isfinite().roll(64, dims=-1)
        assert torch.equal(k.float()[fine], want.float()[fine]), scale
