"""The scales that a calibration takes for an 8-bit cache, on the CPU."""

from __future__ import annotations

import pytest
import torch
from trianglemix import cached


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("odd", [float("nan"), float("inf"), -float("inf")])
def test_numbers_that_are_not_finite_give_no_scale(dtype, odd):
    """The largest of the finite ones counts; a head without any has the scale 1."""
    x = torch.zeros(4, 3, 128, dtype=dtype)
    x[1, 0, 4], x[2, 0, 9] = -896.0, odd
    x[3, 1, 7] = odd
    x[0, 2, 1] = 112.0
    assert torch.equal(cached.head_scales(x), torch.tensor([2.0, 1.0, 0.25]))


def test_scales_stay_in_the_range_that_caches_take():
    x = torch.zeros(2, 2, 128, dtype=torch.bfloat16)
    x[0, 0, 0], x[1, 1, 1] = torch.finfo(torch.bfloat16).max, 1.0
    assert torch.equal(cached.head_scales(x, margin=1e6), torch.tensor([2.0 ** 126, 1e6 / 448]))
