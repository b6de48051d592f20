"""Tokens by top-p and min-p where the settings are at an end of their range."""
import math

import pytest
import torch

from test_sampling_nucleus_gpu import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("temperature", [math.inf, 3e38, 1e35, 1e10])
def test_high_temperatures(guard_regions, temperature):
    """All tokens alike: of a row of 5,000, and of the 50 and the 300 largest."""
    gen = torch.Generator().manual_seed(13)
    z = torch.randn((4, 5000), generator=gen) * 2.5
    for k in (0, 50, 300):
        check(z, [temperature] * 4, [k] * 4, [0.999, 0.7, 1.0, 0.5], [0.0, 0.0, 0.5, 0.9], torch.rand(4, generator=gen).tolist())
