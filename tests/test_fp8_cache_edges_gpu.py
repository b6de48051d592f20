"""The cache in 8 bits at the ends of its ranges: numbers of every size, scratch memory of exactly the size asked for, launches counted."""
import ctypes
import math

import pytest
import torch

import plain_fp8_cache as plain
from qwen_decoder_b200 import kernels
from test_fp8_cache_gpu import a_cache, check_prefill, check_write

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def test_write_of_the_largest_and_the_smallest_numbers(guard_regions):
    """Every scale that there is, from 2^-126 to that of the largest float32 number; q is zeros."""
    H, G, d, ps = 1, 1, 64, 16
    gen = torch.Generator().manual_seed(41)
    x = torch.zeros((255, 3 * d))
    sizes = torch.exp2(torch.arange(-126, 129, dtype=torch.float64)).clamp(max=torch.finfo(torch.float32).max)
    x[:, d:] = (sizes[:, None] * (torch.rand((255, 2 * d), generator=gen, dtype=torch.float64) * 2 - 1)).float()
    x[:, d + 7] = x[:, 2 * d + 9] = sizes.float()
    x[-1, 2 * d + 9] = -torch.finfo(torch.float32).max
    check_write(x, None, H, G, d, 0, True, ps, torch.randperm(255, generator=gen).to(torch.int32), 16)
