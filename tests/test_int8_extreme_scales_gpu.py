"""Scales of the block-scaled 8-bit cache that no append of ordinary values writes: infinite, 0 and subnormal ones (GPU)."""

import math

import pytest
import torch
from int8_cases import random_cache
from test_int8_append_gpu import DTYPES, check, tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [128, 80, 65])
@pytest.mark.parametrize("old", [math.inf, 0.0, 2.0**-140, 2.0**-126, 2.0**-127, 3e38])
def test_appends_to_blocks_of_any_scale(dtype, d, old):
    """Codes are rounded anew where the scale changes, and stay where it does not: by single rows and by runs."""
    cache = random_cache(12, 16, 2, d, seed=5, layers=1)
    for scales in cache[2:]:
        scales[:8] = old
    blocks = torch.tensor([0, 1, 2, 3, 3, 3, 4, *[5] * 9, 6, 7, 8, 9, 9])
    offsets = torch.tensor([4, 15, 0, 9, 2, 7, 1, *range(1, 10), 0, 3, 8, 1, 6])
    k, v = tokens(len(blocks), 2, d, dtype, 3)
    k[0], v[6] = 0, 0
    check(cache, 0, blocks, offsets, k, v)
