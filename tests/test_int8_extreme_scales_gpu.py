"""Scales of the block-scaled 8-bit cache that no append of ordinary values writes: infinite, 0 and subnormal ones (GPU)."""

import math

import pytest
import torch
from int8_cases import random_cache
from test_int8_append_gpu import DTYPES, check, tokens
from test_int8_attention_gpu import Case

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


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d", [(4, 4, 128), (8, 2, 128), (4, 4, 64), (2, 2, 80), (2, 2, 256), (2, 2, 72)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("which", [2, 3])
def test_rows_that_see_a_block_of_no_finite_scale_are_nan_whole(dtype, hq, hkv, d, bad, which):
    from vllm_rlt_amd import ops

    c = Case([150, 90], hq, hkv, d, dtype=dtype, seed=8, chunks=[100, 90])
    clean = c.prefill()
    h = hkv - 1  # block 7 of sequence 0, its keys 112 to 127, is seen by its rows from 62 on
    c.cache[which][int(c.tables[0, 7]), h] = bad
    for codes in c.cache[:2]:  # codes of 0 among them: infinity times them would be NaN, and times the others not
        codes[int(c.tables[0, 7]), :, h, ::3] = 0
    heads = slice(h * (hq // hkv), hq)
    touched = torch.zeros(clean.shape[:2], dtype=torch.bool, device="cuda")
    touched[62:100, heads] = True
    for out in (c.prefill(), c.prefill(batch_invariant=True)):
        assert out[touched].isnan().all() and out[~touched].isfinite().all()
    lens = torch.tensor([112, 113, 128, 150, 90], dtype=torch.int32, device="cuda")
    out = ops.paged_decode_int8(c.q[:5].contiguous(), *c.cache, c.tables[[0, 0, 0, 0, 1]].contiguous(), lens, scale=c.scale)
    assert out[1:4, heads].isnan().all() and out[[0, 4]].isfinite().all()
