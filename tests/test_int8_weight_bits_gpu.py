"""Weights of block-scaled attention that go into the products in two parts of 11 bits: the result is the 64-bit one's to its
own rounding and what 32-bit sums lose, also where large values cancel (GPU)."""

import pytest
import torch
from fp8_cases import assert_within
from int8_cases import attention
from test_int8_attention_gpu import DTYPES, Case

pytestmark = pytest.mark.gpu
SHAPES = [(4, 4, 128), (8, 2, 128), (4, 4, 64), (2, 2, 256), (6, 2, 80)]


def check(c, out):
    """As Case.check, with weights off by 2^-22 of their size, and 2^-30 of the row's largest (a second part below fp16's normal
    numbers), times codes of up to 128."""
    torch.cuda.synchronize()
    at = 0
    for s, (n, rows) in enumerate(zip(c.lengths, c.chunks or [1] * len(c.lengths))):
        here = slice(at, at + rows)
        want, bound = attention(c.q[here], c.cache, c.tables[s], [n - rows + i + 1 for i in range(rows)], c.scale, weight_unit=2.0**-22)
        ids = c.tables[s, : -(-n // 16)].long()
        largest = c.cache[3][ids].double().amax(0).repeat_interleave(c.q.shape[1] // c.cache[3].shape[1])
        assert_within(out[here], want, bound + n * 128 * 2.0**-30 * largest[None, :, None])
        at += rows


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
def test_decode(dtype, hq, hkv, d):
    c = Case([1, 17, 100, 300, 700, 1300], hq, hkv, d, dtype=dtype, seed=d, spread=0.5)
    check(c, c.decode())


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
def test_prefill(dtype, hq, hkv, d):
    c = Case([70, 300, 2000, 33], hq, hkv, d, dtype=dtype, seed=d, spread=0.5, chunks=[30, 130, 40, 33])
    check(c, c.prefill())
    check(c, c.prefill(batch_invariant=True))
