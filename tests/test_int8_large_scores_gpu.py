"""Attention over the block-scaled cache at scores of any size, from finite queries and scales (GPU).

Every score is a whole number times one factor, and sums of products are exact: keys of the same
score tie to the bit, and the others are so far below that they weigh nothing.  So the result
is the mean of the values of the row's best keys, to the rounding of weights and outputs alone.
"""

import math

import pytest
import torch
from fp8_cases import assert_within
from int8_cases import values
from test_int8_attention_gpu import DTYPES, Case

pytestmark = pytest.mark.gpu
SHAPES = [(4, 4, 128), (8, 2, 64), (2, 2, 256), (6, 2, 80), (2, 2, 72)]  # (72: the kernel for any shape)


class Large(Case):
    """Queries of one number a row, keys of one code each (larger and larger ones) in blocks of scales 1, 2 and 4 times one
    that puts the largest scores near 2^power in binary orders."""

    def __init__(self, power, lengths, hq, hkv, d, dtype, chunks=None):
        super().__init__(lengths, hq, hkv, d, dtype=dtype, seed=d, chunks=chunks)
        g = torch.Generator().manual_seed(power)
        self.rows = torch.randint(1, 8, self.q.shape[:2], generator=g).double() * torch.where(torch.rand(self.q.shape[:2], generator=g) < 0.2, -1, 1)
        self.q.copy_(self.rows[..., None].expand(self.q.shape))
        self.scale = 0.7 / math.sqrt(d)
        unit = 0.77 * 2.0 ** (power - math.ceil(math.log2(7 * 100 * 4 * d * self.scale / math.log(2))))
        self.codes = []  # of each sequence's keys, [hkv, keys]; with the block's 1, 2 or 4
        for s, n in enumerate(lengths):
            n = max(n, 0)
            ids = self.tables[s, : -(-n // 16)].long().cpu()
            code = torch.randint(1, 50, (len(ids) * 16, hkv), generator=g) + torch.arange(len(ids) * 16)[:, None] * 50 // max(len(ids) * 16, 1)
            grow = torch.randint(0, 3, (len(ids), hkv), generator=g)
            self.cache[0][ids.cuda()] = code.view(-1, 16, hkv, 1).expand(-1, -1, -1, d).to(torch.int8).cuda()
            self.cache[2][ids.cuda()] = (unit * 2.0**grow).float().cuda()
            self.codes.append((code * 2 ** grow.repeat_interleave(16, 0))[:n].t().double())

    def best(self, rows, s, limits):
        """(result, bound) of packed rows of sequence s that see so many keys."""
        kc, vc, ks, vs = self.cache
        group = self.q.shape[1] // kc.shape[2]
        n = max(limits)
        ids = self.tables[s, : -(-n // 16)].long()
        v = values(vc[ids], vs[ids]).flatten(0, 1)[:n].transpose(0, 1).repeat_interleave(group, 0).cpu()  # [hq, keys, d]
        score = self.rows[rows].t()[..., None] * self.codes[s][:, :n].repeat_interleave(group, 0)[:, None]  # [hq, rows, keys]
        score = score.masked_fill(torch.arange(n) >= torch.tensor(limits)[:, None], -math.inf)
        won = (score == score.amax(-1, keepdim=True)).double()
        p = won / won.sum(-1, keepdim=True)
        out, spread = p @ v, p @ v.abs()
        # A weight is rounded by half a step of fp16, or of two parts of it (whose second one is off by up to 2^-30 of the
        # largest as well, times codes of up to 128); 2^-20 for the sums and joins; the result by half a step.
        dtype = self.q.dtype
        bound = torch.finfo(dtype).eps / 2 * out.abs() + (2.0**-20 + (2.0**-22 if dtype == torch.float32 else 2.0**-11)) * spread
        bound = bound + (won.sum(-1, keepdim=True) * vs[ids].double().max().item() * 128 * 2.0**-30 if dtype == torch.float32 else 0)
        return out.transpose(0, 1).cuda(), bound.transpose(0, 1).cuda()

    def check(self, out):
        torch.cuda.synchronize()
        at = 0
        for s, (n, c) in enumerate(zip(self.lengths, self.chunks or [1] * len(self.lengths))):
            rows = slice(at, at + c)
            assert_within(out[rows], *self.best(rows, s, [n - c + i + 1 for i in range(c)]))
            at += c


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
@pytest.mark.parametrize("power", [24, 28, 30, 31, 60, 100])
def test_the_best_keys_share_the_weight(dtype, hq, hkv, d, power):
    # Tiles that every row sees, then masked ones; cut sequences and whole ones; the maximum moves from tile to tile.
    c = Large(power, [700, 4000, 65, 130], hq, hkv, d, dtype, chunks=[100, 40, 65, 2])
    c.check(c.prefill())
    c.check(c.prefill(batch_invariant=True))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
@pytest.mark.parametrize("power", [24, 28, 31, 60, 100])
def test_decode_of_the_best_keys(dtype, hq, hkv, d, power):
    c = Large(power, [1, 16, 33, 700, 1500, 4000], hq, hkv, d, dtype)
    c.check(c.decode())
