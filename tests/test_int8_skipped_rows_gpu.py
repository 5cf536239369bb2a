"""Appends to the block-scaled 8-bit cache with rows that are skipped between the rows of a block (GPU).

A row is skipped whose block is outside the pool or whose offset is outside its page: padding, or a
token that was taken out of a batch.  The rows around it are one block's all the same, and its scale and codes
are the definition's, which knows no order.
"""

import pytest
import torch
from int8_cases import random_cache
from test_int8_append_gpu import DTYPES, check, slots, tokens

pytestmark = pytest.mark.gpu
SHAPES = [(4, 128, 16), (3, 64, 16), (2, 256, 16), (1, 512, 16), (2, 80, 32), (2, 128, 64), (1, 128, 256), (2, 65, 16), (1, 36, 100), (2, 128, 5)]


def skip(blocks, offsets, rows, page, pool):
    """Every way in which a row is of no slot, in turn, a valid block among them."""
    ways = [(-1, 3), (pool, 0), (1 << 40, 1), (0, -1), (pool - 1, page), (1, 1 << 33), (-(1 << 35), 0)]
    for i, r in enumerate(rows):
        blocks[r], offsets[r] = ways[i % len(ways)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hkv,d,page", SHAPES)
@pytest.mark.parametrize("part", [0.1, 0.5, 0.93])
def test_tokens_taken_out_of_chunks(dtype, hkv, d, page, part):
    print(f"[skipped] {dtype} {hkv} x {d} page {page} {part}", flush=True)
    runs = [(0, 1), (page - 1, 3), (0, page), (page // 2, page), (page // 3, 2 * page + 1), (0, 3), (page // 2, 70), (0, 9)]
    pool = sum(-(-(f + n) // page) for f, n in runs) + 3
    blocks, offsets = slots(runs, page, pool, seed=page)
    g = torch.Generator().manual_seed(int(part * 100))
    out = (torch.rand(len(blocks), generator=g) < part).nonzero()[:, 0].tolist()
    skip(blocks, offsets, out, page, pool)
    k, v = tokens(len(blocks), hkv, d, dtype, seed=hkv, spread=3.0)
    check(random_cache(pool, page, hkv, d, seed=d, layers=2), 1, blocks, offsets, k, v)


@pytest.mark.parametrize("d", [128, 64, 256, 65])
@pytest.mark.parametrize("later", [8.0, 0.125])
def test_a_skipped_row_between_two_of_a_block(d, later):
    cache = random_cache(6, 16, 2, d, seed=1, layers=1)
    k, v = tokens(4, 2, d, torch.bfloat16, 2)
    k[2:], v[2:] = k[2:] * later, v[2:] * later
    check(cache, 0, torch.tensor([3, -1, 3, 3]), torch.tensor([4, 0, 5, 6]), k, v)
    check(cache, 0, torch.tensor([3, 2, 3, 3]), torch.tensor([4, -1, 0, 6]), k, v)  # (a row of another block, of no offset)


@pytest.mark.parametrize("d,page", [(128, 16), (64, 16), (256, 16), (65, 16), (128, 64), (128, 128), (65, 128)])
def test_gaps_of_every_place_and_length(d, page):
    """A block's rows with up to 32 skipped ones between them, or a page's, at every place of a tile and a wave's sight."""
    most = max(32, page)
    for lead in (0, 1, 3, 9, 14, 15, 16, 31, 40, 47, 62, 63, 64):
        for gap in sorted({1, 2, 13, 30, most - 1, most}):
            n = lead + 3 + 2 * gap + 2
            pool = n + 4
            blocks, offsets = torch.arange(n) + 3, torch.full((n,), 2)
            blocks[[lead, lead + 1 + gap, lead + 2 + 2 * gap]] = 1
            offsets[[lead, lead + 1 + gap, lead + 2 + 2 * gap]] = torch.tensor([3, 1, 2])
            skip(blocks, offsets, [*range(lead + 1, lead + 1 + gap), *range(lead + 2 + gap, lead + 2 + 2 * gap)], page, pool)
            k, v = tokens(n, 1, d, torch.float16, seed=gap, spread=3.0)
            print(f"[skipped] {d} page {page}: {lead} rows, gaps of {gap}", flush=True)
            check(random_cache(pool, page, 1, d, seed=lead, layers=1), 0, blocks, offsets, k, v)


@pytest.mark.parametrize("d", [128, 64, 65])
def test_padding_before_and_behind_a_batch(d):
    for before, n, behind in [(0, 1, 300), (0, 40, 5000), (300, 20, 0), (70, 5, 1), (17, 33, 100), (0, 0, 200), (1000, 64, 1000)]:
        total = before + n + behind
        blocks, offsets = torch.full((total,), -1), torch.zeros(total, dtype=torch.int64)
        at = 5 + torch.arange(n)
        blocks[before : before + n], offsets[before : before + n] = 3 + at // 16, at % 16
        k, v = tokens(total, 2, d, torch.bfloat16, seed=n, spread=2.0)
        check(random_cache(10, 16, 2, d, seed=n, layers=1), 0, blocks, offsets, k, v)
        blocks[before : before + n], offsets[before : before + n] = torch.arange(n) % 70, 7  # a block each
        check(random_cache(70, 16, 2, d, seed=n, layers=1), 0, blocks, offsets, k, v)
