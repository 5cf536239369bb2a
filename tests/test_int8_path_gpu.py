"""The block-scaled 8-bit cache as a program uses it: slot maps, append, chunked prefill, decode, exit copies (GPU).

A plain cache on the CPU follows every append by its definition; the device's cache has to
hold the same bits after each step, and attention is compared in 64 bits over it.
"""

import pytest
import torch
from fp8_cases import assert_within
from int8_cases import append, attention, values
from test_int8_append_gpu import same

pytestmark = pytest.mark.gpu
SLOTS, PLANES, WIDTH, PAGE, HQ, HKV, D, LAYERS, LAYER = 5, 2, 12, 16, 8, 4, 128, 2, 1


class Program:
    """Two loop depths ("planes") of a few requests, their blocks anywhere in the pool, nothing initialised."""

    def __init__(self, dtype, seed):
        self.g, self.dtype = torch.Generator().manual_seed(seed), dtype
        blocks = SLOTS * PLANES * WIDTH
        self.tables = torch.randperm(blocks, generator=self.g).to(torch.int32).view(SLOTS, PLANES, WIDTH)
        shape = (blocks, LAYERS, PAGE, HKV, D)
        codes = [torch.randint(-127, 128, shape, generator=self.g, dtype=torch.int8) for _ in "kv"]
        scales = [torch.full((blocks, LAYERS, HKV), float("nan")) for _ in "kv"]
        self.plain = [*codes, *scales]
        self.cache = [t.cuda() for t in self.plain]
        self.dev_tables = self.tables.cuda()

    def step(self, desc):
        """One batch of chunks, (slot, plane, first position, tokens) each, through slot maps, append and attention."""
        from vllm_rlt_amd import ops

        desc = torch.tensor(desc)
        n, total = len(desc), int(desc[:, 3].sum())
        capacity, size = total + 7, n + 1
        cu, lens = torch.empty(size + 1, dtype=torch.int32, device="cuda"), torch.empty(size, dtype=torch.int32, device="cuda")
        pos, seq, wb, wo = (torch.empty(capacity, dtype=torch.int64, device="cuda") for _ in range(4))
        tables = torch.empty(size, WIDTH, dtype=torch.int32, device="cuda")
        ops.build_chunk_metadata(desc.pin_memory(), n, size, self.dev_tables, PAGE, cu, lens, pos, seq, wb, wo, tables, WIDTH)
        # Tokens grow from step to step, so that scales move and held codes are rounded again.
        q, k, v = ((torch.randn(capacity, h, D, generator=self.g) * (1 + pos[:, None, None].cpu() / 16)).to(self.dtype) for h in (HQ, HKV, HKV))
        q = (q / 4).cuda()
        ops.kv_append_int8(*self.cache, LAYER, wb, wo, k.cuda(), v.cuda())
        append(self.plain, LAYER, wb.cpu(), wo.cpu(), k, v)
        same(self.cache, self.plain)
        at = [t[:, LAYER] for t in self.cache]
        out = torch.full_like(q, 9.0)
        most = int(desc[:, 3].max())
        if most > 1:
            ops.paged_prefill_int8(q, *at, tables, lens, cu, most, out=out)
        else:
            ops.paged_decode_int8(q[:n], *at, tables[:n], lens[:n], out=out[:n])
        assert (out[total:] == 9.0).all()
        row = 0
        for slot, plane, start, count in desc.tolist():
            limits = list(range(start + 1, start + count + 1))
            rows = slice(row, row + count)
            assert_within(out[rows], *attention(q[rows], at, self.dev_tables[slot, plane], limits, D**-0.5))
            row += count

    def copy(self, tokens, source, target):
        """Tokens (slot, position) of plane `source` into plane `target`: read back, then appended."""
        from vllm_rlt_amd import ops

        slots, positions = (torch.tensor(x) for x in zip(*tokens))
        page, offset = positions // PAGE, positions % PAGE
        src, dst = (self.tables[slots, p, page].long() for p in (source, target))
        for layer in range(LAYERS):
            k, v = ops.kv_gather_int8(*self.cache, layer, src.cuda(), offset.cuda(), dtype=torch.float32)
            plain = [values(c, s)[src, layer, offset].float() for c, s in zip(self.plain[:2], self.plain[2:])]
            for got, want in zip((k, v), plain):
                assert torch.equal(got.cpu().nan_to_num(7.0), want.nan_to_num(7.0))
            ops.kv_append_int8(*self.cache, layer, dst.cuda(), offset.cuda(), k, v)
            append(self.plain, layer, dst, offset, *plain)
        same(self.cache, self.plain)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_chunks_exit_copies_and_decode_steps_over_one_cache(dtype):
    p = Program(dtype, 0)
    p.step([[0, 0, 0, 70], [3, 1, 0, 17], [2, 0, 0, 1]])
    p.copy([(0, i) for i in range(70)], 0, 1)  # a prompt that left the loop after the first depth
    p.step([[0, 0, 70, 60], [1, 1, 0, 33], [3, 1, 17, 2], [0, 1, 70, 9]])
    p.step([[3, 1, 19, 1], [0, 0, 130, 1], [2, 0, 1, 1], [1, 1, 33, 1]])
    p.copy([(2, 0), (2, 1), (0, 79)], 0, 1)  # single tokens, into blocks that they begin and that go on
    p.step([[0, 0, 131, 1], [2, 0, 2, 1], [2, 1, 2, 1], [0, 1, 80, 1]])


def test_a_block_that_is_given_back_begins_again():
    """What a block held, a scale of NaN included, does not reach the next sequence that owns it."""
    from vllm_rlt_amd import ops

    p = Program(torch.bfloat16, 1)
    for scale in p.cache[2:] + p.plain[2:]:
        scale.fill_(float("inf"))
    p.step([[0, 0, 0, 40]])
    p.step([[0, 0, 0, 20], [1, 0, 0, 1]])
    blocks = p.tables[0, 0, :2].long().cuda().repeat_interleave(PAGE)[:20]
    k, _ = ops.kv_gather_int8(*p.cache, LAYER, blocks, torch.arange(20, device="cuda") % PAGE)
    assert k.isfinite().all()


def test_pages_move_as_bytes():
    """Codes and scales of a page copied by indexing serve the copy's table."""
    from vllm_rlt_amd import ops

    p = Program(torch.bfloat16, 2)
    p.step([[0, 0, 0, 50]])
    old, new = p.tables[0, 0, :4].long().cuda(), p.tables[4, 1, :4].long().cuda()
    for t in p.cache:
        t[new] = t[old]
    at = [t[:, LAYER] for t in p.cache]
    q = torch.randn(2, HQ, D, generator=p.g).bfloat16().cuda()[:1].repeat(2, 1, 1)
    lens = torch.tensor([50, 50], dtype=torch.int32, device="cuda")
    out = ops.paged_decode_int8(q, *at, torch.stack([old, new]).int(), lens)
    assert torch.equal(out[0], out[1])
