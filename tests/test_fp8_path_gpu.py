"""The 8-bit cache as a program uses it: slot maps, rotation and append, chunked prefill, decode, exit copies (GPU)."""

import torch
import pytest
from fp8_cases import assert_within, attention, quantise
from test_fp8_append_gpu import rotary_table, rotate

pytestmark = pytest.mark.gpu


def test_chunks_then_decode_steps_over_one_cache():
    from vllm_rlt_amd import ops

    g = torch.Generator().manual_seed(0)
    slots, planes, width, page, hq, hkv, d, layers, layer = 5, 2, 12, 16, 8, 4, 128, 2, 1
    blocks = slots * planes * width
    resident = torch.randperm(blocks, generator=g).to(torch.int32).view(slots, planes, width)
    codes = [torch.full((blocks, layers, page, hkv, d), 0x7F, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2)]
    scales = [torch.full((blocks, layers, page, hkv), 0xFF, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu) for _ in range(2)]
    table, axis_map = rotary_table(64, 4096), (0,) * 24 + (1,) * 20 + (2,) * 20
    dev_table, dev_resident = table.cuda(), resident.cuda()
    history = {}  # (slot, depth): rotated keys and values of every token so far, in float32

    def step(desc):
        """One batch of chunks (single tokens among them) through the whole path."""
        desc = torch.tensor(desc)
        n, capacity = len(desc), int(desc[:, 3].sum()) + 7
        size = n + 1
        cu, lens = torch.empty(size + 1, dtype=torch.int32, device="cuda"), torch.empty(size, dtype=torch.int32, device="cuda")
        pos, seq, wb, wo = (torch.empty(capacity, dtype=torch.int64, device="cuda") for _ in range(4))
        tables = torch.empty(size, width, dtype=torch.int32, device="cuda")
        ops.build_chunk_metadata(desc.pin_memory(), n, size, dev_resident, page, cu, lens, pos, seq, wb, wo, tables, width)
        q, k, v = (torch.randn(capacity, h, d, generator=g).bfloat16() for h in (hq, hkv, hkv))
        spots = torch.stack([pos, pos // 2, pos % 7], 1)
        turned = ops.rope_axes_kv_append(*codes, layer, wb, wo, q.cuda(), k.cuda(), v.cuda(), spots, dev_table, axis_map, *scales)
        out = torch.full_like(turned, 9.0)
        cache = [*(c[:, layer] for c in codes), *(s[:, layer] for s in scales)]
        if int(desc[:, 3].max()) > 1:
            ops.paged_prefill_fp8(turned, *cache, tables, lens, cu, int(desc[:, 3].max()), out=out)
        else:
            ops.paged_decode_fp8(turned[:n], *cache, tables[:n], lens[:n], out=out[:n])
        total = int(desc[:, 3].sum())
        assert (out[total:] == 9.0).all()
        # The definition: quantised history of every request, attention in 64 bits.
        at = 0
        for slot, depth, start, count in desc.tolist():
            rows = slice(at, at + count)
            p = torch.arange(start, start + count)
            p = torch.stack([p, p // 2, p % 7], 1)
            assert torch.equal(turned[rows].cpu(), rotate(q[rows], p, table, axis_map).bfloat16())
            old = history.get((slot, depth), (torch.empty(0, hkv, d), torch.empty(0, hkv, d)))
            assert len(old[0]) == start
            keys = torch.cat([old[0], rotate(k[rows], p, table, axis_map)])
            vals = torch.cat([old[1], v[rows].float()])
            history[slot, depth] = keys, vals
            flat = [torch.zeros(-(-len(keys) // page) * page, hkv, d) for _ in range(2)]
            flat[0][: len(keys)], flat[1][: len(keys)] = keys, vals
            (kc, ks), (vc, vs) = (quantise(x.view(-1, page, hkv, d)) for x in flat)
            mine = [t.cuda() for t in (kc, vc, ks, vs)]
            limits = list(range(start + 1, start + count + 1))
            want = attention(turned[rows], mine, torch.arange(kc.shape[0], device="cuda"), limits, d**-0.5, 2.0**-8)
            assert_within(out[rows], *want)
            at += count

    step([[0, 0, 0, 70], [3, 1, 0, 17], [2, 0, 0, 1]])
    step([[0, 0, 70, 60], [1, 1, 0, 33], [3, 1, 17, 2]])
    step([[3, 1, 19, 1], [0, 0, 130, 1], [2, 0, 1, 1], [1, 1, 33, 1]])
    step([[0, 0, 131, 1], [2, 0, 2, 1]])


def test_exit_copies_and_gathers_move_the_cache_as_bytes():
    """The framework's exit copies and ordered gathers serve an 8-bit cache through 16-bit views of its codes and scales."""
    from vllm_rlt_amd import ops

    g = torch.Generator().manual_seed(1)
    blocks, layers, page, hkv, d = 9, 2, 16, 4, 128
    codes = [torch.randint(0, 256, (blocks, layers, page, hkv, d), generator=g, dtype=torch.uint8).cuda() for _ in range(2)]
    scales = [torch.randint(0, 255, (blocks, layers, page, hkv), generator=g, dtype=torch.uint8).cuda() for _ in range(2)]
    before = [t.clone() for t in codes + scales]
    tables = torch.tensor([[[3, 4], [5, 6]]], dtype=torch.int32, device="cuda")  # one slot, two planes
    desc = torch.tensor([[0, 0, 21]], device="cuda")
    views = [t.view(torch.float16) for t in codes], [t.view(torch.float16).unsqueeze(3) for t in scales]
    for pair in views:
        ops.kv_finalize(desc, tables, *pair, 2)
    for t, old in zip(codes + scales, before):
        want = old.clone()
        want[6, :, 5] = old[4, :, 5]
        assert torch.equal(t, want)
    k, _ = ops.kv_gather(*views[0], 1, tables[0, 1], 30)
    assert torch.equal(k.view(torch.uint8), codes[0][tables[0, 1].long(), 1].flatten(0, 1)[:30])
