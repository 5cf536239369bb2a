"""Block-scaled decode of batches so large that a workgroup walks several splits of its row (GPU).

A launch has at most 32768 workgroups: of 520 rows x 16 KV heads, three for the eight splits of 4096 keys.
"""

import pytest
import torch
from test_int8_attention_gpu import DTYPES, Case

pytestmark = pytest.mark.gpu

# Last splits that are full, and ones so short that some waves have no tile of theirs; rows of few splits and of none.
LENGTHS = [4096, 4095, 3585, 3600, 3617, 2049, 1537, 1600, 2081, 1, 0, 700, 512, 513, 3072 + 97, 2560]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d", [(16, 16, 64), (16, 16, 128), (16, 16, 80), (8, 8, 256), (40, 20, 112)])
def test_rows_of_a_large_batch_have_the_bits_of_a_small_one(dtype, hq, hkv, d):
    from vllm_rlt_amd import ops

    c = Case(LENGTHS, hq, hkv, d, dtype=dtype, seed=d)
    small = c.decode()
    c.check(small)
    times = 33 if hkv > 8 else 66
    rows = torch.arange(len(LENGTHS), device="cuda").repeat(times)
    rows = rows[torch.randperm(len(rows), generator=torch.Generator().manual_seed(1)).cuda()]
    items, splits = len(rows) * hkv, 8
    assert items * splits > 32768 and 32768 // items < splits
    for _ in range(3):
        large = ops.paged_decode_int8(c.q[rows], *c.cache, c.tables[rows], c.lens[rows], scale=c.scale)
        assert torch.equal(large, small[rows])


def test_a_captured_call_walks_them_again():
    from vllm_rlt_amd import ops

    c = Case(LENGTHS, 16, 16, 128, seed=3)
    rows = torch.arange(len(LENGTHS), device="cuda").repeat(33)
    q, tables, lens = c.q[rows], c.tables[rows], c.lens[rows]
    ws = torch.empty(ops.decode_int8_workspace_bytes(len(rows), tables.shape[1], 16, 16, 128, 16), dtype=torch.uint8, device="cuda")
    out = torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.paged_decode_int8(q, *c.cache, tables, lens, scale=c.scale, out=out, workspace=ws)
    for shorter in (0, 5, 600):
        c.lens.copy_(torch.tensor([max(n - shorter, 0) for n in LENGTHS], dtype=torch.int32))
        lens.copy_(c.lens[rows])
        out.fill_(7), ws.fill_(255)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, c.decode()[rows])
