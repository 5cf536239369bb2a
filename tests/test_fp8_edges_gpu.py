"""8-bit KV cache: arguments, values and batches at the ends of their ranges (GPU)."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("python", [False, True])
def test_chunk_tables_whose_rows_share_memory_are_refused(python, monkeypatch):
    from test_chunk_metadata_gpu import batch, buffers, expected
    from vllm_rlt_amd import ops

    if python:
        monkeypatch.setattr(ops, "_host_calls", lambda t: (None, 0))
    desc, tables = batch(3, 3, 2, 5, 16, 9, 1)
    outs = buffers(3, 40, 5)
    memory = torch.empty(11, dtype=torch.int32, device="cuda")
    for shared in (memory[:5].expand(3, 5), memory.unfold(0, 5, 3)):  # rows 0 and 3 entries apart
        with pytest.raises(ValueError, match="out_table_stride"):
            ops.build_chunk_metadata(desc.cuda(), 3, 3, tables.cuda(), 16, *outs[:6], shared, 5)
    # A single row has no stride of its own.
    one = torch.empty(1, 5, dtype=torch.int32, device="cuda").as_strided((1, 5), (0, 1))
    ops.build_chunk_metadata(desc[:1].cuda(), 1, 1, tables.cuda(), 16, *outs[:6], one, 5)
    assert torch.equal(one.cpu(), expected(desc, 1, 1, tables, 16, 40, 5)[-1])
