"""The 8-bit cache's calls checked and launched from C++ give the Python path's results and errors (GPU)."""

import pytest
import torch
from fp8_cases import random_cache, tables_for
from test_fp8_append_gpu import rotary_table, same_bits

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["host calls", "python"])
def path(request, monkeypatch):
    from vllm_rlt_amd import ops

    if request.param == "python":
        monkeypatch.setattr(ops, "_host_calls", lambda t: (None, 0))
    return request.param


def both(monkeypatch, call):
    """The call's result by both paths."""
    from vllm_rlt_amd import ops

    first = call()
    with monkeypatch.context() as m:
        m.setattr(ops, "_host_calls", lambda t: (None, 0))
        second = call()
    return first, second


def test_the_host_calls_are_taken(monkeypatch):
    """No call of ordinary tensors goes through the Python launch."""
    from vllm_rlt_amd import _native, ops

    class Lib:
        def __getattr__(self, name):
            raise AssertionError(f"{name} went through Python")

    _native.load()
    c = Calls()
    monkeypatch.setattr(_native, "_lib", Lib())
    c.decode(), c.prefill(), c.append(), c.rope(), c.slots()
    torch.cuda.synchronize()
    assert ops is not None


class Calls:
    def __init__(self):
        tables, blocks = tables_for([40, 700], 16, 1)
        self.pool = [t.cuda() for t in random_cache(blocks, 16, 4, 64, layers=2)]
        self.layer = [t[:, 1] for t in self.pool]
        self.tables, self.lens = tables.cuda(), torch.tensor([40, 700], dtype=torch.int32, device="cuda")
        g = torch.Generator().manual_seed(0)
        self.q = torch.randn(50, 8, 64, generator=g).bfloat16().cuda()
        self.k = torch.randn(50, 4, 64, generator=g).bfloat16().cuda()
        self.cu = torch.tensor([0, 20, 50], dtype=torch.int32, device="cuda")
        self.wb = torch.arange(50, device="cuda") % blocks
        self.wo = torch.arange(50, device="cuda") % 16
        self.table = rotary_table(32, 64, "cuda")
        self.positions = torch.arange(50, device="cuda")[:, None].repeat(1, 2)

    def decode(self, **kw):
        from vllm_rlt_amd import ops

        return ops.paged_decode_fp8(self.q[:2], *self.layer, self.tables, self.lens, **kw)

    def prefill(self, **kw):
        from vllm_rlt_amd import ops

        return ops.paged_prefill_fp8(self.q, *self.layer, self.tables, self.lens, self.cu, 30, **kw)

    def append(self, **kw):
        from vllm_rlt_amd import ops

        ops.kv_append_fp8(*self.pool, 0, self.wb, self.wo, self.k, self.k, **kw)
        return [t.clone() for t in self.pool]

    def rope(self, axes=(0,) * 16 + (1,) * 16, **kw):
        from vllm_rlt_amd import ops

        out = ops.rope_axes_kv_append(*self.pool[:2], 0, self.wb, self.wo, self.q, self.k, self.k, self.positions, self.table, axes,
                                      *self.pool[2:], **kw)
        return [out, *(t.clone() for t in self.pool)]

    def slots(self):
        from vllm_rlt_amd import ops

        resident = self.tables.clamp(min=0)[:, None].contiguous()
        desc = torch.tensor([[0, 0, 3, 9], [1, 0, 100, 30]], device="cuda")
        short = lambda *n: torch.empty(n, dtype=torch.int32, device="cuda")  # noqa: E731
        long = lambda: torch.empty(44, dtype=torch.int64, device="cuda")  # noqa: E731
        outs = [short(3), short(2), long(), long(), long(), long(), short(2, resident.shape[2])]
        for d in (desc, desc.cpu().pin_memory()):
            ops.build_chunk_metadata(d, 2, 2, resident, 16, *outs, resident.shape[2])
        return outs


def test_both_paths_give_the_same_bits(monkeypatch):
    c = Calls()
    out = torch.empty_like(c.q)
    ws = torch.empty(1 << 24, dtype=torch.uint8, device="cuda")
    for call in (
        c.decode, lambda: c.decode(scale=0.25), lambda: c.decode(workspace=ws, out=out[:2]), c.prefill,
        lambda: c.prefill(out=out, workspace=ws, scale=0.3), lambda: c.prefill(batch_invariant=True), c.append,
        lambda: c.append(n_rows=7), c.rope, lambda: c.rope(n_rows=3, out=out), lambda: c.rope(axes=[0] * 32), c.slots,
    ):
        a, b = both(monkeypatch, call)
        a, b = (x if isinstance(x, list) else [x] for x in (a, b))
        assert len(a) == len(b) and all(same_bits(x, y) for x, y in zip(a, b))


def test_errors_are_the_same(path):
    c = Calls()
    with pytest.raises(ValueError, match="n_rows"):
        c.append(n_rows=51)
    with pytest.raises(ValueError):
        c.append(n_rows=-1)
    with pytest.raises(ValueError, match="axis past the last"):
        c.rope(axes=(3,) * 32)
    with pytest.raises(ValueError, match="out must match"):
        c.decode(out=c.q[:3])
    with pytest.raises(ValueError, match="workspace"):
        c.decode(workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    for call in (c.decode, c.prefill):  # numbers one above the other, the memory of one
        with pytest.raises(ValueError, match="workspace"):
            call(workspace=torch.empty(1, dtype=torch.uint8, device="cuda").expand(1 << 24))
    c.lens = c.lens.long()
    with pytest.raises(ValueError, match="context_lengths"):
        c.prefill()
