"""Slot maps and block tables of packed chunks against plain integer loops (GPU): every value exact."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def expected(desc, count, size, tables, page, capacity, width):
    slots, planes, table_width = tables.shape
    cu, lengths = [0], []
    positions, sequences, blocks, offsets = [0] * capacity, [-1] * capacity, [-1] * capacity, [0] * capacity
    out = torch.zeros(size, width, dtype=torch.int32)
    for i in range(size):
        slot, depth, start, tokens = desc[i].tolist() if i < count else (0, 0, 0, 0)
        plane = depth if planes > 1 else 0
        valid = (i < count and 0 <= slot < slots and 0 <= plane < planes and start >= 0 and tokens >= 0
                 and start + tokens <= table_width * page)
        first = cu[-1]
        n = min(max(tokens, 0), capacity - first)
        lengths.append(start + n if valid else 0)
        cu.append(first + n)
        if valid:
            out[i] = tables[slot, plane, :width]
        for t in range(n):
            pos = start + t if valid else 0
            positions[first + t], sequences[first + t] = pos, i
            blocks[first + t] = int(tables[slot, plane, pos // page]) if valid else -1
            offsets[first + t] = pos % page
    long = lambda x: torch.tensor(x, dtype=torch.int64)  # noqa: E731
    return (torch.tensor(cu, dtype=torch.int32), torch.tensor(lengths, dtype=torch.int32), long(positions), long(sequences),
            long(blocks), long(offsets), out)


def buffers(size, capacity, width, spare=3):
    """Outputs filled with 77, a little larger than asked (the token buffers are the capacity itself)."""
    short = lambda *n: torch.full(n, 77, dtype=torch.int32, device="cuda")  # noqa: E731
    long = lambda: torch.full((capacity,), 77, dtype=torch.int64, device="cuda")  # noqa: E731
    return [short(size + 1 + spare), short(size + spare), long(), long(), long(), long(), short(size + spare, width + spare)]


def build(desc, count, size, tables, page, outs, width, pinned):
    from vllm_rlt_amd import ops

    d = desc.pin_memory() if pinned and len(desc) else desc.cuda()
    ops.build_chunk_metadata(d, count, size, tables.cuda(), page, *outs, width)
    torch.cuda.synchronize()


def check(desc, count, size, tables, page, capacity, width, pinned=False):
    outs = buffers(size, capacity, width)
    build(desc, count, size, tables, page, outs, width, pinned)
    cu, lengths, *tokens, rows = expected(desc, count, size, tables, page, capacity, width)
    for got, want, n in ((outs[0], cu, size + 1), (outs[1], lengths, size)):
        assert torch.equal(got[:n].cpu(), want) and (got[n:] == 77).all()
    for got, want in zip(outs[2:6], tokens):
        assert torch.equal(got.cpu(), want)
    assert torch.equal(outs[6][:size, :width].cpu(), rows)
    assert (outs[6][size:] == 77).all() and (outs[6][:, width:] == 77).all()


def batch(n, slots, planes, width, page, longest, seed):
    g = torch.Generator().manual_seed(seed)
    tables = torch.randint(0, 5000, (slots, planes, width), generator=g, dtype=torch.int32)
    tokens = torch.randint(0, longest + 1, (n,), generator=g)
    start = (torch.rand(n, generator=g) * (width * page - tokens + 1)).long()
    desc = torch.stack([torch.randint(0, slots, (n,), generator=g), torch.randint(0, planes, (n,), generator=g), start, tokens], 1)
    return desc.contiguous(), tables


@pytest.mark.parametrize("pinned", [False, True])
@pytest.mark.parametrize("n,planes,width,page,longest", [(1, 1, 1, 16, 1), (1, 4, 300, 16, 4000), (8, 4, 64, 16, 512), (3, 1, 9, 5, 40), (65, 4, 40, 16, 70), (300, 2, 33, 16, 9), (700, 1, 20, 1, 2)])
@pytest.mark.parametrize("room", [0, 37])
def test_equals_the_definition(pinned, n, planes, width, page, longest, room):
    desc, tables = batch(n, n + 2, planes, width, page, longest, n)
    capacity = int(desc[:, 3].sum()) + room
    check(desc, n, n, tables, page, capacity, width, pinned)
    check(desc, n - 1, n + 2, tables, page, capacity, max(1, width // 2), pinned)


def test_single_tokens_of_every_depth_as_decode_metadata_gives_them():
    from vllm_rlt_amd import ops

    desc, tables = batch(40, 40, 4, 12, 16, 1, 5)
    desc[:, 3] = 1
    desc[:, 2].clamp_(max=12 * 16 - 1)
    outs = buffers(40, 40, 12, spare=0)
    build(desc, 40, 40, tables, 16, outs, 12, False)
    long = lambda: torch.empty(40, dtype=torch.int64, device="cuda")  # noqa: E731
    slots, positions, blocks, offsets = long(), long(), long(), long()
    lengths, rows = torch.empty(40, dtype=torch.int32, device="cuda"), torch.empty(40, 12, dtype=torch.int32, device="cuda")
    ops.build_decode_metadata(desc[:, :3].contiguous().cuda(), 40, 40, tables.cuda(), 16, slots, positions, lengths, blocks, offsets, rows, 12)
    for a, b in zip((outs[1], outs[2], outs[4], outs[5], outs[6]), (lengths, positions, blocks, offsets, rows)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("pinned", [False, True])
def test_descriptors_outside_the_tables_and_too_many_tokens(pinned):
    desc, tables = batch(12, 6, 4, 10, 16, 20, 7)
    desc[:, 3].clamp_(min=1)
    desc[0, 0], desc[1, 0], desc[2, 1], desc[3, 1], desc[4, 2], desc[5, 3] = 6, -1, 4, -1, -7, -3
    desc[6, 2] = 10 * 16 - int(desc[6, 3]) + 1  # one token past the table
    desc[7, 2], desc[8, 2], desc[9, 0] = 1 << 62, (1 << 63) - 1, 1 << 40
    total = int(desc[:, 3].clamp(min=0).sum())
    for capacity in (total, total + 5, total - 4, int(desc[:4, 3].sum()), 1, 0):
        check(desc, 12, 13, tables, 16, capacity, 10, pinned)
    desc[10, 3] = 1 << 62
    check(desc, 12, 12, tables, 16, total, 10, pinned)


def test_empty_batches():
    tables = torch.ones(2, 1, 4, dtype=torch.int32)
    none = torch.empty(0, 4, dtype=torch.int64)
    for size, capacity in ((0, 0), (0, 9), (3, 9)):
        check(none, 0, size, tables, 16, capacity, 4)


@pytest.mark.parametrize("n,longest", [(1, 9000), (3, 9000), (300, 9000), (1100, 40)])
def test_long_chunks_and_many_sequences(n, longest):
    # One round of workgroups for any number of sequences, whichever of them holds the tokens.
    g = torch.Generator().manual_seed(n)
    tables = torch.randint(0, 5000, (4, 2, 600), generator=g, dtype=torch.int32)
    desc = torch.stack([torch.randint(0, 4, (n,), generator=g), torch.randint(0, 2, (n,), generator=g),
                        torch.randint(0, 300, (n,), generator=g), torch.randint(0, 30, (n,), generator=g)], 1)
    desc[n // 2, 3] = longest
    check(desc, n, n + 1, tables, 16, int(desc[:, 3].sum()) + 700, 600)


@pytest.mark.parametrize("pinned", [False, True])
def test_graph_replays_read_the_descriptors_again(pinned):
    from vllm_rlt_amd import ops

    desc, tables = batch(9, 12, 4, 30, 16, 50, 3)
    capacity, dev, tab = 9 * 50, desc.pin_memory() if pinned else desc.cuda(), tables.cuda()
    outs = buffers(9, capacity, 30, spare=0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.build_chunk_metadata(dev, 9, 9, tab, 16, *outs, 30)
    for seed in range(4):
        new, _ = batch(9, 12, 4, 30, 16, 50, 20 + seed)
        dev.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(outs, expected(new, 9, 9, tables, 16, capacity, 30)):
            assert torch.equal(got.cpu(), want)


def test_refusals():
    from vllm_rlt_amd import ops

    desc, tables = batch(3, 3, 2, 5, 16, 9, 1)
    outs = buffers(3, 40, 5, spare=0)
    base = dict(desc=desc.cuda(), count=3, size=3, tables=tables.cuda(), page=16, outs=outs, width=5)

    def call(**kw):
        a = base | kw
        ops.build_chunk_metadata(a["desc"], a["count"], a["size"], a["tables"], a["page"], *a["outs"], a["width"])

    def swap(i, t):
        return dict(outs=[*outs[:i], t, *outs[i + 1 :]])

    call()
    for kw, match in [
        (dict(desc=desc), "pinned"),
        (dict(desc=desc[:, :3].contiguous().cuda()), r"\[n, 4\]"),
        (dict(desc=desc.int().cuda()), "int64"),
        (dict(desc=desc.cuda().t().contiguous().t()), "contiguous"),
        (dict(tables=tables.cuda()[:, 0]), "tables must be"),
        (dict(count=4), "count"),
        (dict(count=-1), "count"),
        (dict(size=4), "smaller than size"),
        (dict(size=2), "count"),
        (dict(width=6), "out_width"),
        (dict(page=0), "page_size"),
        (swap(0, outs[0].long()), "cu_seqlens"),
        (swap(2, outs[2][:-1]), "share a length"),
        (swap(3, outs[3].int()), "sequences"),
        (swap(6, outs[6][:2]), "smaller than size"),
        (swap(6, outs[6].t()), "out_tables"),
    ]:
        with pytest.raises(ValueError, match=match):
            call(**kw)
