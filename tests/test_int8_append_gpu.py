"""Appends to the block-scaled 8-bit cache and reading it back, against their definitions (GPU).

The definition is a sequence of operations that are each rounded to float32, so codes
and scales are compared bit for bit; what they stand for is compared in 64 bits.
"""

import pytest
import torch
from int8_cases import append, random_cache, values

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def tokens(n, hkv, d, dtype, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    size = torch.exp2(torch.randn(n, 1, 1, generator=g) * spread)
    return [(torch.randn(n, hkv, d, generator=g) * size).to(dtype) for _ in range(2)]


def slots(runs, page, blocks, seed=0):
    """Slots of runs (first offset, tokens) in random blocks, each run's one after another."""
    g = torch.Generator().manual_seed(seed)
    perm, used, b, o = torch.randperm(blocks, generator=g), 0, [], []
    for first, n in runs:
        at = first + torch.arange(n)
        b.append(perm[used + at // page])
        o.append(at % page)
        used += -(-(first + n) // page)
    assert used <= blocks
    return torch.cat(b), torch.cat(o)


def same(got, want):
    for g, w in zip(got, want):
        g = g.cpu()
        assert torch.equal(g.view(torch.int8 if g.dtype == torch.int8 else torch.int32)[~w.isnan()] if g.dtype != torch.int8 else g,
                           w.view(torch.int32)[~w.isnan()] if w.dtype != torch.int8 else w)
        if g.dtype != torch.int8:
            assert torch.equal(g.isnan(), w.isnan())


def check(cache, layer, blocks, offsets, k, v, n_rows=None):
    """The call on a copy of the cache against the definition; returns the new cache."""
    from vllm_rlt_amd import ops

    got = [t.cuda() for t in cache]
    n = len(blocks) if n_rows is None else n_rows
    ops.kv_append_int8(*got, layer, blocks.cuda(), offsets.cuda(), k.cuda(), v.cuda(), n_rows=n_rows)
    want = [t.clone() for t in cache]
    append(want, layer, blocks[:n], offsets[:n], k[:n], v[:n])
    torch.cuda.synchronize()
    same(got, want)
    return want


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hkv,d,page", [(4, 128, 16), (8, 64, 16), (2, 256, 16), (3, 128, 32), (1, 80, 16), (5, 128, 7), (2, 64, 1), (2, 512, 16),
                                        (4, 128, 64), (2, 128, 100), (3, 64, 16)])
def test_runs_of_every_length_and_place(dtype, hkv, d, page):
    print(f"[append] {dtype} {hkv} x {d} page {page}", flush=True)
    runs = [(0, 1), (page - 1, 1), (0, page), (page // 2, page), (page // 3, 2 * page + 1), (0, 3), (page - 1, 2), (page // 2, 1)]
    blocks, offsets = slots(runs, page, 24, seed=page)
    cache = random_cache(25, page, hkv, d, seed=d, layers=2, spread=1.0)
    k, v = tokens(len(blocks), hkv, d, dtype, seed=hkv)
    check(cache, 1, blocks, offsets, k, v)
    check(cache, 0, blocks, offsets, k, v, n_rows=len(blocks) // 2)


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_blocks_and_single_tokens(dtype):
    # A packed batch of chunks, and a decode batch of a block each, larger than one workgroup or wave serves.
    runs = [((5 * i) % 16, 1 + (11 * i) % 70) for i in range(40)]
    blocks, offsets = slots(runs, 16, 240, seed=1)
    cache = random_cache(240, 16, 4, 128, seed=3, layers=2)
    check(cache, 1, blocks, offsets, *tokens(len(blocks), 4, 128, dtype, 5))
    runs = [((7 * i) % 16, 1) for i in range(230)]
    blocks, offsets = slots(runs, 16, 240, seed=2)
    check(cache, 0, blocks, offsets, *tokens(len(blocks), 4, 128, dtype, 6))


@pytest.mark.parametrize("d", [128, 80])
def test_a_block_filled_token_by_token(d):
    """Each step's codes are the definition's; a value is off by half a step of each scale it was rounded to."""
    from vllm_rlt_amd import ops

    k, v = tokens(16, 2, d, torch.float32, seed=4, spread=1.5)
    cache = [t.cuda() for t in random_cache(3, 16, 2, d, seed=1, layers=1)]
    want = [t.cpu().clone() for t in cache]
    slack = [torch.zeros(16, 2, dtype=torch.float64) for _ in "kv"]
    for i in range(16):
        at = torch.tensor([1]), torch.tensor([i])
        before = [t.cpu()[1, 0].clone() for t in cache[2:]]
        ops.kv_append_int8(*cache, 0, at[0].cuda(), at[1].cuda(), k[i : i + 1].cuda(), v[i : i + 1].cuda())
        append(want, 0, *at, k[i : i + 1], v[i : i + 1])
        same(cache, want)
        for x, old, codes, scales, off in zip((k, v), before, cache[:2], cache[2:], slack):
            now = scales.cpu()[1, 0].double()
            grew = now != old.double()
            off[:i] += torch.where(grew & (i > 0), now / 2, 0.0)
            off[i] = now / 2
            got = values(codes.cpu()[1, 0], scales.cpu()[1, 0])[: i + 1]
            assert ((got - x[: i + 1].double()).abs() <= (off[: i + 1] * (1 + 2.0**-16))[..., None]).all()


def test_order_inside_a_block_and_skipped_rows():
    # Offsets of a block in any order; rows of no block, of no offset and behind n_rows leave the cache as it is.
    cache = random_cache(8, 16, 4, 128, seed=2, layers=2)
    k, v = tokens(12, 4, 128, torch.bfloat16, 3, spread=2.0)
    blocks = torch.tensor([-1, 3, 3, 3, 3, 8, 5, 5, 1 << 40, 2, 2, 2])
    offsets = torch.tensor([0, 9, 2, 15, 5, 3, 16, -1, 0, 4, 1 << 33, 0])
    want = check(cache, 1, blocks, offsets, k, v)
    assert torch.equal(want[0][5], cache[0][5])
    check(cache, 1, blocks, offsets, k, v, n_rows=0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [128, 80])
def test_blocks_of_zeros_and_of_the_smallest_and_largest_values(dtype, d):
    tiny, huge = torch.finfo(dtype).smallest_normal, torch.finfo(dtype).max
    cache = random_cache(9, 16, 2, d, seed=5, layers=1)
    cache[2][4], cache[3][4] = 0.0, 0.0  # an empty block's scale
    k, v = tokens(40, 2, d, dtype, 2)
    k[0:3], v[0:3] = 0, 0
    k[3:6], v[3:6] = tiny, -tiny
    k[6:9] *= 2.0**-10
    k[9, :, 3], v[9, :, 5] = huge, -huge
    k[10], v[10] = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps, 0  # the smallest number
    blocks = torch.tensor([0] * 3 + [1] * 3 + [2] * 3 + [3] + [4] + [5] * 16 + [6] * 13)
    offsets = torch.tensor([0, 1, 2, 0, 1, 2, 3, 4, 5, 7, 3, *range(16), *range(13)])
    check(cache, 0, blocks, offsets, k, v)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [128, 80])
def test_values_that_are_not_finite_make_their_block_nan_until_it_begins_again(dtype, d):
    cache = random_cache(6, 16, 2, d, seed=5, layers=1)
    k, v = tokens(5, 2, d, dtype, 2)
    k[1, 0, 7], k[3, 1, d - 1], v[4, 1, 0] = torch.nan, torch.inf, -torch.inf
    blocks, offsets = torch.tensor([0, 0, 1, 2, 3]), torch.tensor([4, 5, 6, 0, 15])
    after = check(cache, 0, blocks, offsets, k, v)
    assert after[2][:, 0].isnan().tolist() == [[True, False], [False, False], [False, True], [False, False], [False, False], [False, False]]
    assert after[3][:, 0].isnan().tolist() == [[False, False]] * 3 + [[False, True]] + [[False, False]] * 2
    k, v = tokens(3, 2, d, dtype, 8)
    after = check(after, 0, torch.tensor([0, 2, 3]), torch.tensor([6, 0, 0]), k, v)
    assert after[2][0, 0, 0].isnan() and not after[2][2].isnan().any() and not after[3][3].isnan().any()


def strided(t, how):
    if how == "heads first":
        return torch.empty(t.shape[1], t.shape[0], t.shape[2], dtype=t.dtype, device="cuda").transpose(0, 1).copy_(t)
    if how == "dims apart":
        return torch.empty(t.shape[0], t.shape[2], t.shape[1], dtype=t.dtype, device="cuda").transpose(1, 2).copy_(t)
    if how == "of a larger row":
        return torch.empty(t.shape[0], 3, *t.shape[1:], dtype=t.dtype, device="cuda")[:, 1].copy_(t)
    return torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t)  # off 16 bytes


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("how", ["heads first", "dims apart", "off 16 bytes", "of a larger row"])
def test_strides(dtype, how):
    from vllm_rlt_amd import ops

    cache = random_cache(8, 16, 4, 128, seed=2, layers=2)
    k, v = tokens(40, 4, 128, dtype, 3)
    blocks, offsets = slots([(3, 20), (0, 1), (9, 19)], 16, 8)
    want = check(cache, 1, blocks, offsets, k, v)
    got = [t.cuda() for t in cache]
    ops.kv_append_int8(*got, 1, blocks.cuda(), offsets.cuda(), strided(k.cuda(), how), strided(v.cuda(), how))
    same(got, want)
    # The cache: head-major pages, dims apart, codes off any alignment, scales of another order.
    for lay in (lambda t: t.transpose(2, 3).contiguous().transpose(2, 3), lambda t: t.transpose(3, 4).contiguous().transpose(3, 4),
                lambda t: torch.zeros(t.numel() + 3, dtype=t.dtype, device="cuda")[3:].view(t.shape).copy_(t)):
        got = [*(lay(t.cuda()) for t in cache[:2]), *(t.cuda().transpose(0, 2).contiguous().transpose(0, 2) for t in cache[2:])]
        ops.kv_append_int8(*got, 1, blocks.cuda(), offsets.cuda(), k.cuda(), v.cuda())
        same(got, want)
        a = ops.kv_gather_int8(*got, 1, blocks.cuda(), offsets.cuda(), dtype)
        b = ops.kv_gather_int8(*(t.cuda() for t in want), 1, blocks.cuda(), offsets.cuda(), dtype)
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hkv,d,page", [(4, 128, 16), (8, 64, 16), (2, 256, 32), (3, 128, 16), (1, 80, 7), (16, 128, 16), (5, 512, 16)])
def test_reading_back(dtype, hkv, d, page):
    from vllm_rlt_amd import ops

    cache = random_cache(30, page, hkv, d, seed=d, layers=3, spread=6.0)
    cache[2][7, 2, 0], cache[3][9, 2, hkv - 1] = torch.nan, 0.0
    g = torch.Generator().manual_seed(1)
    n = 700
    blocks, offsets = torch.randint(0, 30, (n,), generator=g), torch.randint(0, page, (n,), generator=g)  # some of them twice
    blocks[[3, 50, 333]], offsets[[9, 51]] = torch.tensor([-1, 30, 1 << 40]), torch.tensor([page, -1])
    out = torch.zeros(2, n, hkv, d)
    inside = (blocks >= 0) & (blocks < 30) & (offsets >= 0) & (offsets < page)
    for i, (c, s) in enumerate(((cache[0], cache[2]), (cache[1], cache[3]))):
        out[i, inside] = c[blocks[inside], 2, offsets[inside]].float() * s[blocks[inside], 2][..., None]
    got = ops.kv_gather_int8(*(t.cuda() for t in cache), 2, blocks.cuda(), offsets.cuda(), dtype)
    for x, y in zip(got, out):  # the product is rounded to 32 bits and then once more
        assert x.shape == (n, hkv, d) and x.dtype == dtype and torch.equal(x.cpu().nan_to_num(9.0), y.to(dtype).nan_to_num(9.0))
    few = ops.kv_gather_int8(*(t.cuda() for t in cache), 2, blocks.cuda(), offsets.cuda(), n_rows=5)
    assert few[0].shape == (5, hkv, d) and torch.equal(few[1].cpu(), out[1, :5])
    assert ops.kv_gather_int8(*(t.cuda() for t in cache), 2, blocks.cuda(), offsets.cuda(), n_rows=0)[0].shape == (0, hkv, d)


def test_offsets_past_32_bits():
    from vllm_rlt_amd import ops

    layers, hkv, d, n = 256, 2, 128, 9
    cache = random_cache(n, 16, hkv, d, seed=3)
    blocks = (1 << 32) // (layers * 16 * hkv * d) + n + 1
    big = [torch.empty((blocks, layers, *t.shape[1:]), dtype=t.dtype, device="cuda") for t in cache]
    for x, t in zip(big, cache):
        x[blocks - n :, layers - 1].copy_(t)
    wb, wo = slots([(3, 20), (0, 1), (9, 19)], 16, n)
    k, v = tokens(40, hkv, d, torch.bfloat16, 3)
    want = check([t[:, None].clone() for t in cache], 0, wb, wo, k, v)
    at = (wb + blocks - n).cuda(), wo.cuda()
    ops.kv_append_int8(*big, layers - 1, *at, k.cuda(), v.cuda())
    same([t[blocks - n :, layers - 1] for t in big], [t[:, 0] for t in want])
    got = ops.kv_gather_int8(*big, layers - 1, *at, torch.float16)
    small = ops.kv_gather_int8(*(t.cuda() for t in want), 0, wb.cuda(), wo.cuda(), torch.float16)
    assert all(torch.equal(x, y) for x, y in zip(got, small))


def test_streams_and_graphs():
    from vllm_rlt_amd import ops

    cache = random_cache(8, 16, 4, 128, seed=2, layers=1)
    blocks, offsets = slots([(3, 20), (1, 1), (9, 19)], 16, 8)
    at = blocks.cuda(), offsets.cuda()
    k, v = (t.cuda() for t in tokens(40, 4, 128, torch.bfloat16, 3))
    got = [t.cuda() for t in cache]
    ops.kv_append_int8(*[t.clone() for t in got], 0, *at, k, v)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.kv_append_int8(*got, 0, *at, k, v)
        read = ops.kv_gather_int8(*got, 0, *at, torch.bfloat16)
    want = [t.clone() for t in cache]
    for i in range(4):
        nk, nv = tokens(40, 4, 128, torch.bfloat16, 30 + i, spread=2.0)
        k.copy_(nk), v.copy_(nv)
        graph.replay()
        append(want, 0, blocks, offsets, nk, nv)
        torch.cuda.synchronize()
        same(got, want)
        eager = ops.kv_gather_int8(*got, 0, *at, torch.bfloat16)
        assert all(torch.equal(x, y) for x, y in zip(read, eager))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [t.cuda() for t in cache]
        ops.kv_append_int8(*other, 0, *at, k, v)
        read = ops.kv_gather_int8(*other, 0, *at)
    torch.cuda.current_stream().wait_stream(side)
    again = [t.cuda() for t in cache]
    ops.kv_append_int8(*again, 0, *at, k, v)
    assert all(torch.equal(x, y) for x, y in zip(other, again))
    assert all(torch.equal(x, y) for x, y in zip(read, ops.kv_gather_int8(*again, 0, *at)))


@pytest.mark.parametrize("python", [False, True])
def test_refusals(python, monkeypatch):
    from vllm_rlt_amd import ops

    if python:
        monkeypatch.setattr(ops, "_host_calls", lambda t: (None, 0))
    kc, vc, ks, vs = (t.cuda() for t in random_cache(4, 16, 2, 64, layers=2))
    k = torch.zeros(3, 2, 64, device="cuda")
    one = torch.zeros(3, dtype=torch.int64, device="cuda")
    base = dict(kc=kc, vc=vc, ks=ks, vs=vs, layer=0, b=one, o=torch.arange(3, device="cuda"), k=k, v=k, n=None)

    def call(**kw):
        a = base | kw
        ops.kv_append_int8(a["kc"], a["vc"], a["ks"], a["vs"], a["layer"], a["b"], a["o"], a["k"], a["v"], a["n"])

    def read(dtype=torch.float32, **kw):
        a = base | kw
        return ops.kv_gather_int8(a["kc"], a["vc"], a["ks"], a["vs"], a["layer"], a["b"], a["o"], dtype, a["n"])

    call(), read()
    for kw, match in [
        (dict(kc=kc.view(torch.uint8)), "int8 codes"), (dict(ks=ks.half()), "float32"), (dict(vs=vs[:, :1]), "scales must be"),
        (dict(vc=vc[:2]), "share shape"), (dict(kc=kc[0], vc=vc[0]), "caches must be"), (dict(layer=2), "layer"), (dict(layer=-1), "layer"),
        (dict(b=one.int()), "blocks"), (dict(o=one[::2]), "offsets"), (dict(n=4), "n_rows"), (dict(n=-1), "n_rows"),
        (dict(kc=kc.cpu()), "ROCm device"), (dict(b=one.cpu()), "ROCm device"),
    ]:
        for f in (call, read):
            with pytest.raises(ValueError, match=match):
                f(**kw)
    for kw, match in [(dict(k=k[:, :1]), "k must have shape"), (dict(v=k[..., :32]), "v must have shape"), (dict(v=k.half()), "share a dtype"),
                      (dict(k=k.double(), v=k.double()), "float32, float16, or bfloat16"), (dict(k=k[:2]), "n_rows")]:
        with pytest.raises(ValueError, match=match):
            call(**kw)
    with pytest.raises(ValueError, match="float32, float16, or bfloat16"):
        read(dtype=torch.float64)


def test_both_paths_give_the_same_bits(monkeypatch):
    from vllm_rlt_amd import ops

    cache = random_cache(8, 16, 4, 128, seed=2, layers=2)
    blocks, offsets = (t.cuda() for t in slots([(3, 20), (0, 1), (9, 19)], 16, 8))
    k, v = (t.cuda() for t in tokens(40, 4, 128, torch.float16, 3))
    results = []
    for python in (False, True):
        with monkeypatch.context() as m:
            if python:
                m.setattr(ops, "_host_calls", lambda t: (None, 0))
            got = [t.cuda() for t in cache]
            ops.kv_append_int8(*got, 1, blocks, offsets, k, v, n_rows=33)
            results.append([*got, *ops.kv_gather_int8(*got, 1, blocks, offsets, torch.bfloat16, n_rows=17)])
    assert all(torch.equal(a, b) for a, b in zip(*results))
