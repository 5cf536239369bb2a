"""Quantising append and rotation by several axes, bit for bit against their definitions (GPU).

Scales are powers of two, so quantising rounds once: codes and scale bytes have to
equal the definition's.  The rotation's products and sums are float32 operations
that the CPU does alike, so its results do too.
"""

import pytest
import torch
from fp8_cases import quantise, random_cache

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def same_bits(a, b):
    """Equal bits, any NaN code for any other."""
    a, b = a.cpu(), b.cpu()
    if a.dtype == torch.float8_e4m3fn:
        x, y = a.view(torch.uint8), b.view(torch.uint8)
        nan = (x & 0x7F == 0x7F) & (y & 0x7F == 0x7F)
        return bool(((x == y) | nan).all())
    if a.dtype == torch.float8_e8m0fnu:
        return torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    return torch.equal(torch.nan_to_num(a, nan=7.5), torch.nan_to_num(b, nan=7.5)) and torch.equal(a.isnan(), b.isnan())


def rows_of(n, heads, d, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, heads, d, generator=g) * torch.exp(torch.randn(n, heads, 1, generator=g) * 3)
    return x.to(dtype)


def put(cache, layer, blocks, offsets, k, v, n):
    """The append of the first n rows on the CPU; slots outside the pool are skipped."""
    kc, vc, ks, vs = cache
    for x, codes, scales in ((k, kc, ks), (v, vc, vs)):
        c, s = quantise(x)
        for i in range(n):
            b, o = int(blocks[i]), int(offsets[i])
            if 0 <= b < kc.shape[0] and 0 <= o < kc.shape[2]:
                codes[b, layer, o] = c[i]
                scales[b, layer, o] = s[i]


def slots(n, blocks, page, seed):
    g = torch.Generator().manual_seed(seed)
    at = torch.randperm(blocks * page, generator=g)[:n]
    return at // page, at % page


def to_gpu(cache, head_major=False):
    """Copies on the device; head_major: with every head's tokens of a page together, behind the same shape."""
    if not head_major:
        return [t.cuda() for t in cache]
    return [t.transpose(2, 3).contiguous().cuda().transpose(2, 3) for t in cache]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,hkv,d,page", [(1, 1, 64, 16), (37, 16, 128, 16), (64, 8, 128, 16), (5, 3, 80, 16), (9, 2, 7, 5), (3, 4, 256, 16), (2, 2, 512, 4), (300, 4, 32, 1)])
@pytest.mark.parametrize("head_major", [False, True])
def test_append_equals_the_definition(dtype, n, hkv, d, page, head_major):
    from vllm_rlt_amd import ops

    blocks = -(-n // page) + 2
    cache = random_cache(blocks, page, hkv, d, seed=n, layers=3)
    wb, wo = slots(n, blocks, page, n)
    k, v = rows_of(n, hkv, d, dtype, 1), rows_of(n, hkv, d, dtype, 2)
    dev = to_gpu(cache, head_major)
    ops.kv_append_fp8(*dev, 1, wb.cuda(), wo.cuda(), k.cuda(), v.cuda())
    put(cache, 1, wb, wo, k, v, n)
    for a, b in zip(dev, cache):
        assert same_bits(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_at_the_edges_of_the_types(dtype):
    from vllm_rlt_amd import ops

    info = torch.finfo(dtype)
    edge = [0.0, -0.0, 1.0, 448.0, 449.0, 447.9, 3.5, 3.515625, info.max, -info.max, info.tiny, info.smallest_normal * 448,
            info.smallest_normal / 4, torch.inf, -torch.inf, torch.nan, 1.75, 1.7578125, 2.0**-9, 17.0, 18.0, 19.0]
    g = torch.Generator().manual_seed(3)
    n, d = 400, 64
    pick = torch.randint(0, len(edge), (n, 2, d), generator=g)
    x = torch.tensor(edge)[pick]
    few = torch.randint(0, d, (n, 2, 1), generator=g)  # most of a row zero, so that every value is a largest one somewhere
    x[: n // 2] = torch.where(torch.arange(d) == few, x, 0.0)[: n // 2]
    x = x.to(dtype)
    x[0] = 0.0
    cache = random_cache(n // 16 + 1, 16, 2, d, layers=1)
    wb, wo = slots(n, n // 16 + 1, 16, 9)
    dev = to_gpu(cache)
    ops.kv_append_fp8(*dev, 0, wb.cuda(), wo.cuda(), x.cuda(), x.flip(0).cuda())
    put(cache, 0, wb, wo, x, x.flip(0), n)
    for a, b in zip(dev, cache):
        assert same_bits(a, b)


@pytest.mark.parametrize("which", ["rows apart", "dims apart", "off 16 bytes"])
def test_append_reads_any_strides_and_skips_bad_slots(which):
    from vllm_rlt_amd import ops

    n, hkv, d = 33, 4, 128
    k, v = rows_of(n, hkv, d, torch.bfloat16, 4), rows_of(n, hkv, d, torch.bfloat16, 5)
    if which == "rows apart":
        kd = torch.empty(n, 3, hkv, d, dtype=k.dtype, device="cuda")[:, 1].copy_(k)
        vd = torch.empty(2 * n, hkv + 1, d, dtype=k.dtype, device="cuda")[::2, 1:].copy_(v)
    elif which == "dims apart":
        kd = torch.empty(d, hkv, n, dtype=k.dtype, device="cuda").permute(2, 1, 0).copy_(k)
        vd = torch.empty(n, d, hkv, dtype=k.dtype, device="cuda").permute(0, 2, 1).copy_(v)
    else:
        kd = torch.empty(n * hkv * d + 1, dtype=k.dtype, device="cuda")[1:].view(n, hkv, d).copy_(k)
        vd = torch.empty(n, hkv, d + 3, dtype=k.dtype, device="cuda")[..., 3:].copy_(v)
    cache = random_cache(6, 16, hkv, d, seed=8, layers=2)
    wb, wo = slots(n, 6, 16, 5)
    wb[3], wb[4], wo[5], wo[6] = -1, 6, 16, -2
    dev = to_gpu(cache)
    ops.kv_append_fp8(*dev, 1, wb.cuda(), wo.cuda(), kd, vd, n_rows=30)
    put(cache, 1, wb, wo, k, v, 30)
    for a, b in zip(dev, cache):
        assert same_bits(a, b)


def test_a_block_past_32_bits():
    from vllm_rlt_amd import ops

    hkv, d, page = 16, 128, 16
    blocks = (1 << 32) // (page * hkv * d) + 2  # the last block begins past element 2^32
    codes = [torch.zeros(blocks, 1, page, hkv, d, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2)]
    scales = [torch.zeros(blocks, 1, page, hkv, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu) for _ in range(2)]
    k, v = rows_of(1, hkv, d, torch.bfloat16, 6), rows_of(1, hkv, d, torch.bfloat16, 7)
    at = [torch.tensor([x], device="cuda") for x in (blocks - 1, 3)]
    ops.kv_append_fp8(*codes, *scales, 0, *at, k.cuda(), v.cuda())
    for x, c, s in zip((k, v), codes, scales):
        want, byte = quantise(x)
        assert same_bits(c[blocks - 1, 0, 3], want[0]) and same_bits(s[blocks - 1, 0, 3], byte[0])
        assert int(c.view(torch.uint8)[: blocks - 1].count_nonzero()) == 0
    # ... and decode reads it there.
    q = torch.randn(1, hkv, d, device="cuda").bfloat16()
    tables = torch.tensor([[blocks - 1]], dtype=torch.int32, device="cuda")
    codes[0][blocks - 1, 0, :3], codes[1][blocks - 1, 0, :3] = codes[0][blocks - 1, 0, 3], codes[1][blocks - 1, 0, 3]
    for s in scales:
        s.view(torch.uint8)[blocks - 1, 0, :3] = s.view(torch.uint8)[blocks - 1, 0, 3]
    out = ops.paged_decode_fp8(q, *(c[:, 0] for c in codes), *(s[:, 0] for s in scales), tables,
                               torch.tensor([4], dtype=torch.int32, device="cuda"))
    want, byte = quantise(v)  # four equal keys: the value itself
    want = (want.double() * byte.double()[..., None])[0]
    assert ((out.cpu()[0].double() - want).abs() <= want.abs() * (2.0**-8 + 2.0**-20)).all()


# ------------------------------------------------------------------ rotation
def rotary_table(half, positions, device="cpu"):
    freq = 10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)
    angles = torch.arange(positions, dtype=torch.float64)[:, None] * freq
    return torch.stack([angles.cos(), angles.sin()], -1).float().to(device)


def rotate(x, positions, table, axes):
    """The definition in float32 on the CPU."""
    half = table.shape[1]
    turn = table[positions[:, list(axes)], torch.arange(half)][:, None]
    c, s = turn[..., 0], turn[..., 1]
    x = x.float()
    lo, hi = x[..., :half], x[..., half : 2 * half]
    return torch.cat([lo * c - hi * s, hi * c + lo * s, x[..., 2 * half :]], -1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize(
    "n,hq,hkv,d,half,axes,interleaved",
    [(1, 16, 16, 128, 64, 3, False), (45, 16, 16, 128, 64, 3, True), (19, 32, 8, 128, 64, 1, False), (7, 8, 2, 64, 32, 2, False),
     (5, 4, 4, 128, 32, 4, True), (6, 3, 1, 80, 40, 3, False), (4, 2, 2, 10, 3, 2, False), (3, 2, 1, 256, 128, 4, False),
     (2, 1, 1, 512, 256, 3, True), (130, 16, 4, 128, 48, 3, False)],
)
def test_rotation_equals_the_definition(dtype, quantised, n, hq, hkv, d, half, axes, interleaved):
    from vllm_rlt_amd import ops

    g = torch.Generator().manual_seed(n + d)
    axis_map = tuple(j % axes if interleaved else min(j * axes // half, axes - 1) for j in range(half))
    positions = torch.randint(0, 4000, (n, axes), generator=g)
    positions[0] = 3999
    table = rotary_table(half, 4000)
    q, k, v = (rows_of(n, h, d, dtype, s) for s, h in ((1, hq), (2, hkv), (3, hkv)))
    page, blocks = 16, -(-n // 16) + 1
    wb, wo = slots(n, blocks, page, n)
    write = n - n // 4
    turned_q, turned_k = rotate(q, positions, table, axis_map).to(dtype), rotate(k, positions, table, axis_map)
    if quantised:
        cache = random_cache(blocks, page, hkv, d, seed=n, layers=2)
        dev = to_gpu(cache)
        caches, scales = dev[:2], dev[2:]
        put(cache, 1, wb, wo, turned_k, v, write)
    else:
        cache = [torch.randn(blocks, 2, page, hkv, d, generator=g).to(dtype) for _ in range(2)]
        dev = to_gpu(cache)
        caches, scales = dev, [None, None]
        for x, c in ((turned_k.to(dtype), cache[0]), (v, cache[1])):
            c[wb[:write], 1, wo[:write]] = x[:write]
    out = ops.rope_axes_kv_append(*caches, 1, wb.cuda(), wo.cuda(), q.cuda(), k.cuda(), v.cuda(), positions.cuda(), table.cuda(),
                                  axis_map, *scales, n_rows=write)
    assert same_bits(out, turned_q)
    for a, b in zip(dev, cache):
        assert same_bits(a, b)
    # The table's rounding aside, a rotation in 64 bits: each product and the sum rounded to float32, the result to q's type.
    lo, hi = q.double()[..., :half], q.double()[..., half : 2 * half]
    turn = table[positions[:, list(axis_map)], torch.arange(half)][:, None].double()
    first = lo * turn[..., 0] - hi * turn[..., 1]
    size = (lo * turn[..., 0]).abs() + (hi * turn[..., 1]).abs()
    unit = torch.finfo(dtype).eps / 2
    assert ((out.cpu()[..., :half].double() - first).abs() <= unit * first.abs() + 2.0**-22 * size + torch.finfo(dtype).smallest_normal * 2 * unit).all()


def test_rotation_in_place_with_strides_and_positions_outside_the_table():
    from vllm_rlt_amd import ops

    n, hq, hkv, d, half = 21, 8, 4, 128, 64
    axis_map = (0,) * 24 + (1,) * 20 + (2,) * 20
    table = rotary_table(half, 100)
    g = torch.Generator().manual_seed(2)
    positions = torch.randint(0, 100, (n, 3), generator=g)
    positions[4, 1], positions[9, 2], positions[10, 0] = 100, -1, 1 << 40
    outside = [4, 9, 10]
    q, k, v = (rows_of(n, h, d, torch.bfloat16, s) for s, h in ((1, hq), (2, hkv), (3, hkv)))
    clamped = positions.clone()
    clamped[outside] = 0
    want = rotate(q, clamped, table, axis_map).to(q.dtype)
    want[outside] = 0
    wb, wo = slots(n, 3, 16, 1)
    cache = random_cache(3, 16, hkv, d, seed=4, layers=1)
    dev = to_gpu(cache, head_major=True)
    fused = torch.randn(n, hq + 2 * hkv, d, dtype=torch.bfloat16, device="cuda")  # q, k and v as one projection's views
    qd, kd, vd = fused[:, :hq], fused[:, hq : hq + hkv], fused[:, hq + hkv :]
    qd.copy_(q), kd.copy_(k), vd.copy_(v)
    got = ops.rope_axes_kv_append(*dev[:2], 0, wb.cuda(), wo.cuda(), qd, kd, vd, positions.t().contiguous().cuda().t(), table.cuda(),
                                  axis_map, *dev[2:], out=qd)
    assert got.data_ptr() == qd.data_ptr() and same_bits(got, want)
    assert same_bits(kd, k) and same_bits(vd, v)
    skipped = wb.clone()
    skipped[outside] = -1
    put(cache, 0, skipped, wo, rotate(k, clamped, table, axis_map), v, n)
    for a, b in zip(dev, cache):
        assert same_bits(a, b)


def test_refusals():
    from vllm_rlt_amd import ops

    cache = to_gpu(random_cache(2, 16, 2, 64, layers=2))
    kc, vc, ks, vs = cache
    wb, wo = torch.zeros(1, dtype=torch.int64, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda")
    x = torch.zeros(1, 2, 64, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="e4m3fn"):
        ops.kv_append_fp8(kc.view(torch.uint8), vc.view(torch.uint8), ks, vs, 0, wb, wo, x, x)
    with pytest.raises(ValueError, match="e8m0fnu"):
        ops.kv_append_fp8(kc, vc, ks.view(torch.uint8), vs, 0, wb, wo, x, x)
    with pytest.raises(ValueError, match="without head_dim"):
        ops.kv_append_fp8(kc, vc, ks[..., :1], vs[..., :1], 0, wb, wo, x, x)
    with pytest.raises(ValueError, match="share a dtype"):
        ops.kv_append_fp8(*cache, 0, wb, wo, x, x.half())
    with pytest.raises(ValueError, match="must have shape"):
        ops.kv_append_fp8(*cache, 0, wb, wo, x[..., :32], x)
    with pytest.raises(ValueError, match="float32, float16, or bfloat16"):
        ops.kv_append_fp8(*cache, 0, wb, wo, x.double(), x.double())
    with pytest.raises(ValueError, match="layer"):
        ops.kv_append_fp8(*cache, 2, wb, wo, x, x)
    with pytest.raises(ValueError, match="n_rows"):
        ops.kv_append_fp8(*cache, 0, wb, wo, x, x, n_rows=2)
    with pytest.raises(ValueError):
        ops.kv_append_fp8(*cache, 0, wb, wo, x, x, n_rows=-1)
    ops.kv_append_fp8(*cache, 0, wb[:0], wo[:0], x[:0], x[:0])  # nothing to do

    table, positions = rotary_table(32, 10, "cuda"), torch.zeros(1, 2, dtype=torch.int64, device="cuda")
    axes = (0,) * 16 + (1,) * 16

    def rope(**kw):
        a = dict(q=x, k=x, v=x, positions=positions, table=table, axes=axes, key_scales=ks, value_scales=vs, caches=(kc, vc)) | kw
        return ops.rope_axes_kv_append(*a["caches"], 0, wb, wo, a["q"], a["k"], a["v"], a["positions"], a["table"], a["axes"],
                                       a["key_scales"], a["value_scales"])

    rope()
    for kw, match in [
        (dict(value_scales=None), "go together"),
        (dict(key_scales=None, value_scales=None), "q's dtype"),
        (dict(axes=(0,) * 16 + (2,) * 16), "axis past the last"),
        (dict(axes=axes[:-1]), "one axis for each"),
        (dict(table=table.double()), "table must be"),
        (dict(table=rotary_table(33, 10, "cuda"), axes=(0,) * 33), "head_dim / 2"),
        (dict(table=table[:0]), "no positions"),
        (dict(positions=positions.int()), "positions must be"),
        (dict(positions=torch.zeros(1, 5, dtype=torch.int64, device="cuda")), "1 to 4 axes"),
        (dict(positions=torch.zeros(2, 2, dtype=torch.int64, device="cuda")), "positions must be"),
        (dict(q=x[:, :1]), "multiple of 2"),
        (dict(k=x.half()), "dtype"),
    ]:
        with pytest.raises(ValueError, match=match):
            rope(**kw)
