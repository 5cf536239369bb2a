"""8-bit KV cache: arguments, values and batches at the ends of their ranges (GPU)."""

import pytest
import torch
from fp8_cases import assert_within, attention
from test_fp8_attention_gpu import DTYPES, Case

pytestmark = pytest.mark.gpu
SHAPES = [(4, 4, 128), (8, 2, 128), (4, 4, 64), (2, 2, 80)]


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


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
@pytest.mark.parametrize("scale", [0.0, -0.0, 1e-40, -1e-44])
def test_softmax_scales_of_zero_and_below_the_smallest_normal(dtype, hq, hkv, d, scale):
    # Every visible key weighs alike, masked ones nothing.
    c = Case([150, 3000, 30], hq, hkv, d, dtype=dtype, seed=8, chunks=[100, 90, 40])
    c.scale = scale
    c.check(c.prefill())
    c.check(c.prefill(batch_invariant=True))
    c.q, c.chunks = c.q[:3], None
    c.check(c.decode())


def channels(c, seed, high=6.0):
    """Channels of very different sizes: q and K of the case times powers of two over 2^-high .. 2^high that undo each other on
    the whole, then a softmax scale that puts the largest sums of a score's magnitudes at 100."""
    d = c.q.shape[-1]
    g = torch.Generator().manual_seed(seed)
    e = torch.randint(-int(high), int(high) + 1, (d,), generator=g)
    c.q.mul_(torch.ldexp(torch.ones(d), e).to(c.q.dtype).cuda())
    codes = c.cache[0].float()
    owned = codes.isfinite()
    big = torch.randint(-3, 4, (d,), generator=g)
    codes = torch.where(owned, codes * torch.ldexp(torch.ones(d), big).cuda() / 16, codes)
    c.cache[0].view(torch.uint8).copy_(codes.to(torch.float8_e4m3fn).view(torch.uint8))
    k = (codes.nan_to_num(0.0) * torch.where(c.cache[2].float().isfinite(), c.cache[2].float(), 0.0)[..., None]).flatten(0, 1)
    k = k.abs().transpose(0, 1).repeat_interleave(c.q.shape[1] // k.shape[1], 0)  # [hq, tokens, d]
    c.scale = 100.0 / float((c.q.float().abs().transpose(0, 1) @ k.transpose(1, 2)).max())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d", [*SHAPES, (2, 2, 256)])
def test_decode_scores_of_channels_of_very_different_sizes_are_sums_in_32_bits(dtype, hq, hkv, d):
    c = Case([40, 300, 700, 1200, 100, 90, 80, 70], hq, hkv, d, dtype=dtype, seed=31)
    channels(c, 3)
    c.check(c.decode())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
def test_prefill_scores_of_channels_of_very_different_sizes_are_sums_in_32_bits(dtype, hq, hkv, d):
    c = Case([140, 300, 700], hq, hkv, d, dtype=dtype, seed=31, chunks=[100, 33, 200])
    channels(c, 3)
    c.check(c.prefill())
    c.check(c.prefill(batch_invariant=True))


@pytest.mark.parametrize("hq,hkv,d", SHAPES)
def test_prefill_keys_of_two_to_the_128_take_all_the_weight(hq, hkv, d):
    # Key 60 is what the append makes of the largest finite number in one dim where the queries are 1, and of 0 elsewhere.
    c = Case([150], hq, hkv, d, dtype=torch.bfloat16, seed=8, chunks=[100])
    at = (int(c.tables[0, 3]), 60 % 16)
    c.cache[0].view(torch.uint8)[at] = 0
    c.cache[0].view(torch.uint8)[at][:, 5] = 0x78
    c.cache[2].view(torch.uint8)[at] = 247
    c.q[..., 5] = 1.0
    c.q[..., 6] = 0.0
    c.scale = 0.5
    out = c.prefill()
    v = (c.cache[1].float() * c.cache[3].float()[..., None])[at].repeat_interleave(hq // hkv, 0)
    assert torch.equal(out[10:].float(), v.bfloat16().float().expand(90, -1, -1))
    assert out.isfinite().all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d", [(4, 4, 128), (16, 2, 128), (4, 4, 64), (8, 2, 64), (2, 2, 256), (2, 2, 80)])
def test_decode_keeps_its_probabilities_in_16_bits_or_more(dtype, hq, hkv, d):
    # The bound of attention() with 2^-16 in place of half a step of q's type for a probability.
    c = Case([1, 40, 700, 3000], hq, hkv, d, dtype=dtype, seed=21)
    out = c.decode()
    for r, n in enumerate(c.lengths):
        assert_within(out[r : r + 1], *attention(c.q[r : r + 1], c.cache, c.tables[r], [n], c.scale, 2.0**-16))


@pytest.mark.parametrize("hq,hkv,d", [(4, 4, 128), (16, 2, 128), (4, 4, 64)])
@pytest.mark.parametrize("ahead", [0.3, 2.7, 5.1, 5.5])
def test_a_key_that_dominates_late_weighs_what_it_should(hq, hkv, d, ahead):
    # Key 300 scores `ahead` (natural units) above all others, which agree: the running maximum may still be theirs.
    c = Case([400], hq, hkv, d, dtype=torch.bfloat16, seed=2)
    kc, vc, ks, vs = (t.view(torch.uint8) for t in c.cache)
    kc.zero_(), ks.fill_(127), vs.fill_(127), vc.copy_(torch.randint_like(vc, 0x30, 0x40))
    at = (int(c.tables[0, 300 // 16]), 300 % 16)
    kc[at] = torch.tensor(0x38, dtype=torch.uint8)  # ones
    c.q = torch.full_like(c.q, 1.0)
    c.scale = ahead / d
    want, bound = attention(c.q, c.cache, c.tables[0], [400], c.scale, 2.0**-16)
    assert_within(c.decode(), want, bound)


SMALL = [(torch.bfloat16, -112), (torch.float32, -100), (torch.float32, -60)]


def same_bits_of_small_values(c, call, dtype, shift):
    """V times 2^shift: outputs times 2^shift, bit for bit, as far as they are normal numbers."""
    vs = c.cache[3].view(torch.uint8)
    usual = vs.clone()
    big = call()
    vs.copy_(torch.where(usual == 255, 255, usual + shift))
    small = call()
    assert big.isfinite().all()
    want = big.double() * 2.0**shift
    normal = want.abs() >= torch.finfo(dtype).smallest_normal
    assert normal.float().mean() > 0.9
    assert torch.equal(small[normal].double(), want[normal])


@pytest.mark.parametrize("hq,hkv,d", SHAPES)
@pytest.mark.parametrize("dtype,shift", SMALL)
def test_decode_of_values_of_any_small_size_gives_the_same_bits(dtype, hq, hkv, d, shift):
    c = Case([150, 1500, 30], hq, hkv, d, dtype=dtype, seed=5)
    same_bits_of_small_values(c, c.decode, dtype, shift)


@pytest.mark.parametrize("hq,hkv,d", SHAPES)
@pytest.mark.parametrize("dtype,shift", SMALL)
def test_prefill_of_values_of_any_small_size_gives_the_same_bits(dtype, hq, hkv, d, shift):
    c = Case([150, 1500, 30], hq, hkv, d, dtype=dtype, seed=5, chunks=[100, 90, 30])
    same_bits_of_small_values(c, c.prefill, dtype, shift)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
@pytest.mark.parametrize("invariant", [False, True])
def test_a_value_of_two_to_the_128_is_weighed_and_stays_with_the_rows_that_see_it(dtype, hq, hkv, d, invariant):
    # What the append makes of the largest finite numbers: code 256, scale 2^120.  Key 120 of sequence 0 is seen by its
    # rows from 70 on, key 2000 of sequence 1 by all but its first 10 rows, both in a head's last dim.
    c = Case([150, 2080], hq, hkv, d, dtype=dtype, seed=8, chunks=[100, 90])
    clean = c.prefill(batch_invariant=invariant)
    for s, t, sign in ((0, 120, 0x78), (1, 2000, 0xF8)):
        at = (int(c.tables[s, t // 16]), t % 16, hkv - 1)
        c.cache[1].view(torch.uint8)[at] = 0
        c.cache[1].view(torch.uint8)[at][d - 1] = sign
        c.cache[3].view(torch.uint8)[at] = 247
    out = c.prefill(batch_invariant=invariant)
    heads = slice((hkv - 1) * (hq // hkv), hq)
    sees = torch.zeros(out.shape[:2], dtype=torch.bool, device="cuda")
    sees[70:100, heads] = True
    sees[110:, heads] = True
    others = [h for h in range(hq) if h // (hq // hkv) != hkv - 1]
    assert torch.equal(out[:, others], clean[:, others]) and out[~sees].isfinite().all()
    limits = [50 + i + 1 for i in range(100)], [1990 + i + 1 for i in range(90)]
    for s, rows in ((0, slice(0, 100)), (1, slice(100, 190))):
        want, bound = attention(c.q[rows], c.cache, c.tables[s], limits[s], c.scale, torch.finfo(dtype).eps / 2)
        fits = want.abs() + bound < torch.finfo(dtype).max
        assert fits[..., : d - 1].all()
        assert not ((out[rows].double() - want).abs() > bound)[fits].any() and not out[rows].isnan().any()
        past = want.abs() - bound > torch.finfo(dtype).max * (1 + torch.finfo(dtype).eps)
        assert out[rows][past].isinf().all()
        if dtype != torch.float16:
            assert fits.all()
    # Decode: the last row of sequence 0 at a length that sees the key, and at one that does not.
    from vllm_rlt_amd import ops

    lens = torch.tensor([121, 120], dtype=torch.int32, device="cuda")
    q = c.q[:1].repeat(2, 1, 1)
    got = ops.paged_decode_fp8(q, *c.cache, c.tables[[0, 0]].contiguous(), lens, scale=c.scale)
    want, bound = attention(q, c.cache, c.tables[0], [121, 120], c.scale, torch.finfo(dtype).eps / 2)
    fits = want.abs() + bound < torch.finfo(dtype).max
    assert not ((got.double() - want).abs() > bound)[fits].any() and not got.isnan().any() and fits[1].all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_sequence_without_rows_does_not_change_how_the_others_are_cut(dtype):
    # Balanced chunks beside one idle sequence of a long context: the bits of the batch without it.
    lengths, chunks = [600] * 24, [128] * 24
    c = Case([*lengths, 16000], 16, 4, 128, dtype=dtype, seed=4, chunks=[*chunks, 0])
    from vllm_rlt_amd import ops

    alone = ops.paged_prefill_fp8(c.q, *c.cache, c.tables[:24], c.lens[:24], c.cu[:25], 128, scale=c.scale)
    beside = c.prefill()
    assert torch.equal(alone, beside)
    c.check(beside)


@pytest.mark.parametrize("hq,hkv,d", [(3, 1, 64), (9, 9, 128)])
def test_a_merge_of_more_rows_than_its_grid_holds(hq, hkv, d):
    # Heads that do not fill the merge's 1024 elements, two cut sequences with an uncut one between.
    c = Case([5000, 30, 4000], hq, hkv, d, seed=14, chunks=[2000, 30, 500])
    c.check(c.prefill())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
@pytest.mark.parametrize("byte", [220, 235, 247])
def test_small_weights_of_the_largest_values_count(dtype, hq, hkv, d, byte):
    # Key 30 scores 40 binary orders below key 3, whose value is 1; its own, of 256 and a scale up to 2^120, rules the sum.
    c = Case([40], hq, hkv, d, dtype=dtype, seed=2, chunks=[5])
    kc, vc, ks, vs = (t.view(torch.uint8) for t in c.cache)
    kc.zero_(), ks.fill_(127), vs.fill_(127), vc.zero_()
    for t, key, value, scale in ((3, 0x38, 0x38, 127), (30, 0xB8, 0x78, byte)):  # keys of 1 and -1 in every dim
        at = (int(c.tables[0, t // 16]), t % 16)
        kc[at], vc[at], vs[at] = key, value, scale
    c.q = torch.full_like(c.q, 1.0)
    c.scale = 20 * 0.6931471805599453 / d  # scores of +-20 in binary orders, the others 0
    c.check(c.prefill())
    assert (c.prefill().float() > 2.0 ** (byte - 127 + 8 - 41)).all()
    c.q, c.chunks = c.q[:1], None
    c.check(c.decode())
    assert (c.decode().float() > 2.0 ** (byte - 127 + 8 - 41)).all()
