"""Decode and prefill over the block-scaled 8-bit KV cache against attention in 64 bits (GPU).

The bounds are elementwise and derived in int8_cases.attention.  Blocks that no sequence
owns have NaN scales, and a sequence's last block holds the largest codes behind its end.
"""

import math

import pytest
import torch
from fp8_cases import assert_within, tables_for
from int8_cases import attention, poison, random_cache

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
SHAPES = [(4, 4, 128), (8, 2, 128), (4, 4, 64), (2, 2, 80)]


def queries(n, hq, d, dtype, seed):
    return torch.randn(n, hq, d, generator=torch.Generator().manual_seed(seed)).to(dtype)


class Case:
    def __init__(self, lengths, hq, hkv, d, page=16, dtype=torch.bfloat16, seed=0, spread=2.0, chunks=None):
        self.page, self.lengths = page, list(lengths)
        tables, blocks = tables_for(self.lengths, page, seed)
        cache = random_cache(blocks, page, hkv, d, seed, spread=spread)
        poison(cache, tables, self.lengths, page)
        self.cache = [t.cuda() for t in cache]
        self.tables = tables.cuda()
        self.lens = torch.tensor(self.lengths, dtype=torch.int32, device="cuda")
        self.chunks = chunks
        self.q = queries(sum(chunks) if chunks else len(self.lengths), hq, d, dtype, seed).cuda()
        if chunks:
            self.cu = torch.tensor([0, *chunks], dtype=torch.int32).cumsum(0).to(torch.int32).cuda()
        self.scale = 2.0 / math.sqrt(d)  # keys of about 40 codes of 2^-6

    def decode(self, **kw):
        from vllm_rlt_amd import ops

        return ops.paged_decode_int8(kw.pop("q", self.q), *kw.pop("cache", self.cache), self.tables, self.lens, scale=self.scale, **kw)

    def prefill(self, **kw):
        from vllm_rlt_amd import ops

        return ops.paged_prefill_int8(kw.pop("q", self.q), *kw.pop("cache", self.cache), self.tables, self.lens, self.cu,
                                      max(self.chunks), scale=self.scale, **kw)

    def check(self, out):
        torch.cuda.synchronize()
        if self.chunks is None:
            for r, n in enumerate(self.lengths):
                assert_within(out[r : r + 1], *attention(self.q[r : r + 1], self.cache, self.tables[r], [max(n, 0)], self.scale))
            return
        at = 0
        for s, (n, c) in enumerate(zip(self.lengths, self.chunks)):
            limits = [max(n - c + i + 1, 0) for i in range(c)]
            if c:
                assert_within(out[at : at + c], *attention(self.q[at : at + c], self.cache, self.tables[s], limits, self.scale))
            at += c


EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 512, 513, 700, 1023, 1024, 1025]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d", [(16, 16, 128), (8, 4, 128), (32, 8, 128), (8, 1, 128), (16, 1, 128), (6, 2, 128), (4, 4, 64), (8, 2, 64),
                                      (4, 2, 256), (20, 1, 64)])
def test_decode_at_length_edges(dtype, hq, hkv, d):
    print(f"[decode] {dtype} {hq}/{hkv} x {d}", flush=True)
    c = Case(EDGES, hq, hkv, d, dtype=dtype, seed=hq + d)
    c.check(c.decode())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d,page", [(3, 3, 80, 16), (4, 2, 128, 5), (2, 1, 7, 16), (2, 2, 512, 16), (5, 1, 128, 1), (7, 1, 96, 32),
                                           (40, 2, 64, 64), (4, 2, 128, 48), (2, 2, 256, 128)])
def test_decode_of_other_shapes(dtype, hq, hkv, d, page):
    print(f"[decode] {dtype} {hq}/{hkv} x {d} page {page}", flush=True)
    c = Case([0, 1, 5, 33, 130, 601], hq, hkv, d, page=page, dtype=dtype, seed=d)
    c.check(c.decode())


@pytest.mark.parametrize("lengths", [[5000], [3000, 1, 17000], [33000, 40000, 2], [900] * 70, [64] * 300])
@pytest.mark.parametrize("hq,hkv", [(4, 4), (16, 2)])
def test_decode_of_long_rows_and_many_rows(lengths, hq, hkv):
    print(f"[decode] {len(lengths)} rows to {max(lengths)}, {hq}/{hkv}", flush=True)
    c = Case(lengths, hq, hkv, 128, seed=len(lengths))
    c.check(c.decode())


@pytest.mark.parametrize("hq,hkv,d", [(16, 16, 128), (16, 2, 128), (8, 4, 64), (4, 4, 64)])
def test_a_row_depends_on_itself_only(hq, hkv, d):
    # The same rows alone, in a batch with longer tables, and in a large batch: equal bits.
    from vllm_rlt_amd import ops

    lengths = [1, 40, 300, 513, 1500, 2500]
    c = Case(lengths, hq, hkv, d, seed=3)
    together = c.decode()
    for r, n in enumerate(lengths):
        width = max(1, -(-n // 16))
        alone = ops.paged_decode_int8(c.q[r : r + 1], *c.cache, c.tables[r : r + 1, :width].contiguous(), c.lens[r : r + 1], scale=c.scale)
        assert torch.equal(alone[0], together[r]), n
    many = ops.paged_decode_int8(c.q.repeat(60, 1, 1), *c.cache, c.tables.repeat(60, 1), c.lens.repeat(60), scale=c.scale)
    assert torch.equal(many, together.repeat(60, 1, 1))


@pytest.mark.parametrize("hq,hkv,d,page,lengths", [(4, 1, 64, 16, [300000]), (1, 1, 64, 16, [300000]), (8, 2, 128, 48, [47, 48, 600, 1025]),
                                                  (2, 2, 128, 128, [1, 129, 1500]), (3, 3, 256, 32, [33, 700]), (16, 1, 64, 64, [63, 513])])
def test_decode_of_the_longest_rows_and_other_pages(hq, hkv, d, page, lengths):
    print(f"[decode] {hq}/{hkv} x {d} page {page} {lengths}", flush=True)
    c = Case(lengths, hq, hkv, d, page=page, seed=13)
    c.check(c.decode())


@pytest.mark.parametrize("hq,hkv,d,lengths", [(1, 1, 64, [16384, 16400, 8200, 300]), (4, 1, 64, [32768, 32784, 16500, 16384, 600])])
def test_rows_cut_into_more_splits_than_the_longest(hq, hkv, d, lengths):
    # A row just past 64 splits has half as many, twice as long.
    print(f"[decode] {lengths}", flush=True)
    c = Case(lengths, hq, hkv, d, seed=8)
    c.check(c.decode())


def strided(t, how):
    if how == "heads first":
        return torch.empty(t.shape[1], t.shape[0], t.shape[2], dtype=t.dtype, device="cuda").transpose(0, 1).copy_(t)
    if how == "dims apart":
        return torch.empty(t.shape[0], t.shape[2], t.shape[1], dtype=t.dtype, device="cuda").transpose(1, 2).copy_(t)
    return torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t)  # off 16 bytes


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("how", ["heads first", "dims apart", "off 16 bytes"])
@pytest.mark.parametrize("hq,hkv", [(8, 8), (8, 2)])
def test_strides_of_q_and_out(dtype, how, hq, hkv):
    c = Case([70, 0, 600], hq, hkv, 128, dtype=dtype, seed=5)
    out = strided(torch.zeros_like(c.q), how)
    assert c.decode(q=strided(c.q, how), out=out).data_ptr() == out.data_ptr()
    c.check(out)
    p = Case([70, 300], hq, hkv, 128, dtype=dtype, seed=5, chunks=[30, 140])
    out = strided(torch.zeros_like(p.q), how)
    p.prefill(q=strided(p.q, how), out=out)
    p.check(out)
    p.prefill(q=out.copy_(p.q), out=out)  # in place
    p.check(out)


@pytest.mark.parametrize("how", ["layer slice", "head major", "dims apart", "off 16 bytes"])
@pytest.mark.parametrize("hq,hkv", [(4, 4), (8, 2)])
def test_layouts_of_the_cache(how, hq, hkv):
    def lay(t):
        if how == "layer slice":
            return torch.zeros(t.shape[0], 3, *t.shape[1:], dtype=t.dtype, device="cuda")[:, 1].copy_(t)
        if how == "head major":
            return t.transpose(1, t.ndim - 2).contiguous().transpose(1, t.ndim - 2)
        if how == "dims apart":
            return t.transpose(-1, -2).contiguous().transpose(-1, -2)
        return torch.zeros(t.numel() + 5, dtype=t.dtype, device="cuda")[5:].view(t.shape).copy_(t)

    c = Case([70, 1, 600], hq, hkv, 128, seed=6)
    c.check(c.decode(cache=[lay(t) for t in c.cache]))
    p = Case([70, 300], hq, hkv, 128, seed=6, chunks=[30, 140])
    p.check(p.prefill(cache=[lay(t) for t in p.cache]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d,page", [(4, 4, 128, 16), (8, 2, 128, 16), (4, 4, 64, 16), (3, 1, 64, 16), (2, 1, 80, 16), (2, 2, 128, 8),
                                           (4, 2, 256, 16), (4, 4, 128, 32), (2, 2, 64, 128), (4, 2, 128, 48)])
@pytest.mark.parametrize("prefixes,chunks", [([0], [1]), ([0, 70, 5], [3, 200, 64]), ([1000, 0, 63, 129], [1, 65, 1, 130]), ([40, 200], [0, 33])])
def test_prefill(dtype, hq, hkv, d, page, prefixes, chunks):
    print(f"[prefill] {dtype} {hq}/{hkv} x {d} page {page} {prefixes} {chunks}", flush=True)
    c = Case([p + n for p, n in zip(prefixes, chunks)], hq, hkv, d, page=page, dtype=dtype, seed=d + len(chunks), chunks=chunks)
    c.check(c.prefill())


@pytest.mark.parametrize("dtype", DTYPES)
def test_prefill_of_long_prefixes_and_many_sequences(dtype):
    c = Case([9000 + 40, 4000 + 300], 4, 4, 128, dtype=dtype, seed=1, chunks=[40, 300])
    c.check(c.prefill())
    chunks = [(7 * i) % 23 for i in range(90)]
    c = Case([n + (13 * i) % 50 for i, n in enumerate(chunks)], 4, 2, 128, dtype=dtype, seed=2, chunks=chunks)
    c.check(c.prefill())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [128, 80])
def test_rows_that_see_no_key_are_zero_and_rows_of_no_sequence_are_left(dtype, d):
    from vllm_rlt_amd import ops

    # A context shorter than its chunk: the first rows see nothing.
    c = Case([40, 0, 100], 4, 4, d, dtype=dtype, seed=9, chunks=[70, 20, 100])
    q = torch.cat([c.q, queries(37, 4, d, dtype, 4).cuda()])
    out = torch.full_like(q, 5.0)
    ops.paged_prefill_int8(q, *c.cache, c.tables, c.lens, c.cu, 100, out=out, scale=c.scale)
    c.check(out[:190])
    assert (out[:30] == 0).all() and (out[70:90] == 0).all()
    assert (out[190:] == 5.0).all()


def test_lengths_past_the_table_and_below_zero():
    c = Case([64, 64, 64], 4, 4, 128, seed=2)
    c.lens = torch.tensor([100000, -3, 64], dtype=torch.int32, device="cuda")
    c.lengths = [64, 0, 64]
    c.check(c.decode())
    p = Case([64, 64], 4, 4, 128, seed=2, chunks=[20, 20])
    p.lens = torch.tensor([100000, -3], dtype=torch.int32, device="cuda")
    p.lengths = [64, 0]
    p.check(p.prefill())


@pytest.mark.parametrize("hq,hkv,d", [(4, 4, 128), (8, 2, 128), (2, 2, 80)])
def test_table_entries_outside_the_pool_read_block_0(hq, hkv, d):
    c = Case([200, 64], hq, hkv, d, seed=2)
    for t, s in zip(c.cache, (20, -9, 0.02, 0.03)):
        t[:1].fill_(s)
    c.tables[0, 3], c.tables[0, 7] = 1 << 30, -5
    c.check(c.decode())
    c.chunks, c.cu = [70, 3], torch.tensor([0, 70, 73], dtype=torch.int32, device="cuda")
    c.q = queries(73, hq, d, torch.bfloat16, 3).cuda()
    c.check(c.prefill())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_block_that_is_not_finite_reaches_only_the_rows_that_see_it(dtype, hq, hkv, d, bad):
    from vllm_rlt_amd import ops

    for which in (2, 3):
        c = Case([150, 90], hq, hkv, d, dtype=dtype, seed=8, chunks=[100, 90])
        clean = c.prefill()
        h = hkv - 1  # block 7 of sequence 0, its keys 112 to 127, is seen by its rows from 62 on
        c.cache[which][int(c.tables[0, 7]), h] = bad
        out = c.prefill()
        heads = slice(h * (hq // hkv), hq)
        touched = torch.zeros(out.shape[:2], dtype=torch.bool, device="cuda")
        touched[62:100, heads] = True
        assert not out[touched].isfinite().any() if math.isnan(bad) else not out[touched].isfinite().all(-1).any(), which
        assert torch.equal(out[~touched], clean[~touched]), which
        # Decode: the row that sees the block has NaN, the others their bits.
        q, lens = c.q[:3], torch.tensor([112, 113, 90], dtype=torch.int32, device="cuda")
        out = ops.paged_decode_int8(q, *c.cache, c.tables[[0, 0, 1]].contiguous(), lens, scale=c.scale)
        assert out[[0, 2]].isfinite().all() and not out[1, heads].isfinite().all(-1).any(), which


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
def test_queries_that_are_not_finite_or_huge(dtype, hq, hkv, d):
    c = Case([150, 300], hq, hkv, d, dtype=dtype, seed=8, chunks=[100, 90])
    clean = c.prefill()
    q = c.q.clone()
    q[[3, 70, 120], 1, 9] = torch.tensor([torch.nan, torch.inf, -torch.inf], device="cuda").to(dtype)
    out = c.prefill(q=q)
    keep = torch.ones(out.shape[:2], dtype=torch.bool, device="cuda")
    keep[[3, 70, 120], 1] = False
    assert torch.equal(out[keep], clean[keep])
    assert out[~keep].isnan().all()
    # Scores of every size: one key takes all the weight, whatever its score.
    c.q = (c.q * 3000).to(dtype)
    c.check(c.prefill())
    c.q, c.chunks = c.q[:2], None
    c.check(c.decode())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
@pytest.mark.parametrize("scale", [0.0, -0.0, 1e-40, -1e-44, -0.17])
def test_softmax_scales_of_zero_and_below(dtype, hq, hkv, d, scale):
    c = Case([150, 3000, 30], hq, hkv, d, dtype=dtype, seed=8, chunks=[100, 90, 40])
    c.scale = scale
    c.check(c.prefill())
    c.check(c.prefill(batch_invariant=True))
    c.q, c.chunks = c.q[:3], None
    c.check(c.decode())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
def test_scales_far_apart(dtype, hq, hkv, d):
    # Blocks of one head from 2^-20 to 2^20 of the usual size: the largest values rule, nothing overflows or turns into NaN.
    c = Case([500, 700, 30], hq, hkv, d, dtype=dtype, seed=4, spread=20.0)
    c.scale = 2.0**-18 / math.sqrt(d)
    if dtype == torch.float16:  # outputs of up to 127 * 2^14 leave fp16
        c.cache[3].clamp_(max=2.0**-3)
    c.check(c.decode())
    c.chunks, c.cu = [200, 130, 7], torch.tensor([0, 200, 330, 337], dtype=torch.int32, device="cuda")
    c.q = queries(337, hq, d, dtype, 3).cuda()
    c.check(c.prefill())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
def test_blocks_of_zeros_keep_their_weight(dtype, hq, hkv, d):
    # V blocks of scale 0 and 2^-126, K blocks of scale 0: their keys count in the sum of the weights.
    c = Case([300, 90], hq, hkv, d, dtype=dtype, seed=4, chunks=[200, 90])
    t = c.tables.clamp(min=0).long()
    c.cache[3][t[0, 3]], c.cache[3][t[0, 9]], c.cache[3][t[1, 5]] = 0.0, 2.0**-126, 0.0
    c.cache[2][t[0, 2]], c.cache[2][t[1, 5]] = 0.0, 0.0
    c.cache[2][t[0, 3]] *= 4  # and carry most of it
    c.check(c.prefill())
    c.q, c.chunks = c.q[:2], None
    c.check(c.decode())


@pytest.mark.parametrize("hq,hkv,d", SHAPES)
@pytest.mark.parametrize("dtype,shift", [(torch.bfloat16, -112), (torch.float32, -100), (torch.float32, -60), (torch.bfloat16, 100), (torch.float32, 110)])
def test_values_of_any_size_give_the_same_bits(hq, hkv, d, dtype, shift):
    """V times 2^shift: outputs times 2^shift, bit for bit, as far as they are normal numbers."""
    c = Case([150, 1500, 30], hq, hkv, d, dtype=dtype, seed=5, chunks=[100, 90, 30])
    usual = c.cache[3].clone()
    for call in (c.prefill, lambda: c.decode(q=c.q[:3].contiguous())):
        c.cache[3].copy_(usual)
        whole = call()
        c.cache[3].copy_(usual * 2.0**shift)
        got = call()
        assert whole.isfinite().all()
        want = whole.double() * 2.0**shift
        normal = want.abs() >= torch.finfo(dtype).smallest_normal
        assert normal.float().mean() > 0.9 and torch.equal(got[normal].double(), want[normal])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
@pytest.mark.parametrize("power", [0, 60, 110])
def test_small_weights_of_the_largest_values_count(dtype, hq, hkv, d, power):
    # Key 30 scores 40 binary orders below key 3, whose value is 1; its own, of 127 and a scale up to 2^110, rules the sum.
    c = Case([40], hq, hkv, d, dtype=dtype, seed=2, chunks=[5])
    for t, x in zip(c.cache, (0, 0, 1.0, 1.0)):
        t.fill_(x)
    for t, key, value, scale in ((3, 1, 1, 1.0), (30, -1, 127, 2.0**power)):
        block = int(c.tables[0, t // 16])
        c.cache[0][block, t % 16], c.cache[1][block, t % 16], c.cache[3][block] = key, value, scale
    c.q = torch.full_like(c.q, 1.0)
    c.scale = 20 * 0.6931471805599453 / d  # scores of +-20 in binary orders, the others 0
    c.check(c.prefill())
    if power:
        assert (c.prefill().float() > 2.0 ** (power + 6 - 41)).all()
    c.q, c.chunks = c.q[:1], None
    c.check(c.decode())


def channels(c, seed, high=6):
    """Channels of very different sizes: q and K of the case times powers of two, then a softmax scale that puts the largest
    sums of a score's magnitudes at 100."""
    d = c.q.shape[-1]
    g = torch.Generator().manual_seed(seed)
    c.q.mul_(torch.ldexp(torch.ones(d), torch.randint(-high, high + 1, (d,), generator=g)).to(c.q.dtype).cuda())
    shrink = torch.ldexp(torch.ones(d), torch.randint(-5, 1, (d,), generator=g)).cuda()
    c.cache[0].copy_((c.cache[0].float() * shrink).round().to(torch.int8))
    k = (c.cache[0].float() * c.cache[2].nan_to_num(0.0)[:, None, :, None]).flatten(0, 1)
    k = k.abs().transpose(0, 1).repeat_interleave(c.q.shape[1] // k.shape[1], 0)  # [hq, tokens, d]
    c.scale = 100.0 / float((c.q.float().abs().transpose(0, 1) @ k.transpose(1, 2).contiguous()).max())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d", [*SHAPES, (2, 2, 256)])
def test_scores_of_channels_of_very_different_sizes_are_sums_in_32_bits(dtype, hq, hkv, d):
    c = Case([40, 300, 700, 1200, 100, 90, 80, 70], hq, hkv, d, dtype=dtype, seed=31)
    channels(c, 3)
    c.check(c.decode())
    p = Case([140, 300, 700], hq, hkv, d, dtype=dtype, seed=31, chunks=[100, 33, 200])
    channels(p, 3)
    p.check(p.prefill())
    p.check(p.prefill(batch_invariant=True))


@pytest.mark.parametrize("hq,hkv,d", [(4, 4, 128), (16, 2, 128), (4, 4, 64)])
@pytest.mark.parametrize("ahead", [0.3, 2.7, 5.1, 5.5, 12.0])
def test_a_key_that_dominates_late_weighs_what_it_should(hq, hkv, d, ahead):
    # Key 300 scores `ahead` (natural units) above all others, which agree: the running maximum may still be theirs.
    c = Case([400], hq, hkv, d, seed=2, chunks=[60])
    c.cache[0].zero_(), c.cache[2].fill_(1.0), c.cache[3].fill_(1.0)
    c.cache[0][int(c.tables[0, 300 // 16]), 300 % 16] = 1
    c.q = torch.full_like(c.q, 1.0)
    c.scale = ahead / d
    c.check(c.prefill())
    c.q, c.chunks = c.q[:1], None
    c.check(c.decode())


def test_streams_graphs_and_given_buffers():
    from vllm_rlt_amd import ops

    c = Case([700, 90, 1], 8, 8, 128, seed=1)
    p = Case([700, 90], 8, 8, 128, seed=1, chunks=[200, 60])
    want, want_p = c.decode(), p.prefill()
    need = ops.decode_int8_workspace_bytes(3, c.tables.shape[1], 8, 8, 128, 16)
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    need_p = ops.prefill_int8_workspace_bytes(260, 2, p.tables.shape[1], 8, 8, 128, 16)
    ws_p = torch.empty(max(need_p, 1), dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a, b = c.decode(workspace=ws), p.prefill(workspace=ws_p)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, want) and torch.equal(b, want_p)
    if need:
        with pytest.raises(ValueError, match="workspace"):
            c.decode(workspace=ws[: need - 1])
    out, out_p = torch.empty_like(c.q), torch.empty_like(p.q)
    # Two graphs, each with a workspace of its own, replayed with eager work and changed inputs between.
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    with torch.cuda.graph(graphs[0]):
        c.decode(workspace=ws, out=out)
    with torch.cuda.graph(graphs[1]):
        p.prefill(workspace=ws_p, out=out_p)
    for i in range(4):
        c.q.copy_(queries(3, 8, 128, torch.bfloat16, 50 + i))
        p.q.copy_(queries(260, 8, 128, torch.bfloat16, 60 + i))
        c.lens.copy_(torch.tensor([700 - 100 * i, 90, i], dtype=torch.int32))
        out.fill_(3), out_p.fill_(3)
        graphs[i % 2].replay(), graphs[1 - i % 2].replay()
        torch.cuda.synchronize()
        # Bits, not values: row 2 comes to see blocks of nobody, and is NaN either way.
        assert torch.equal(out.view(torch.int16), c.decode().view(torch.int16))
        assert torch.equal(out_p.view(torch.int16), p.prefill().view(torch.int16))


def test_a_captured_prefill_follows_the_lengths_of_each_replay():
    p = Case([6000, 500, 40], 8, 2, 128, seed=4, chunks=[70, 300, 40])
    out = torch.empty_like(p.q)
    graph = torch.cuda.CUDAGraph()
    p.prefill()
    with torch.cuda.graph(graph):
        p.prefill(out=out)
    for lengths, chunks in [([6000, 500, 40], [70, 300, 40]), ([70, 300, 40], [70, 300, 40]), ([6000, 500, 40], [400, 10, 0]),
                            ([900, 500, 40], [1, 1, 1]), ([6000, 0, 0], [410, 0, 0])]:
        p.lengths, p.chunks = lengths, chunks
        p.lens.copy_(torch.tensor(lengths, dtype=torch.int32))
        p.cu.copy_(torch.tensor([0, *chunks], dtype=torch.int32).cumsum(0))
        out.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        n = sum(chunks)
        p.check(out[:n])
        assert (out[n:] == 7).all()


def test_two_calls_at_once():
    c = Case([4000, 90, 700, 2500], 8, 8, 128, seed=1)
    p = Case([5000, 90], 8, 4, 128, seed=1, chunks=[200, 60])
    want, want_p = c.decode(), p.prefill()
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for i in range(12):
        with torch.cuda.stream(streams[i % 3]):
            got.append((c.decode(), p.prefill()))
    torch.cuda.synchronize()
    assert all(torch.equal(a, want) and torch.equal(b, want_p) for a, b in got)


def test_repeated_calls_give_the_same_bits():
    c = Case([3000, 64, 700], 16, 16, 128, seed=1)
    p = Case([900, 400], 16, 4, 128, seed=1, chunks=[300, 129])
    first, first_p = c.decode(), p.prefill()
    for _ in range(5):
        assert torch.equal(c.decode(), first) and torch.equal(p.prefill(), first_p)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("prefixes,chunks", [([3000, 5, 0], [70, 140, 260]), ([0], [2100]), ([8191, 511, 512, 513], [1, 1, 129, 128]), ([30, 2000], [400, 0])])
def test_prefill_of_cut_keys_and_the_batch_invariant_form(dtype, prefixes, chunks):
    from vllm_rlt_amd import ops

    lengths = [p + n for p, n in zip(prefixes, chunks)]
    c = Case(lengths, 8, 8, 128, dtype=dtype, seed=len(chunks), chunks=chunks)
    c.check(c.prefill())
    whole = c.prefill(batch_invariant=True)
    c.check(whole)
    at = 0
    for s, n in enumerate(chunks):  # a sequence alone gives the batch's bits
        if n:
            alone = ops.paged_prefill_int8(c.q[at : at + n], *c.cache, c.tables[s : s + 1], c.lens[s : s + 1],
                                           torch.tensor([0, n], dtype=torch.int32, device="cuda"), n, scale=c.scale, batch_invariant=True)
            assert torch.equal(alone, whole[at : at + n])
        at += n


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d", [(6, 2, 128), (5, 1, 64), (28, 4, 128), (40, 1, 128), (24, 8, 64), (200, 1, 64)])
def test_prefill_of_groups_of_any_size(dtype, hq, hkv, d):
    """Tiles hold the query heads of a row together: groups that do not divide them, and ones larger than a wave's rows or a tile."""
    for prefixes, chunks in [([0, 300, 77, 1500], [1, 9, 43, 130]), ([2000], [3]), ([5, -3] * 35, [2, 4] * 35)]:
        lengths = [max(p + c, 0) for p, c in zip(prefixes, chunks)]
        c = Case(lengths, hq, hkv, d, dtype=dtype, seed=hq, chunks=chunks)
        out = c.prefill()
        c.check(out)
        whole = c.prefill(batch_invariant=True)
        c.check(whole)
        if len(chunks) > 64:
            assert torch.equal(out, whole)


@pytest.mark.parametrize("hq,hkv,d", [(3, 1, 64), (9, 9, 128)])
def test_cut_sequences_of_many_rows(hq, hkv, d):
    # Heads that do not fill a merge's workgroup, two cut sequences with an uncut one between, rows that see no key.
    c = Case([5000, 30, 4000, 1500], hq, hkv, d, seed=14, chunks=[2000, 30, 500, 2000])
    out = c.prefill()
    c.check(out)
    assert (out[2530:3030] == 0).all()


def test_row_ranges_that_overlap_stay_inside_the_workspace():
    # cu_seqlens must rise; where they do not, no result is promised, but nothing else is written.
    from vllm_rlt_amd import ops

    c = Case([4096], 1, 1, 64, seed=6, chunks=[1280])
    tables, lens = c.tables.repeat(64, 1), c.lens.repeat(64)
    cu = torch.tensor([0, 1280], dtype=torch.int32, device="cuda").repeat(33)[:65].contiguous()
    need = ops.prefill_int8_workspace_bytes(1280, 64, tables.shape[1], 1, 1, 64, 16)
    memory = torch.full((need + (1 << 24),), 7, dtype=torch.uint8, device="cuda")
    out = torch.full((1280 + 64, 1, 64), 3.0, dtype=torch.bfloat16, device="cuda")
    ops.paged_prefill_int8(c.q, *c.cache, tables, lens, cu, 1280, out=out[:1280], scale=c.scale, workspace=memory[:need])
    torch.cuda.synchronize()
    assert (memory[need:] == 7).all() and (out[1280:] == 3).all()


@pytest.mark.parametrize("hq,hkv,d", [(2, 2, 64), (4, 2, 64), (2, 2, 128), (2, 2, 80)])
def test_offsets_past_32_bits(hq, hkv, d):
    from vllm_rlt_amd import ops

    c = Case([70, 600, 5], hq, hkv, d, seed=3, chunks=[30, 140, 5])
    layers, n = 256, c.cache[0].shape[0]
    blocks = (1 << 32) // (layers * 16 * hkv * d) + n + 1  # the cache's blocks begin past element 2^32
    big = []
    for t in c.cache:
        whole = torch.empty((blocks, layers, *t.shape[1:]), dtype=t.dtype, device="cuda")
        whole[blocks - n :, layers - 1].copy_(t)
        big.append(whole[:, layers - 1])
    tables = torch.where(c.tables >= 0, c.tables + blocks - n, -1)
    q = c.q[:3].contiguous()
    got = ops.paged_decode_int8(q, *big, tables, c.lens, scale=c.scale)
    assert torch.equal(got, ops.paged_decode_int8(q, *c.cache, c.tables, c.lens, scale=c.scale))
    got = ops.paged_prefill_int8(c.q, *big, tables, c.lens, c.cu, 140, scale=c.scale)
    assert torch.equal(got, c.prefill())


@pytest.mark.parametrize("python", [False, True])
def test_refusals(python, monkeypatch):
    from vllm_rlt_amd import ops

    if python:
        monkeypatch.setattr(ops, "_host_calls", lambda t: (None, 0))
    c = Case([20, 30], 4, 2, 64, seed=1, chunks=[3, 4])
    kc, vc, ks, vs = c.cache
    d = dict(q=c.q[:2], kc=kc, vc=vc, ks=ks, vs=vs, tables=c.tables, lens=c.lens, out=None, workspace=None)

    def decode(**kw):
        a = d | kw
        return ops.paged_decode_int8(a["q"], a["kc"], a["vc"], a["ks"], a["vs"], a["tables"], a["lens"], a["out"], a["workspace"])

    def prefill(cu=c.cu, longest=4, **kw):
        a = d | dict(q=c.q) | kw
        return ops.paged_prefill_int8(a["q"], a["kc"], a["vc"], a["ks"], a["vs"], a["tables"], a["lens"], cu, longest, a["out"])

    decode(), prefill()
    for call in (decode, prefill):
        for kw, match in [
            (dict(kc=kc.view(torch.uint8)), "int8 codes"),
            (dict(vs=vs.half()), "float32"),
            (dict(ks=ks[:, :1]), "scales must be"),
            (dict(vc=vc[:-1]), "share shape"),
            (dict(kc=kc[None], vc=vc[None]), "caches must be"),
            (dict(q=c.q[..., :32]), "q must have shape"),
            (dict(q=c.q[:, :3]), "positive multiple"),
            (dict(q=c.q.double()), "float32, float16, or bfloat16"),
            (dict(tables=c.tables.long()), "block_tables"),
            (dict(tables=c.tables.t()), "block_tables"),
            (dict(lens=c.lens.long()), "context_lengths"),
            (dict(lens=c.lens[:1]), "one entry"),
            (dict(out=c.q.float()), "out must match"),
            (dict(kc=kc.cpu()), "same ROCm device"),
            (dict(kc=kc[:, :, :0], vc=vc[:, :, :0], ks=ks[:, :0], vs=vs[:, :0]), "positive multiple"),
            (dict(kc=kc[:, :0], vc=vc[:, :0]), "page_size"),
        ]:
            with pytest.raises(ValueError, match=match):
                call(**kw)
    with pytest.raises(ValueError, match="one entry per row"):
        decode(q=c.q[:3])
    with pytest.raises(ValueError, match="one entry per sequence"):
        prefill(cu=c.cu[:2])
    with pytest.raises(ValueError, match="max_seqlen_q"):
        prefill(longest=-1)
    assert decode(q=c.q[:0], tables=c.tables[:0], lens=c.lens[:0]).shape == (0, 4, 64)
    assert prefill(q=c.q[:0]).shape == (0, 4, 64)


def test_both_paths_give_the_same_bits_and_the_host_calls_are_taken(monkeypatch):
    from vllm_rlt_amd import _native, ops

    c = Case([40, 700], 8, 4, 64, seed=1)
    p = Case([400, 700], 8, 4, 64, seed=1, chunks=[20, 30])
    ws = torch.empty(1 << 24, dtype=torch.uint8, device="cuda")
    out = torch.empty_like(p.q)
    calls = [c.decode, lambda: c.decode(workspace=ws), p.prefill, lambda: p.prefill(out=out, workspace=ws).clone(),
             lambda: p.prefill(batch_invariant=True)]
    first = [call() for call in calls]
    with monkeypatch.context() as m:
        m.setattr(ops, "_host_calls", lambda t: (None, 0))
        second = [call() for call in calls]
    assert all(torch.equal(a, b) for a, b in zip(first, second))

    class Library:
        def __getattr__(self, name):
            raise AssertionError(f"{name} went through Python")

    monkeypatch.setattr(_native, "_lib", Library())
    for call in calls:
        call()
    pool = [t[:, None].contiguous() for t in c.cache]
    at = torch.zeros(3, dtype=torch.int64, device="cuda"), torch.arange(3, device="cuda")
    k = torch.zeros(3, 4, 64, device="cuda")
    ops.kv_append_int8(*pool, 0, *at, k, k)
    ops.kv_gather_int8(*pool, 0, *at, torch.bfloat16)
    torch.cuda.synchronize()
