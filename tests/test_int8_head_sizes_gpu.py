"""The block-scaled 8-bit cache at head sizes between and beyond its kernels' (GPU).

Attention: multiples of 16 up to 256 run the kernels of the next larger size; the others a kernel for any shape, which goes through the tests of the kernels on the matrix cores.  Appends and reads: heads of whole
16-byte packets have a power of two of lanes, not all of them of use.
"""

import pytest
import test_int8_append_gpu as append_tests
import test_int8_attention_gpu as attention_tests
import torch
from int8_cases import append, random_cache
from test_int8_attention_gpu import DTYPES, Case

pytestmark = pytest.mark.gpu
SIZES = [(4, 4, 16), (4, 2, 32), (4, 2, 48), (6, 2, 80), (3, 3, 96), (20, 1, 112), (4, 4, 144), (8, 2, 192), (2, 2, 240)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d", SIZES)
def test_multiples_of_16(dtype, hq, hkv, d):
    c = Case([0, 1, 15, 16, 17, 33, 64, 65, 129, 513, 1500], hq, hkv, d, dtype=dtype, seed=d)
    c.check(c.decode())
    p = Case([3, 270, 69, 1020, 2500], hq, hkv, d, dtype=dtype, seed=d, chunks=[3, 200, 64, 20, 5])
    p.check(p.prefill())
    p.check(p.prefill(batch_invariant=True))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d", [(4, 4, 16), (6, 2, 80), (3, 3, 112), (2, 2, 176)])
def test_nothing_is_stored_past_a_head(dtype, hq, hkv, d):
    for c in (Case([700, 30], hq, hkv, d, dtype=dtype, seed=1), Case([2000, 30], hq, hkv, d, dtype=dtype, seed=1, chunks=[30, 9])):
        wide = torch.full((len(c.q), hq, d + 16), 7.0, dtype=dtype, device="cuda")
        c.check((c.prefill if c.chunks else c.decode)(out=wide[..., :d]))
        assert (wide[..., d:] == 7.0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv", [(2, 2), (6, 2)])
def test_heads_of_256(dtype, hq, hkv):
    c = Case([0, 64, 65, 1000, 2100, 5], hq, hkv, 256, dtype=dtype, seed=3, chunks=[0, 64, 1, 300, 129, 5])
    c.check(c.prefill())
    whole = c.prefill(batch_invariant=True)
    c.check(whole)
    assert torch.equal(c.prefill(batch_invariant=True), whole)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(
    "name,more",
    [
        ("test_a_block_that_is_not_finite_reaches_only_the_rows_that_see_it", (float("nan"),)),
        ("test_queries_that_are_not_finite_or_huge", ()),
        ("test_softmax_scales_of_zero_and_below", (-0.17,)),
        ("test_scales_far_apart", ()),
        ("test_blocks_of_zeros_keep_their_weight", ()),
    ],
)
def test_heads_of_256_where_it_can_go_wrong(name, more, dtype):
    getattr(attention_tests, name)(dtype, 2, 2, 256, *more)


@pytest.mark.parametrize("dtype,d", [(torch.float32, 256), (torch.bfloat16, 80), (torch.float16, 176)])
def test_captured_calls(dtype, d):
    p = Case([700, 64, 2100], 4, 2, d, dtype=dtype, seed=6, chunks=[70, 64, 33])
    c = Case([700, 64, 2100], 4, 2, d, dtype=dtype, seed=7)
    first = p.prefill(), c.decode()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = p.prefill(), c.decode()
    for shift in (0, 1, 0):
        for x in (p, c):
            x.q.add_(shift)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, (p.prefill(), c.decode())):
            assert torch.equal(a, b)
        for x in (p, c):
            x.q.sub_(shift)
    if dtype == torch.float32:
        p.check(first[0])
        c.check(first[1])


@pytest.mark.parametrize("hq,hkv,d", [(2, 1, 64), (1, 1, 128), (1, 1, 48)])
def test_prefill_of_the_longest_rows(hq, hkv, d):
    c = Case([200005, 70000, 33], hq, hkv, d, seed=13, chunks=[5, 40, 33])
    c.check(c.prefill())
    c.check(c.prefill(batch_invariant=True))


@pytest.mark.parametrize("how", ["heads first", "dims apart", "off 16 bytes"])
def test_strides_of_a_padded_head(how):
    c = Case([70, 300, 2200], 6, 2, 80, seed=5, chunks=[30, 140, 11])
    out = attention_tests.strided(torch.zeros_like(c.q), how)
    c.prefill(q=attention_tests.strided(c.q, how), out=out)
    c.check(out)


def test_values_next_to_a_padded_head_do_not_reach_it():
    """q, K and V of the neighbouring heads change; a head's bits do not, with infinities and NaN among q."""
    c = Case([900, 40], 3, 3, 80, seed=2, chunks=[40, 20])
    first = c.prefill()[:, 1].clone()
    q = c.q.clone()
    q[:, 0], q[:, 2] = float("inf"), float("nan")
    for codes in c.cache[:2]:
        codes[:, :, 0], codes[:, :, 2] = 127, -127
    assert torch.equal(c.prefill(q=q)[:, 1], first)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(
    "name,more",
    [
        ("test_decode_at_length_edges", ()),
        ("test_a_block_that_is_not_finite_reaches_only_the_rows_that_see_it", (float("nan"),)),
        ("test_a_block_that_is_not_finite_reaches_only_the_rows_that_see_it", (float("inf"),)),
        ("test_queries_that_are_not_finite_or_huge", ()),
        ("test_softmax_scales_of_zero_and_below", (0.0,)),
        ("test_softmax_scales_of_zero_and_below", (-0.17,)),
        ("test_scales_far_apart", ()),
        ("test_blocks_of_zeros_keep_their_weight", ()),
        ("test_scores_of_channels_of_very_different_sizes_are_sums_in_32_bits", ()),
    ],
)
def test_the_kernel_for_any_shape(name, more, dtype):
    getattr(attention_tests, name)(dtype, 2, 2, 72, *more)


@pytest.mark.parametrize("d", [256, 208])
def test_offsets_past_32_bits_of_large_heads(d):
    attention_tests.test_offsets_past_32_bits(2, 2, d)


@pytest.mark.parametrize("name", ["test_table_entries_outside_the_pool_read_block_0", "test_offsets_past_32_bits", "test_a_row_depends_on_itself_only"])
def test_the_kernel_for_any_shape_and_its_reads(name):
    getattr(attention_tests, name)(2, 2, 72)


def test_rows_of_the_kernel_for_any_shape():
    attention_tests.test_rows_that_see_no_key_are_zero_and_rows_of_no_sequence_are_left(torch.bfloat16, 72)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hkv,d,page", [(3, 8, 16), (2, 24, 16), (5, 40, 32), (3, 80, 16), (2, 96, 16), (1, 176, 16), (2, 320, 16), (2, 504, 7), (2, 36, 16), (3, 65, 16)])
def test_appends_and_reads_of_any_head_size(dtype, hkv, d, page):
    append_tests.test_runs_of_every_length_and_place(dtype, hkv, d, page)
    append_tests.test_reading_back(dtype, hkv, d, page)


@pytest.mark.parametrize("dtype", DTYPES)
def test_an_append_stores_nothing_past_a_head(dtype):
    from vllm_rlt_amd import ops

    cache = random_cache(6, 16, 3, 96, seed=5, layers=2)
    wide = [t.cuda() for t in cache]
    got = [t[..., :80] for t in wide[:2]] + wide[2:]
    k, v = append_tests.tokens(40, 3, 80, dtype, 6, spread=3.0)
    blocks, offsets = append_tests.slots([(9, 30), (0, 1), (5, 9)], 16, 6)
    ops.kv_append_int8(*got, 1, blocks.cuda(), offsets.cuda(), k.cuda(), v.cuda())
    want = [t[..., :80].clone() for t in cache[:2]] + [t.clone() for t in cache[2:]]
    append(want, 1, blocks, offsets, k, v)
    append_tests.same(got, want)
    for t, old in zip(wide[:2], cache[:2]):
        assert torch.equal(t[..., 80:].cpu(), old[..., 80:])
