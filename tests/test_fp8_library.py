"""The 8-bit cache's entry points refuse bad arguments before any launch (CPU only)."""

import pytest
import torch


def library():
    from vllm_rlt_amd import _native

    if not _native.LIBRARY_PATH.exists():
        from vllm_rlt_amd._build import build

        build()
    return _native.load(), _native


def refused(rc, native, text, code=None):
    assert rc == (native.RLT_EINVAL if code is None else code)
    assert text in native.last_error()


def test_append():
    lib, native = library()
    s = native.int64_array([1, 1, 1, 1, 1])

    def call(dtype=2, rows=1, layer=0, layers=1, blocks=4, page=16, heads=2, d=64, scales=1, k=1, strides=s):
        return lib.rlt_kv_append_fp8(1, 1, strides, scales, scales, s, k, s, 1, s, 1, 1, rows, layer, layers, blocks, page, heads, d,
                                     dtype, None)

    refused(call(dtype=9), native, "dtype")
    refused(call(rows=-1), native, "n_rows")
    refused(call(layer=1), native, "layer")
    refused(call(blocks=0), native, "positive")
    refused(call(heads=0), native, "positive")
    refused(call(d=513), native, "head_dim", native.RLT_EUNSUPPORTED)
    refused(call(scales=None), native, "NULL")
    refused(call(k=None), native, "NULL")
    refused(call(rows=1 << 26), native, "too many rows", native.RLT_EUNSUPPORTED)
    refused(call(strides=native.int64_array([1, 1, -1, 1, 1])), native, "negative")
    assert call(rows=0) == native.RLT_OK


def test_rotation():
    lib, native = library()
    s = native.int64_array([1, 1, 1, 1, 1])

    def call(axes=2, most=10, axis_of=bytes([0, 1]), half=2, rows=1, write=1, hq=2, hkv=1, d=4, dtype=2, table=1, scales=(1, 1), strides=s):
        return lib.rlt_rope_axes_kv_append(1, 1, s, *scales, strides, 1, s, 1, s, 1, s, 1, s, 1, s, axes, table, most, axis_of, half, 1, 1,
                                           rows, write, 0, 1, 4, 16, hq, hkv, d, dtype, None)

    refused(call(axes=0), native, "axes")
    refused(call(axes=5), native, "axes")
    refused(call(axis_of=bytes([0, 2])), native, "axis past the last")
    refused(call(half=3), native, "more dims")
    refused(call(half=0), native, "more dims")
    refused(call(most=0), native, "no positions")
    refused(call(write=2), native, "n_write")
    refused(call(hq=0), native, "num_q_heads")
    refused(call(table=None), native, "NULL")
    refused(call(scales=(1, None)), native, "NULL")
    refused(call(strides=None), native, "NULL")
    refused(call(dtype=3), native, "dtype")
    assert call(rows=0, write=0) == native.RLT_OK


def test_attention():
    lib, native = library()
    s = native.int64_array([1, 1, 1, 1])

    def decode(q=1, rows=1, hq=2, hkv=1, d=64, page=16, blocks=4, width=3, dtype=2, ws=1, ws_bytes=1 << 40):
        return lib.rlt_paged_decode_fp8(q, s, 1, 1, s, 1, 1, s, 1, width, width, 1, 1, s, rows, hq, hkv, d, page, blocks, 1.0, dtype, ws,
                                        ws_bytes, None)

    def prefill(q=1, rows=1, hq=2, hkv=1, d=64, page=16, blocks=4, width=3, dtype=2, cu=1, seqs=1, longest=1):
        return lib.rlt_paged_prefill_fp8(q, s, 1, 1, s, 1, 1, s, 1, width, width, 1, cu, seqs, rows, longest, 1, s, hq, hkv, d, page,
                                         blocks, 1.0, dtype, 1, 1 << 40, None)

    for call in (decode, prefill):
        refused(call(dtype=7), native, "dtype")
        refused(call(hq=3, hkv=2), native, "positive multiple")
        refused(call(hkv=0), native, "positive multiple")
        refused(call(rows=-1), native, "negative")
        refused(call(d=0), native, "positive")
        refused(call(d=520), native, "head_dim", native.RLT_EUNSUPPORTED)
        refused(call(width=0), native, "positive")
        refused(call(width=(1 << 26) + 1), native, "2^30", native.RLT_EUNSUPPORTED)
        refused(call(rows=1 << 23), native, "too many rows", native.RLT_EUNSUPPORTED)
        refused(call(q=None), native, "NULL")
        assert call(rows=0) == native.RLT_OK
    refused(prefill(cu=None), native, "NULL")
    refused(prefill(longest=-1), native, "max_seqlen_q")
    need = lib.rlt_paged_decode_fp8_workspace_bytes(3, 100, 16, 16, 128, 16)
    if need:
        refused(decode(rows=3, hq=16, hkv=16, d=128, width=100, ws_bytes=need - 1), native, "workspace", native.RLT_EWORKSPACE)


def test_launches_past_the_largest_grid():
    lib, native = library()
    q, kv, sc = (native.int64_array(x) for x in ([4096, 64, 1], [4096, 256, 64, 1], [64, 4, 1]))
    rows = (1 << 23) - 1
    refused(lib.rlt_paged_decode_fp8(16, q, 16, 16, kv, 16, 16, sc, 16, 3, 3, 16, 16, q, rows, 64, 4, 64, 16, 4, 1.0, 2, 16, 1 << 60,
                                     None), native, "too many rows", native.RLT_EUNSUPPORTED)
    refused(lib.rlt_paged_prefill_fp8(16, q, 16, 16, kv, 16, 16, sc, 16, 3, 3, 16, 16, 1, rows, rows, 16, q, 512, 4, 64, 16, 4, 1.0, 2,
                                      None, 0, None), native, "too many rows", native.RLT_EUNSUPPORTED)


def test_chunk_metadata():
    lib, native = library()

    def call(count=1, size=2, width=8, planes=1, page=16, capacity=9, out_width=8, stride=8, desc=1, positions=1):
        return lib.rlt_build_chunk_metadata(desc, count, size, 1, 4, width, planes, page, 1, 1, positions, 1, 1, 1, capacity, 1, stride,
                                            out_width, None)

    refused(call(count=3), native, "count")
    refused(call(count=-1), native, "count")
    refused(call(planes=0), native, "positive")
    refused(call(page=0), native, "positive")
    refused(call(out_width=9), native, "out_width")
    refused(call(stride=7), native, "out_table_stride")
    refused(call(capacity=-1), native, "31 bits", native.RLT_EUNSUPPORTED)
    refused(call(width=1 << 28), native, "31 bits", native.RLT_EUNSUPPORTED)
    refused(call(desc=None), native, "NULL")
    refused(call(positions=None), native, "NULL")
    refused(call(size=(1 << 24) - 1), native, "too many sequences", native.RLT_EUNSUPPORTED)


def test_host_tensors_are_refused():
    from vllm_rlt_amd import ops

    codes = torch.zeros(1, 16, 1, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)
    scales = torch.zeros(1, 16, 1, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    x, one = torch.zeros(1, 1, 64), torch.zeros(1, dtype=torch.int64)
    tables, lens = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    for call in (
        lambda: ops.paged_decode_fp8(x, codes, codes, scales, scales, tables, lens),
        lambda: ops.paged_prefill_fp8(x, codes, codes, scales, scales, tables, lens, torch.tensor([0, 1], dtype=torch.int32), 1),
        lambda: ops.kv_append_fp8(codes[:, None], codes[:, None], scales[:, None], scales[:, None], 0, one, one, x, x),
        lambda: ops.rope_axes_kv_append(codes[:, None], codes[:, None], 0, one, one, x, x, x, one[:, None], torch.zeros(4, 32, 2),
                                        (0,) * 32, scales[:, None], scales[:, None]),
        lambda: ops.build_chunk_metadata(torch.zeros(1, 4, dtype=torch.int64), 1, 1, torch.zeros(1, 1, 1, dtype=torch.int32), 16, lens,
                                         lens, one, one, one, one, tables, 1),
    ):
        with pytest.raises(ValueError, match="ROCm device"):
            call()


def test_the_decode_workspace_holds_the_splits_of_shorter_rows():
    # 64 splits of 256 (512 on the matrix cores) keys in a row of 16384 (32768); a row of one page more has 33.
    lib, _ = library()
    for heads, page_keys in (((1, 1), 256), ((4, 1), 512)):
        for pages in (64 * page_keys // 16, 64 * page_keys // 16 + 1, 64 * page_keys // 16 + 1000):
            assert lib.rlt_paged_decode_fp8_workspace_bytes(1, pages, *heads, 64, 16) >= 64 * heads[0] * (64 + 2) * 4
        assert lib.rlt_paged_decode_fp8_workspace_bytes(1, page_keys // 16, *heads, 64, 16) == 0


def test_a_page_of_no_tokens_is_refused():
    lib, native = library()
    for page in (0, -16):
        assert lib.rlt_paged_decode_fp8_workspace_bytes(1, 4, 2, 2, 128, page) == 0
        assert lib.rlt_paged_prefill_fp8_workspace_bytes(1, 1, 4, 2, 2, 128, page) == 0
