"""The block-scaled 8-bit cache's entry points refuse bad arguments before any launch (CPU only)."""

import pytest
import torch
from test_fp8_library import library, refused


def test_append():
    lib, native = library()
    s = native.int64_array([1, 1, 1, 1, 1])

    def call(dtype=2, rows=1, layer=0, layers=1, blocks=4, page=16, heads=2, d=64, scales=16, k=16, strides=s, scale_strides=s, at=16):
        return lib.rlt_kv_append_int8(16, 16, strides, scales, scales, scale_strides, k, s, 16, s, at, at, rows, layer, layers, blocks, page,
                                      heads, d, dtype, None)

    refused(call(dtype=9), native, "dtype")
    refused(call(rows=-1), native, "n_rows")
    for layer in (-1, 1):
        refused(call(layer=layer), native, "layer")
    refused(call(blocks=0), native, "positive")
    refused(call(page=0), native, "positive")
    refused(call(heads=0), native, "positive")
    refused(call(d=513), native, "head_dim", native.RLT_EUNSUPPORTED)
    refused(call(rows=1 << 24), native, "too many rows", native.RLT_EUNSUPPORTED)
    refused(call(page=(1 << 30) + 1), native, "tokens a page", native.RLT_EUNSUPPORTED)
    refused(call(scales=None), native, "NULL")
    refused(call(k=None), native, "NULL")
    refused(call(at=None), native, "NULL")
    refused(call(scale_strides=None), native, "NULL")
    refused(call(scales=18), native, "4 bytes")
    refused(call(strides=native.int64_array([1, 1, -1, 1, 1])), native, "negative")
    refused(call(scale_strides=native.int64_array([1, 1, -1])), native, "negative")
    assert call(rows=0) == native.RLT_OK


def test_gather():
    lib, native = library()
    s = native.int64_array([1, 1, 1, 1, 1])

    def call(dtype=2, rows=1, layer=0, page=16, heads=2, d=64, scales=16, out=16, blocks=16):
        return lib.rlt_kv_gather_int8(16, 16, s, scales, scales, s, blocks, 16, rows, out, out, layer, 1, 4, page, heads, d, dtype, None)

    refused(call(dtype=9), native, "dtype")
    refused(call(rows=-1), native, "n_rows")
    refused(call(layer=1), native, "layer")
    refused(call(page=0), native, "positive")
    refused(call(d=0), native, "positive")
    refused(call(d=513), native, "head_dim", native.RLT_EUNSUPPORTED)
    refused(call(rows=1 << 24), native, "too many rows", native.RLT_EUNSUPPORTED)
    for kw in (dict(scales=None), dict(out=None), dict(blocks=None)):
        refused(call(**kw), native, "NULL")
    refused(call(scales=17), native, "4 bytes")
    assert call(rows=0) == native.RLT_OK


def test_attention():
    lib, native = library()
    s = native.int64_array([1, 1, 1, 1])

    def decode(q=16, rows=1, hq=2, hkv=1, d=64, page=16, blocks=4, width=3, dtype=2, ws=16, ws_bytes=1 << 40, scales=16, ss=s):
        return lib.rlt_paged_decode_int8(q, s, 16, 16, s, scales, scales, ss, 16, width, width, 16, 16, s, rows, hq, hkv, d, page, blocks,
                                         1.0, dtype, ws, ws_bytes, None)

    def prefill(q=16, rows=1, hq=2, hkv=1, d=64, page=16, blocks=4, width=3, dtype=2, cu=16, seqs=1, longest=1, ws=16, ws_bytes=1 << 40,
                scales=16, ss=s):
        return lib.rlt_paged_prefill_int8(q, s, 16, 16, s, scales, scales, ss, 16, width, width, 16, cu, seqs, rows, longest, 16, s, hq,
                                          hkv, d, page, blocks, 1.0, dtype, ws, ws_bytes, None)

    for call in (decode, prefill):
        refused(call(dtype=7), native, "dtype")
        refused(call(hq=3, hkv=2), native, "positive multiple")
        refused(call(hkv=0), native, "positive multiple")
        refused(call(rows=-1), native, "negative")
        refused(call(d=0), native, "positive")
        refused(call(page=0), native, "positive")
        refused(call(blocks=0), native, "positive")
        refused(call(d=520), native, "head_dim", native.RLT_EUNSUPPORTED)
        refused(call(width=0), native, "positive")
        refused(call(width=(1 << 26) + 1), native, "2^30", native.RLT_EUNSUPPORTED)
        refused(call(rows=1 << 23), native, "too many rows", native.RLT_EUNSUPPORTED)
        refused(call(q=None), native, "NULL")
        refused(call(scales=None), native, "NULL")
        refused(call(ss=None), native, "NULL")
        refused(call(scales=18), native, "4 bytes")
        assert call(rows=0) == native.RLT_OK
    refused(prefill(cu=None), native, "NULL")
    refused(prefill(longest=-1), native, "max_seqlen_q")
    need = lib.rlt_paged_decode_int8_workspace_bytes(3, 100, 16, 16, 128, 16)
    if need:
        for kw in (dict(ws_bytes=need - 1), dict(ws=None), dict(ws=24)):
            refused(decode(rows=3, hq=16, hkv=16, d=128, width=100, **kw), native, "workspace", native.RLT_EWORKSPACE)
    need = lib.rlt_paged_prefill_int8_workspace_bytes(300, 3, 100, 16, 16, 128, 16)
    if need:
        for kw in (dict(ws_bytes=need - 1), dict(ws=24)):
            refused(prefill(rows=300, seqs=3, hq=16, hkv=16, d=128, width=100, **kw), native, "workspace", native.RLT_EWORKSPACE)
    for page in (0, -16):
        assert lib.rlt_paged_decode_int8_workspace_bytes(1, 4, 2, 2, 128, page) == 0
        assert lib.rlt_paged_prefill_int8_workspace_bytes(1, 1, 4, 2, 2, 128, page) == 0


def test_launches_past_the_largest_grid():
    lib, native = library()
    q, kv, sc = (native.int64_array(x) for x in ([4096, 64, 1], [4096, 256, 64, 1], [4, 1]))
    rows = (1 << 23) - 1
    refused(lib.rlt_paged_decode_int8(16, q, 16, 16, kv, 16, 16, sc, 16, 3, 3, 16, 16, q, rows, 64, 4, 64, 16, 4, 1.0, 2, 16, 1 << 60,
                                      None), native, "too many rows", native.RLT_EUNSUPPORTED)
    refused(lib.rlt_paged_prefill_int8(16, q, 16, 16, kv, 16, 16, sc, 16, 3, 3, 16, 16, 1, rows, rows, 16, q, 512, 4, 64, 16, 4, 1.0, 2,
                                       None, 0, None), native, "too many rows", native.RLT_EUNSUPPORTED)


@pytest.mark.parametrize("d", [64, 128])
def test_workspaces_are_bounded(d):
    """A decode's: rows, splits of 512 keys, 64 at most; a prefill's: 768 KiB (head_dim + 4) and 65 rows, a plan of 64 sequences."""
    lib, _ = library()
    for rows, hq, hkv, width in [(1, 16, 16, 64), (7, 32, 8, 100), (256, 16, 2, 1 << 20)]:
        splits = min(-(-width * 16 // 512), 64)
        assert lib.rlt_paged_decode_int8_workspace_bytes(rows, width, hq, hkv, d, 16) == rows * splits * hq * (d + 4) * 4
    assert lib.rlt_paged_decode_int8_workspace_bytes(5, 32, 16, 16, d, 16) == 0  # one split: no partials
    for rows in (1, 300, 4096, 1 << 20):
        for seqs in (1, 7, 64):
            for hq, hkv in [(16, 16), (32, 8), (5, 5)]:
                need = lib.rlt_paged_prefill_int8_workspace_bytes(rows, seqs, 1 << 14, hq, hkv, d, 16)
                assert 0 < need <= (768 * 1024 + 65 * hq * 4) * (d + 4) + 64 * 28
    assert lib.rlt_paged_prefill_int8_workspace_bytes(4096, 65, 1 << 14, 16, 16, d, 16) == 0


def test_workspaces_of_other_head_sizes():
    """Multiples of 16 as the next of 64, 128 and 256; none for what runs the kernel for any shape."""
    lib, _ = library()
    decode = lambda d, page=16: lib.rlt_paged_decode_int8_workspace_bytes(3, 1 << 10, 8, 2, d, page)  # noqa: E731
    prefill = lambda d, page=16: lib.rlt_paged_prefill_int8_workspace_bytes(300, 3, 1 << 10, 8, 2, d, page)  # noqa: E731
    for d, like in [(16, 64), (48, 64), (80, 128), (112, 128)]:
        assert decode(d) == decode(like) > 0 and prefill(d) == prefill(like) > 0
    assert decode(144) == decode(240) == decode(256) > 0 and prefill(144) == prefill(240) == prefill(256) > 0
    for d in (8, 72, 100, 272, 512):
        assert decode(d) == prefill(d) == 0
    assert decode(128, 8) == prefill(128, 8) == prefill(128, 48) == 0 and decode(128, 48) > 0


def cache(ndim):
    codes = torch.zeros((2, 1, 16, 2, 64)[5 - ndim :], dtype=torch.int8)
    return [codes, codes.clone(), *(torch.zeros(*codes.shape[: ndim - 3], 2) for _ in "kv")]


def test_host_tensors_are_refused():
    from vllm_rlt_amd import ops

    x, one = torch.zeros(1, 2, 64), torch.zeros(1, dtype=torch.int64)
    tables, lens = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    for call in (
        lambda: ops.paged_decode_int8(x, *cache(4), tables, lens),
        lambda: ops.paged_prefill_int8(x, *cache(4), tables, lens, torch.tensor([0, 1], dtype=torch.int32), 1),
        lambda: ops.kv_append_int8(*cache(5), 0, one, one, x, x),
        lambda: ops.kv_gather_int8(*cache(5), 0, one, one),
    ):
        with pytest.raises(ValueError, match="ROCm device"):
            call()


@pytest.mark.parametrize("ndim", [4, 5])
def test_a_cache_of_another_form_is_refused(ndim):
    from vllm_rlt_amd import ops

    kc, vc, ks, vs = cache(ndim)
    ops._require_int8(kc, vc, ks, vs, ndim)
    for bad, match in [
        ((kc.view(torch.uint8), vc, ks, vs), "int8 codes"),
        ((kc, vc.float(), ks, vs), "int8 codes"),
        ((kc, vc, ks.double(), vs), "float32"),
        ((kc, vc, ks, vs.half()), "float32"),
        ((kc[None], vc[None], ks, vs), "caches must be"),
        ((kc, vc[:1, ..., :32], ks, vs), "share shape"),
        ((kc, vc, ks[..., :1], vs), "scales must be"),
        ((kc, vc, ks[None], vs[None]), "scales must be"),
        ((kc, vc, ks, torch.zeros(*ks.shape, 2)[..., 0]), "scales must be"),
    ]:
        with pytest.raises(ValueError, match=match):
            ops._require_int8(*bad, ndim)
