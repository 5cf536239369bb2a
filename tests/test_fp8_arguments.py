"""What the 8-bit cache's calls hand to the library, and what it refuses at the limits (CPU only)."""

import contextlib

import numpy as np
import pytest
import torch


class Library:
    """Stands for the loaded library: keeps the arguments of every call, launches nothing."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return 0

        return call


@pytest.fixture
def library(monkeypatch):
    from vllm_rlt_amd import _native, ops

    lib = Library()
    monkeypatch.setattr(_native, "load", lambda: lib)
    monkeypatch.setattr(ops, "_require_rocm", lambda *t: t[0].device)
    monkeypatch.setattr(ops, "_current", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(ops, "stream_handle", lambda device: None)
    monkeypatch.setattr(torch.Tensor, "is_pinned", lambda t: True)
    return lib


@pytest.mark.parametrize("size", [1, 3])
def test_the_stride_of_out_tables_goes_to_the_library_as_it_is(library, size):
    # Rows that share their memory have stride 0, which the library refuses: it writes size rows of out_width entries.
    from vllm_rlt_amd import ops

    long = lambda: torch.empty(9, dtype=torch.int64)  # noqa: E731
    short = lambda *n: torch.empty(n, dtype=torch.int32)  # noqa: E731
    for out in (short(size, 8), short(1, 8).expand(size, 8), short(size, 12)[:, :8]):
        ops.build_chunk_metadata(torch.zeros(size, 4, dtype=torch.int64), size, size, short(4, 1, 8), 16, short(size + 1), short(size),
                                 long(), long(), long(), long(), out, 8)
        name, args = library.calls.pop()
        assert name == "rlt_build_chunk_metadata" and args[-2] == 8
        assert args[-3] == out.stride(0) or size == 1 and args[-3] >= 8


@pytest.mark.parametrize("kind", [tuple, list, bytes, torch.tensor, np.array, lambda x: np.array(x, dtype=np.int32)])
def test_axes_of_any_sequence_go_to_the_library_as_one_byte_each(library, kind):
    # An array's own bytes would be eight or four an axis.
    from vllm_rlt_amd import ops

    cache = torch.zeros(2, 1, 16, 1, 8)
    x, one = torch.zeros(1, 1, 8), torch.zeros(1, dtype=torch.int64)

    def rope(axes):
        ops.rope_axes_kv_append(cache, cache.clone(), 0, one, one, x, x, x, one[:, None].expand(1, 3), torch.zeros(5, 4, 2), axes)
        return next(a for a in library.calls.pop()[1] if isinstance(a, bytes))

    assert rope(kind((0, 1, 2, 1))) == bytes([0, 1, 2, 1])
    for bad in ([0, 1, 2, -1], [0, 1, 2, 256], np.array([0, 1, 2, 300])):
        with pytest.raises(ValueError):
            rope(bad)


@pytest.mark.parametrize("rows", [4 * ((1 << 24) - 1) + 1, (1 << 26) - 1])
def test_appends_of_more_rows_than_a_grid_holds_are_refused(rows):
    # Four rows a workgroup of 256 threads, of which a launch has fewer than 2^24.
    from test_fp8_library import library, refused

    lib, native = library()
    s = native.int64_array([1 << 20, 1 << 18, 256, 64, 1])
    x = native.int64_array([128, 64, 1])
    refused(lib.rlt_kv_append_fp8(16, 16, s, 16, 16, s, 16, x, 16, x, 16, 16, rows, 0, 1, 4, 16, 2, 64, 2, None), native, "too many rows",
            native.RLT_EUNSUPPORTED)
    refused(lib.rlt_rope_axes_kv_append(16, 16, s, 16, 16, s, 16, x, 16, x, 16, x, 16, x, 16, x, 1, 16, 10, bytes(32), 32, 16, 16, rows,
                                        rows, 0, 1, 4, 16, 2, 2, 64, 2, None), native, "too many rows", native.RLT_EUNSUPPORTED)


@pytest.mark.parametrize("rows,seqs,width,heads,d,most", [(32768, 32, 256, 32, 128, 100), (4096, 8, 1056, 16, 128, 82), (1 << 18, 64, 4096, 16, 64, 52)])
def test_the_prefill_workspace_holds_cut_sequences_only(rows, seqs, width, heads, d, most):
    # MiB, whatever the rows: 2 * 128 * 768 / heads rows of partials of 4 (d + 2) bytes a head.
    from test_fp8_library import library

    lib, _ = library()
    assert 0 < lib.rlt_paged_prefill_fp8_workspace_bytes(rows, seqs, width, heads, heads, d, 16) <= most << 20
