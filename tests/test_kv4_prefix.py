"""Host-side checks of the attention behind a shared beginning that need no GPU: refusals before any launch, and sizes."""

from __future__ import annotations

import ctypes


def test_the_c_entry_points_refuse_bad_arguments() -> None:
    from ivonar_inference_b200 import _native as native

    lib = native.library()
    buffer = ctypes.create_string_buffer(1 << 12)
    at = (ctypes.addressof(buffer) + 15) // 16 * 16   # never read: every call is refused before a launch
    cache = native.IvbKv4Cache
    good, other = cache(at, 2, 2, 64, 16), cache(at, 1, 2, 64, 1_000_000)   # long enough for a pass of its own

    def call(c=good, prefix=other, lengths=at, groups=None, q=at, dtype=native.IVB_F32, heads=4, starts=None, positions=at, rows=2, window=0, sinks=0,
             out=at, workspace=at, nbytes=1 << 40):
        shared = None if prefix is None else ctypes.byref(native.IvbKv4Prefix(prefix, lengths, groups))
        return lib.ivb_kv4_attention_prefix(None if c is None else ctypes.byref(c), shared, q, dtype, 256, 64, heads, starts, positions, rows, 0.125,
                                            window, sinks, out, 256, 64, workspace, nbytes, None, None)

    def refused(word, **kwargs):
        assert call(**kwargs) == native.IVB_EINVAL, kwargs
        assert word in native.last_error() and "ivb_kv4_attention" in native.last_error()

    refused("null cache", c=None)
    refused("null prefix", prefix=None)
    refused("null cache", prefix=cache(None, 1, 2, 64, 400))
    refused("head_dim", prefix=cache(at, 1, 2, 48, 400))
    refused("behind a prefix of 1 x 64", prefix=cache(at, 1, 1, 64, 400))
    refused("behind a prefix of 2 x 32", prefix=cache(at, 1, 2, 32, 400))
    refused("null lengths", lengths=None)
    refused("without groups", prefix=cache(at, 3, 2, 64, 400))
    refused("positions behind", prefix=cache(at, 1, 2, 64, 2**31 - 256 - 16))
    refused("workspace", workspace=None)
    refused("workspace", workspace=at + 8)
    need = lib.ivb_kv4_prefix_workspace_bytes(ctypes.byref(good), ctypes.byref(native.IvbKv4Prefix(other, at, None)), native.IVB_F32, 4, None, 2)
    refused("workspace", nbytes=need - 1)
    refused("type", dtype=3)
    refused("query heads", heads=3)
    refused("window", window=-1)
    refused("positions", positions=None)
    refused("without starts", rows=3)
    refused("null", q=None)
    assert call(starts=at, rows=0) == native.IVB_OK


def test_workspace_sizes() -> None:
    from ivonar_inference_b200 import _native as native

    lib = native.library()

    def size(batch, kv_heads, dim, prefix_len, dtype, heads, starts, rows, prefixes=1):
        c = native.IvbKv4Cache(1 << 20, batch, kv_heads, dim, 100)
        p = native.IvbKv4Prefix(native.IvbKv4Cache(1 << 20, prefixes, kv_heads, dim, prefix_len), 1 << 20, 1 << 20)
        return lib.ivb_kv4_prefix_workspace_bytes(ctypes.byref(c), ctypes.byref(p), dtype, heads, starts, rows)

    for rows, heads, dim in ((4, 16, 64), (64, 16, 64), (96, 32, 128), (3000, 8, 32)):
        n = size(rows, 8, dim, 20000, native.IVB_F32, heads, None, rows)
        assert n > 0 and n % (rows * heads * (8 + 4 * dim)) == 0 and n // (rows * heads * (8 + 4 * dim)) <= 16
        # short beginnings are walked by each row's kernel
        assert size(rows, 8, dim, 10, native.IVB_F32, heads, None, rows) == 0
    assert size(3000, 8, 32, 100, native.IVB_F32, 8, None, 3000) == 3000 * 8 * (8 + 4 * 32)
    # a lone sequence's prompt needs none, nor do calls that are refused
    assert size(1, 8, 64, 1000, native.IVB_BF16, 8, 1 << 20, 500) == 0
    assert size(2, 8, 64, 1000, native.IVB_BF16, 9, None, 2) == 0 and size(2, 8, 64, 1000, native.IVB_BF16, 8, None, 0) == 0
    assert ctypes.sizeof(native.IvbKv4Prefix) == 40
