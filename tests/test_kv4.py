"""Host-side checks of the 4-bit key/value cache that need no GPU: refusals before any launch, and sizes."""

from __future__ import annotations

import ctypes

import pytest


def test_the_c_entry_points_refuse_bad_arguments() -> None:
    from ivonar_inference_b200 import _native as native

    lib = native.library()
    buffer = ctypes.create_string_buffer(4096 + 16)
    address = (ctypes.addressof(buffer) + 15) // 16 * 16   # never read: every call is refused before a launch
    good = native.IvbKv4Cache(address, 2, 2, 64, 16)

    def calls(cache, x=address, dtype=native.IVB_F32, starts=None, positions=address, rows=2, heads=4, window=0, sinks=0):
        ref = None if cache is None else ctypes.byref(cache)
        yield "append", lib.ivb_kv4_append(ref, x, x, dtype, 128, 64, 128, 64, starts, positions, rows, None, None)
        yield "read", lib.ivb_kv4_read(ref, x, x, dtype, 128, 64, 128, 64, starts, positions, rows, None, None)
        yield "attention", lib.ivb_kv4_attention(ref, x, dtype, 256, 64, heads, starts, positions, rows, 0.125, window, sinks, x, 256, 64,
                                                 None, None)

    def refused(word, *args, only=None, **kwargs):
        for name, rc in calls(*args, **kwargs):
            if only is None or name == only:
                assert rc == native.IVB_EINVAL, name
                assert word in native.last_error() and name in native.last_error()

    refused("null cache", None)
    refused("null cache", native.IvbKv4Cache(None, 2, 2, 64, 16))
    for batch, heads, length in ((0, 2, 16), (2, 0, 16), (2, 2, 0), (-1, 2, 16)):
        refused("max_len", native.IvbKv4Cache(address, batch, heads, 64, length))
    for dim in (0, 16, 48, 96, 256):
        refused("head_dim", native.IvbKv4Cache(address, 2, 2, dim, 16))
    refused("aligned", native.IvbKv4Cache(address + 8, 2, 2, 64, 16))
    refused("without starts", good, rows=3)
    refused("rows", good, rows=-1)
    refused("positions", good, positions=None)
    refused("type", good, dtype=3)
    refused("null", good, x=None)
    for heads in (0, 3, -2):
        refused("query heads", good, heads=heads, only="attention")
    refused("window", good, window=-1, only="attention")
    refused("sinks", good, sinks=-1, only="attention")
    # no rows: nothing to do, and nothing is launched
    for name, rc in calls(good, starts=address, rows=0):
        assert rc == native.IVB_OK, name


def test_the_struct_matches_the_c_layout() -> None:
    from ivonar_inference_b200 import _native as native

    # pointer, then four int32 (include/ivonar_b200.h)
    assert ctypes.sizeof(native.IvbKv4Cache) == 24
    assert [getattr(native.IvbKv4Cache, f).offset for f, _ in native.IvbKv4Cache._fields_] == [0, 8, 12, 16, 20]
    assert [f for f, _ in native.IvbKv4Cache._fields_] == ["data", "batch", "kv_heads", "head_dim", "max_len"]


def test_sizes() -> None:
    from ivonar_inference_b200 import _native as native

    lib = native.library()
    assert lib.ivb_kv4_bytes(1, 1, 64, 1) == 2 * 16 * 72
    assert lib.ivb_kv4_bytes(3, 2, 128, 33) == 3 * 2 * 4 * 16 * 136
    assert lib.ivb_kv4_bytes(256, 16, 64, 1 << 24) == 256 * 16 * (1 << 24) * 72
    assert lib.ivb_kv4_bytes(1, 1, 48, 1) == 0 and lib.ivb_kv4_bytes(0, 1, 64, 1) == 0


def test_a_cpu_device_is_refused() -> None:
    from ivonar_inference_b200 import KernelError, KV4Cache

    with pytest.raises(KernelError, match="CUDA"):
        KV4Cache(1, 1, 64, 16, device="cpu")
    with pytest.raises(ValueError, match="head_dim"):
        KV4Cache(1, 1, 65, 16, device="cpu")
