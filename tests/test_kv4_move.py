"""Host-side checks of the cache's fork and compact that need no GPU: refusals before any launch."""

from __future__ import annotations

import ctypes


def test_the_c_entry_points_refuse_bad_arguments() -> None:
    from ivonar_inference_b200 import _native as native

    lib = native.library()
    buffer = ctypes.create_string_buffer(1 << 16)
    at = (ctypes.addressof(buffer) + 15) // 16 * 16   # never read: every call is refused before a launch
    cache = native.IvbKv4Cache
    good = cache(at, 2, 2, 64, 16)                    # 2 x 2 x 2 tiles of 1152 bytes
    elsewhere = at + 9216

    def fork(c=good, source=cache(elsewhere, 3, 2, 64, 32), sources=at, lengths=at):
        ref = [None if x is None else ctypes.byref(x) for x in (c, source)]
        return lib.ivb_kv4_fork(*ref, sources, lengths, None, None)

    def compact(c=good, index=at, starts=None, positions=at, rows=2):
        return lib.ivb_kv4_compact(None if c is None else ctypes.byref(c), index, starts, positions, rows, None, None)

    def refused(call, word, **kwargs):
        assert call(**kwargs) == native.IVB_EINVAL, kwargs
        assert word in native.last_error() and call.__name__ in native.last_error()

    for call in (fork, compact):
        refused(call, "null cache", c=None)
        refused(call, "null cache", c=cache(None, 2, 2, 64, 16))
        refused(call, "head_dim", c=cache(at, 2, 2, 48, 16))
        refused(call, "aligned", c=cache(at + 8, 2, 2, 64, 16))
        refused(call, "max_len", c=cache(at, 2, 2, 64, 0))
    refused(fork, "null cache", source=cache(None, 2, 2, 64, 16))
    refused(fork, "heads", source=cache(elsewhere, 2, 1, 64, 16))
    refused(fork, "32", source=cache(elsewhere, 2, 2, 32, 16))
    refused(fork, "null", sources=None)
    refused(fork, "null", lengths=None)
    # another cache that begins or ends within this one
    for other in (cache(at + 16, 2, 2, 64, 16), cache(elsewhere - 16, 1, 2, 64, 16), cache(at, 1, 2, 64, 16), cache(at, 2, 2, 64, 17)):
        refused(fork, "share memory", source=other)
    many = cache(at, 4097, 2, 64, 16)
    refused(fork, "within one cache", c=many, source=many)
    refused(fork, "within one cache", c=many, source=None)
    refused(compact, "without starts", rows=3)
    refused(compact, "rows", rows=-1)
    refused(compact, "positions", positions=None)
    refused(compact, "null index", index=None)
    assert compact(starts=at, rows=0) == native.IVB_OK
