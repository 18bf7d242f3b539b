"""Host-side checks of the log probabilities that need no GPU: refusals before any launch."""

from __future__ import annotations

import ctypes

import pytest
import torch


def test_the_c_entry_points_refuse_bad_arguments() -> None:
    from ivonar_inference_b200 import _native as native

    lib = native.library()
    at = ctypes.addressof(ctypes.create_string_buffer(4096))   # never read: every call is refused before a launch

    def whole(x=at, dtype=native.IVB_F32, rows=2, vocab=50, stride=50, tokens=at, given=1, t=1.0, top=3, out=at, entropy=at):
        return lib.ivb_log_probs(x, dtype, rows, vocab, stride, tokens, given, t, top, out, entropy, out, out, None)

    def part(x=at, dtype=native.IVB_F32, rows=2, vocab=50, stride=50, tokens=at, given=1, t=1.0, top=3, out=at, v0=0):
        return lib.ivb_log_probs_slice(x, dtype, rows, vocab, v0, stride, tokens, given, t, top, out, None)

    def merge(parts=at, world=2, rows=2, given=1, t=1.0, top=3, out=at, entropy=at):
        return lib.ivb_log_probs_merge(parts, world, rows, given, t, top, out, entropy, out, out, None)

    def refused(call, word, **kwargs):
        assert call(**kwargs) == native.IVB_EINVAL, (call.__name__, kwargs)
        assert word in native.last_error() and "ivb_log_probs" in native.last_error(), native.last_error()

    for call in (whole, part):
        refused(call, "null logits", x=None)
        refused(call, "type", dtype=3)
        refused(call, "stride", stride=-1)
        refused(call, "vocabulary", vocab=0)
        refused(call, "null tokens", tokens=None)
    for call in (whole, part, merge):
        refused(call, "rows", rows=-1)
        refused(call, "tokens", given=-1)
        refused(call, "top", top=-1)
        refused(call, "top", top=257)
        for t in (0.0, -1.0, float("nan"), float("inf"), 1e-38):
            refused(call, "temperature", t=t)
        refused(call, "null", out=None)
        assert call(rows=0) == native.IVB_OK
    refused(whole, "vocabulary of 50", top=51)
    refused(whole, "null output", entropy=None)
    refused(merge, "null", entropy=None)
    refused(part, "from -1", v0=-1)
    refused(part, "on", v0=2**31 - 50)
    refused(merge, "slices", world=0)
    refused(merge, "null", parts=None)


def test_refusals() -> None:
    from ivonar_inference_b200 import KernelError, log_probs

    x, tokens = torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(KernelError, match="CUDA"):
        log_probs(x, tokens)
    for bad in (x[0], x.double(), x.long(), x[:, :0], x[None]):
        with pytest.raises(ValueError, match="logits must be"):
            log_probs(bad, tokens)


def test_a_merge_refuses_sizes_that_a_slice_refuses() -> None:
    """Sizes that 32 bits do not hold would be cut to their low ones in the call."""
    from ivonar_inference_b200.logprobs import log_probs_merge

    for shape in ((2**28,), (2**32 + 1,), (2, 2**24), (1, 2**32)):
        tokens = torch.empty(shape, dtype=torch.int64, device="meta")
        words = 4 + (shape[1] if len(shape) == 2 else 1)
        with pytest.raises(ValueError, match="in one call"):
            log_probs_merge(torch.empty(1, shape[0], words, dtype=torch.int32, device="meta"), tokens)
