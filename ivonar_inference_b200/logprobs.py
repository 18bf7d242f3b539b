"""Log probabilities of given tokens, the entropy and the likeliest alternatives of rows of logits.

`log_probs` takes the logits of one step or of a whole text, as a decoder's head gives them (`B200Decoder.logits`,
`B200TensorParallel.log_probs` for a head that is sharded by vocabulary), and reads them once. Inference only: nothing here is
differentiable. The calls allocate nothing but what they return, do not wait for the GPU, and can be captured in a CUDA graph.
"""

from __future__ import annotations

from typing import NamedTuple

import torch
from torch import Tensor
from torch.autograd import forward_ad

from . import _native as native

_TYPES = {torch.float32: native.IVB_F32, torch.float16: native.IVB_F16, torch.bfloat16: native.IVB_BF16}
MOST_TOP = 256


class LogProbs(NamedTuple):
    """`tokens`: ln p of the given tokens (fp32, their shape); `entropy`: -sum p ln p (fp32 [rows]); `top`, `ids`: ln p (fp32) and
    token (int64) of the likeliest, [rows, top] in descending order of the logits, the lowest of equal ones first."""

    tokens: Tensor
    entropy: Tensor
    top: Tensor
    ids: Tensor


def _check(logits: Tensor, tokens: Tensor, top: int, temperature: float) -> tuple[int, int]:
    """Checks of a call's arguments; rows and tokens a row."""

    if logits.ndim != 2 or logits.shape[1] == 0 or logits.dtype not in _TYPES:
        raise ValueError(f"logits must be an fp32, fp16 or bf16 tensor [rows, vocabulary], not {logits.dtype} {list(logits.shape)}")
    if not logits.is_cuda:
        raise native.KernelError("log probabilities need a CUDA device")
    rows, vocab = logits.shape
    if logits.stride(1) != 1 and vocab > 1:
        raise ValueError("a row's logits must be contiguous")
    if rows >= 2**28 or vocab >= 2**31:
        raise ValueError(f"{rows} rows of {vocab} logits in one call")
    if tokens.dtype is not torch.int64 or tokens.ndim not in (1, 2) or tokens.shape[0] != rows or tokens.device != logits.device:
        raise ValueError(f"tokens must be an int64 tensor [{rows}] or [{rows}, n] on {logits.device}")
    if not tokens.is_contiguous():
        raise ValueError("tokens must be contiguous")
    if not 0 <= top <= MOST_TOP:
        raise ValueError(f"top must be 0 to {MOST_TOP}, not {top}")
    if not 1e-30 <= temperature <= 1e30:
        raise ValueError("temperature must be positive")
    if logits.requires_grad and torch.is_grad_enabled():
        raise ValueError("the logits require a gradient: log_probs has none")
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(logits).tangent is not None:
        raise ValueError("the logits have a tangent: log_probs has none")
    given = 1 if tokens.ndim == 1 else tokens.shape[1]
    if given >= 2**24:
        raise ValueError(f"{given} tokens a row")
    return rows, given


def _call(what: str, index: int, *args) -> None:
    function = getattr(native.library(), what)
    if torch.cuda.current_device() == index:
        rc = function(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = function(*args, torch._C._cuda_getCurrentRawStream(index))
    native.check(rc, what)


def _empty(logits: Tensor, tokens: Tensor, top: int) -> LogProbs:
    # of other types by their own new_empty, and few keywords: each keyword of a creation costs as much as the kernel's launch
    rows, shape = logits.shape[0], tokens.shape
    like = logits if logits.dtype is torch.float32 else logits.new_empty(0, dtype=torch.float32)
    return LogProbs(like.new_empty(shape), like.new_empty(rows), like.new_empty((rows, top)), torch.empty_strided((rows, top), (max(top, 1), 1), dtype=torch.int64, device=logits.device))


def log_probs(logits: Tensor, tokens: Tensor, top: int = 0, temperature: float = 1.0) -> LogProbs:
    """ln p of `tokens` (int64 [rows] or [rows, n]) under p = softmax(logits / temperature), with the entropy and the `top` likeliest.

    `logits` is [rows, vocabulary] in fp32, fp16 or bf16, each row contiguous; sums are held in 32 bits, of exponentials within 2^-22. A token outside the
    vocabulary (padding, such as -1) has NaN. A logit of -inf has no probability; a row that holds a NaN or +inf, or nothing but
    -inf, has NaN for its values and ids that are tokens all the same.
    """

    rows, given = _check(logits, tokens, top, temperature)
    if top > logits.shape[1]:
        raise ValueError(f"top {top} of a vocabulary of {logits.shape[1]}")
    out = _empty(logits, tokens, top)
    _call("ivb_log_probs", logits.device.index, logits.data_ptr(), _TYPES[logits.dtype], rows, logits.shape[1], logits.stride(0), tokens.data_ptr(),
          given, temperature, top, *(x.data_ptr() for x in out))
    return out


def log_probs_slice(logits: Tensor, tokens: Tensor, v0: int, top: int = 0, temperature: float = 1.0) -> Tensor:
    """The part of a rank whose `logits` are those of the tokens v0, v0 + 1, ...: int32 [rows, 4 + n + 2 top], for `log_probs_merge`."""

    rows, given = _check(logits, tokens, top, temperature)
    if not 0 <= v0 < 2**31 - logits.shape[1]:
        raise ValueError(f"{logits.shape[1]} tokens from {v0} on")
    parts = logits.new_empty((rows, 4 + given + 2 * top), dtype=torch.int32)
    _call("ivb_log_probs_slice", logits.device.index, logits.data_ptr(), _TYPES[logits.dtype], rows, logits.shape[1], v0, logits.stride(0),
          tokens.data_ptr(), given, temperature, top, parts.data_ptr())
    return parts


def log_probs_merge(parts: Tensor, tokens: Tensor, top: int = 0, temperature: float = 1.0) -> LogProbs:
    """What `log_probs` gives over the whole vocabulary, of the slices' parts [slices, rows, 4 + n + 2 top]; `tokens`, `top` and
    `temperature` are those of the slices' calls. Where the slices hold fewer than `top` tokens between them, the places behind these
    have the token -1 and NaN. A slice that comes twice counts twice."""

    if tokens.ndim not in (1, 2):
        raise ValueError("tokens must be those of the slices' calls")
    given = 1 if tokens.ndim == 1 else tokens.shape[1]
    rows = tokens.shape[0]
    if rows >= 2**28 or given >= 2**24:
        raise ValueError(f"{rows} rows of {given} tokens in one call")
    if (parts.dtype is not torch.int32 or parts.ndim != 3 or parts.shape[0] == 0 or tuple(parts.shape[1:]) != (rows, 4 + given + 2 * top)
            or not parts.is_contiguous() or not parts.is_cuda):
        raise ValueError(f"parts must be a contiguous int32 CUDA tensor [slices, {rows}, {4 + given + 2 * top}]")
    if not 0 <= top <= MOST_TOP or not 1e-30 <= temperature <= 1e30:
        raise ValueError(f"top {top}, temperature {temperature}")
    out = _empty(parts[0], tokens, top)
    _call("ivb_log_probs_merge", parts.device.index, parts.data_ptr(), parts.shape[0], rows, given, temperature, top, *(x.data_ptr() for x in out))
    return out
