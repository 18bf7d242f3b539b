"""A key/value cache held in 4 bits, and the attention that reads it, with a sliding window and visible first tokens.

`KV4Cache` holds the keys and values of `batch` sequences: per position and head 4-bit codes with one fp16 scale and one fp16
offset per row of `head_dim` values (`head_dim + 8` bytes for keys and values together, against `8 head_dim` in fp32). Rows
are quantised as they are written (`append`), can be read back (`read`), and are attended to as they stand (`attention`): one
token per sequence, a few drafted ones, whole prompts, or all of these in one call; query heads may share key/value heads.

A call's rows are those of its tensors' first axis. With `starts` (int32 [batch + 1] on the device, ascending) rows
`starts[b] .. starts[b + 1] - 1` belong to sequence `b` and hold its positions `positions[b], positions[b] + 1, ...`
(int64 [batch] on the device); without it there is one row per sequence. Rows from `starts[batch]` on are left as they are.
Rows that `starts` counts beyond either end of the tensors are not there (a call may have a part of the rows, with `starts` less the
number of those before it). A row at a negative position is idle: nothing is written or read for it and its attention is zero. A row at `max_len` or
beyond is treated the same way and reported by `check`. A token is attended to once it is written: `append` first,
then `attention`, on one stream.

Inference only: nothing here is differentiable. The calls allocate nothing but the tensors they return, do not wait for the
GPU, and can be captured in a CUDA graph.
"""

from __future__ import annotations

import ctypes

import torch
from torch import Tensor
from torch.autograd import forward_ad

from . import _native as native

_TYPES = {torch.float32: native.IVB_F32, torch.float16: native.IVB_F16, torch.bfloat16: native.IVB_BF16}


class KV4Cache:
    """Keys and values of `batch` sequences of up to `max_len` positions in 4 bits (`head_dim` 32, 64 or 128).

    `data` is the storage, uint8 [batch, kv_heads, tiles of 16 positions, 16 (head_dim + 8)]; it can be handed in (a buffer
    that the caller keeps, or another cache's). `error` is the device word (int32 [1]) that the calls report to.
    """

    def __init__(self, batch: int, kv_heads: int, head_dim: int, max_len: int, device: str | torch.device | None = None,
                 data: Tensor | None = None, error: Tensor | None = None) -> None:
        if head_dim not in (32, 64, 128):
            raise ValueError(f"head_dim must be 32, 64 or 128, not {head_dim}")
        if batch <= 0 or kv_heads <= 0 or not 0 < max_len < 2**31:
            raise ValueError("batch, kv_heads and max_len must be positive")
        self.lib = native.library()
        self.batch, self.kv_heads, self.head_dim, self.max_len = int(batch), int(kv_heads), int(head_dim), int(max_len)
        shape = (self.batch, self.kv_heads, 2 * ((self.max_len + 31) // 32), 16 * (self.head_dim + 8))
        if data is None:
            target = torch.device("cuda" if device is None else device)
            if target.type != "cuda":
                raise native.KernelError("the 4-bit cache needs a CUDA device")
            data = torch.zeros(shape, dtype=torch.uint8, device=target)
            error = torch.zeros(1, dtype=torch.int32, device=target) if error is None else error
        elif data.dtype != torch.uint8 or tuple(data.shape) != shape or not data.is_cuda or not data.is_contiguous():
            raise ValueError(f"data must be a contiguous uint8 CUDA tensor {list(shape)}")
        elif device is not None and torch.device(device) not in (data.device, torch.device("cuda")):
            raise ValueError("data lies on another device")
        if error is not None and (error.dtype != torch.int32 or error.numel() != 1 or error.device != data.device):
            raise ValueError("error must be an int32 tensor of one value on the cache's device")
        self.data, self.error, self.device = data, error, data.device
        self._error = 0 if error is None else error.data_ptr()
        self._index = data.device.index
        self._sequences = (self.batch,)
        self._desc = native.IvbKv4Cache(data.data_ptr(), self.batch, self.kv_heads, self.head_dim, self.max_len)
        self._ref = ctypes.byref(self._desc)

    @property
    def nbytes(self) -> int:
        return self.data.numel()

    def sequence(self, index: int) -> KV4Cache:
        """The cache of one sequence, over the same storage."""

        if not 0 <= index < self.batch:
            raise IndexError(f"sequence {index} of {self.batch}")
        return KV4Cache(1, self.kv_heads, self.head_dim, self.max_len, data=self.data[index:index + 1], error=self.error)

    def check(self) -> None:
        """Wait for the device; raises ValueError if a call since the last check met a row beyond the capacity, and KernelError
        if a wait inside a kernel ran out (the rows that it concerns are then NaN)."""

        if self.error is None:
            raise RuntimeError("this cache was made without an error word")
        code = int(self.error.item())
        if code != native.IVB_OK:
            self.error.zero_()
            if code != native.IVB_ECAPACITY:
                raise native.KernelError(f"the 4-bit attention reported error {code}")
            raise ValueError(f"a row lies beyond the cache's capacity of {self.max_len} positions")

    # ------------------------------------------------------------------------------------------
    def _rows(self, rows: int, positions: Tensor, starts: Tensor | None) -> int:
        """Checks of what names the rows; the device address of `starts`."""

        if (positions.dtype is not torch.int64 or positions.shape != self._sequences or positions.device != self.device
                or not positions.is_contiguous()):
            raise ValueError(f"positions must be an int64 tensor [{self.batch}] on {self.device}")
        if rows >= 2**31:
            raise ValueError(f"{rows} rows in one call")
        if starts is None:
            if rows != self.batch:
                raise ValueError(f"{rows} rows for {self.batch} sequences need starts")
            return 0
        if (starts.dtype is not torch.int32 or starts.shape != (self.batch + 1,) or starts.device != self.device
                or not starts.is_contiguous()):
            raise ValueError(f"starts must be an int32 tensor [{self.batch + 1}] on {self.device}")
        return starts.data_ptr()

    def _values(self, name: str, x: Tensor, heads: int, dtype: torch.dtype | None = None) -> tuple[int, int]:
        """Checks of rows of values; their strides (row, head)."""

        shape = x.shape
        if len(shape) != 3 or shape[1] != heads or shape[2] != self.head_dim:
            raise ValueError(f"{name} must have shape [rows, {heads}, {self.head_dim}], not {list(shape)}")
        if x.dtype not in _TYPES or (dtype is not None and x.dtype is not dtype):
            raise ValueError(f"{name} has type {x.dtype}" + ("" if dtype is None else f", not {dtype}"))
        if x.device != self.device:
            raise ValueError(f"{name} lies on {x.device}, the cache on {self.device}")
        row, head, channel = x.stride()
        if channel != 1:
            raise ValueError(f"the channels of {name} must be contiguous")
        if x.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name} requires a gradient: the 4-bit cache has none")
        if forward_ad._current_level >= 0 and forward_ad.unpack_dual(x).tangent is not None:
            raise ValueError(f"{name} has a tangent: the 4-bit cache has none")
        return row, head

    def _call(self, what: str, function, *args) -> None:
        index = self._index
        if torch.cuda.current_device() == index:
            rc = function(*args, self._error, torch._C._cuda_getCurrentRawStream(index))
        else:
            with torch.cuda.device(index):
                rc = function(*args, self._error, torch._C._cuda_getCurrentRawStream(index))
        if rc != native.IVB_OK:
            native.check(rc, what)

    def append(self, k: Tensor, v: Tensor, positions: Tensor, starts: Tensor | None = None) -> None:
        """Quantise the key and value rows k, v [rows, kv_heads, head_dim] (fp32, fp16 or bf16) into the cache.

        A row that holds an infinity or a NaN reads back as NaN. The row's offset (its least value) is clipped to +-65504 and its
        scale to 65504: values below the offset, or above it by more than 15 times the scale, are clipped to that.
        """

        k_row, k_head = self._values("k", k, self.kv_heads)
        v_row, v_head = self._values("v", v, self.kv_heads, k.dtype)
        rows = k.shape[0]
        if v.shape[0] != rows:
            raise ValueError(f"{rows} rows of keys and {v.shape[0]} of values")
        at = self._rows(rows, positions, starts)
        self._call("ivb_kv4_append", self.lib.ivb_kv4_append, self._ref, k.data_ptr(), v.data_ptr(), _TYPES[k.dtype], k_row, k_head, v_row,
                   v_head, at, positions.data_ptr(), rows)

    def read(self, positions: Tensor, starts: Tensor | None = None, rows: int | None = None, dtype: torch.dtype = torch.float32,
             out: tuple[Tensor, Tensor] | None = None) -> tuple[Tensor, Tensor]:
        """The rows as the cache holds them: keys and values [rows, kv_heads, head_dim] of type `dtype`.

        `rows` is the number of rows (`batch` by default; with `starts`, which lies on the device, it has to be given) or
        comes with `out`, a pair of tensors to write to; rows that the call does not read are left as they are there, and
        hold nothing of use without `out`. A row holds offset + 15 scale at most, which in fp16 may be infinity: a row from -65504
        to 65504 has the scale 8736 and holds 65536.
        """

        if out is not None:
            k, v = out
            k_row, k_head = self._values("out[0]", k, self.kv_heads)
            v_row, v_head = self._values("out[1]", v, self.kv_heads, k.dtype)
            if v.shape[0] != k.shape[0] or rows not in (None, k.shape[0]):
                raise ValueError("out and rows disagree")
            _writable(k)
            _writable(v)
            _apart(k, v, "the outputs")
            rows = k.shape[0]
        else:
            if rows is None:
                if starts is not None:
                    raise ValueError("rows has to be given with starts")
                rows = self.batch
            if dtype not in _TYPES:
                raise ValueError(f"dtype {dtype}")
            k = self.data.new_empty((rows, self.kv_heads, self.head_dim), dtype=dtype)
            v = torch.empty_like(k)
            k_row = v_row = self.kv_heads * self.head_dim
            k_head = v_head = self.head_dim
        at = self._rows(rows, positions, starts)
        self._call("ivb_kv4_read", self.lib.ivb_kv4_read, self._ref, k.data_ptr(), v.data_ptr(), _TYPES[k.dtype], k_row, k_head, v_row, v_head, at,
                   positions.data_ptr(), rows)
        return k, v

    def attention(self, q: Tensor, positions: Tensor, starts: Tensor | None = None, scale: float | None = None, window: int = 0,
                  sinks: int = 0, out: Tensor | None = None) -> Tensor:
        """Causal attention of the queries q [rows, heads, head_dim] over their sequences' caches, in q's type.

        `heads` is a multiple of `kv_heads`: query head h reads key/value head h // (heads // kv_heads). The row at position p
        sees the positions j <= p with j > p - window, and the first `sinks` positions (window 0: every j <= p). `scale` is
        1 / sqrt(head_dim) by default. `out` may be q itself, but not overlap it otherwise. Products are summed and softmax statistics held in 32 bits.
        With fp32 queries the softmax's weights keep 22 bits; with fp16 and bf16 ones they are rounded to fp16 (by 2^-11 of each at most)
        before they meet the values, but for single tokens with up to four query heads a key/value head.
        Values that pass fp16 (see `read`) may give infinity in an fp16 result.
        """

        heads = q.shape[1] if q.ndim == 3 else 0
        if heads == 0 or heads % self.kv_heads != 0:
            raise ValueError(f"q must have shape [rows, a multiple of {self.kv_heads}, {self.head_dim}]")
        q_row, q_head = self._values("q", q, heads)
        rows = q.shape[0]
        if window < 0 or sinks < 0 or window >= 2**31 or sinks >= 2**31:
            raise ValueError("window and sinks must not be negative")
        if out is None:
            out = torch.empty_like(q)
            o_row, o_head, channel = out.stride()
            if channel != 1:  # of queries whose rows overlap, such as a sliding window's
                out = torch.empty_like(q, memory_format=torch.contiguous_format)
                o_row, o_head, _ = out.stride()
        else:
            o_row, o_head = self._values("out", out, heads, q.dtype)
            if out.shape[0] != rows:
                raise ValueError("out and q disagree")
            _writable(out)
            if out.data_ptr() != q.data_ptr() or out.stride() != q.stride():
                _apart(out, q, "out and q")
        at = self._rows(rows, positions, starts)
        self._call("ivb_kv4_attention", self.lib.ivb_kv4_attention, self._ref, q.data_ptr(), _TYPES[q.dtype], q_row, q_head, heads,
                   at, positions.data_ptr(), rows, self.head_dim**-0.5 if scale is None else scale, window, sinks, out.data_ptr(), o_row,
                   o_head)
        return out


def _places(x: Tensor) -> Tensor:
    """The addresses of the rows of x [rows, heads, head_dim], ascending (int64 on the host)."""

    rows, heads, _ = x.shape
    row, head, _ = x.stride()
    at = torch.arange(rows).mul_(row)[:, None] + torch.arange(heads).mul_(head)
    return at.flatten().mul_(x.element_size()).add_(x.data_ptr()).sort().values


def _writable(x: Tensor) -> None:
    """Refuses an output whose rows share memory."""

    rows, heads, dim = x.shape
    if rows == 0:
        return
    row, head, _ = x.stride()
    # one axis within the other's step, as nearly every layout has it; else the rows one by one
    if (heads == 1 or head >= dim) and (rows == 1 or row >= (heads - 1) * head + dim):
        return
    if (rows == 1 or row >= dim) and (heads == 1 or head >= (rows - 1) * row + dim):
        return
    at = _places(x)
    if bool((at.diff() < dim * x.element_size()).any()):
        raise ValueError("the rows of an output must not overlap")


def _apart(a: Tensor, b: Tensor, names: str) -> None:
    """Refuses an output `a` that shares memory with `b`, another one or an input of the same shape and type."""

    rows, heads, dim = a.shape
    if rows == 0:
        return
    size = a.element_size()
    first, second = (a, b) if a.data_ptr() <= b.data_ptr() else (b, a)
    gap = second.data_ptr() - first.data_ptr()
    row, head, _ = first.stride()
    if gap >= ((rows - 1) * row + (heads - 1) * head + dim) * size:
        return
    # side by side in each row, as a fused projection has them
    if first.stride() == second.stride() and ((heads - 1) * head + dim) * size <= gap <= (row - (heads - 1) * head - dim) * size:
        return
    at, other = _places(a), _places(b)
    after = torch.searchsorted(at, other)
    below, above = at[(after - 1).clamp(min=0)], at[after.clamp(max=at.numel() - 1)]
    if bool(((other - below).abs() < dim * size).any()) or bool(((above - other).abs() < dim * size).any()):
        raise ValueError(f"{names} must not overlap")
