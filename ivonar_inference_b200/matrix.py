"""The model's packed projections on the device, as the kernels read them (no reference package needed)."""

from __future__ import annotations

import torch
import torch.nn.functional as F
from torch import Tensor

from . import _native as native
from ._native import KernelError


def _pad_rows(packed: Tensor) -> Tensor:
    row_bytes = int(packed.shape[1])
    padded = (row_bytes + 15) // 16 * 16
    return F.pad(packed, (0, padded - row_bytes)) if padded != row_bytes else packed


def _stack(tensors: list[Tensor], interleave: bool) -> Tensor:
    if len(tensors) == 1:
        return tensors[0]
    if interleave:
        return torch.stack(tensors, dim=1).reshape(-1, *tensors[0].shape[1:])
    return torch.cat(tensors, dim=0)


class DeviceMatrix:
    """A row-stack of packed projections on the device, in the layout the kernels read."""

    def __init__(self, projections: list, device: torch.device, interleave: bool = False, scale_align: int = 1) -> None:
        first = projections[0]
        self.in_features = int(first.in_features)
        for proj in projections:
            if int(proj.in_features) != self.in_features:
                raise KernelError("fused projections must share their input width")
            if int(getattr(proj, "group_size", 128)) != 128:
                raise KernelError("ternary kernels need group size 128")
            if proj.weight_scales.dtype != torch.float16:
                raise KernelError("ternary kernels need float16 group scales")
            if interleave and int(proj.out_features) != int(first.out_features):
                raise KernelError("interleaved projections must share their output width")
        packed = _stack([p.packed_weight.to(device) for p in projections], interleave)
        self.packed = _pad_rows(packed).contiguous()
        scales = _stack([p.weight_scales.to(device) for p in projections], interleave)
        stride = (int(scales.shape[1]) + scale_align - 1) // scale_align * scale_align
        if stride != int(scales.shape[1]):
            scales = F.pad(scales, (0, stride - int(scales.shape[1])))
        self.scales = scales.contiguous()
        biases = [p.bias for p in projections]
        if all(b is None for b in biases):
            self.bias = None
        else:
            filled = [torch.zeros(int(p.out_features)) if b is None else b.float() for p, b in zip(projections, biases)]
            self.bias = _stack([b.to(device) for b in filled], interleave).contiguous()
        self.rows = int(self.packed.shape[0])

    def desc(self) -> native.IvbTernary:
        return native.ternary(self.packed, self.scales, self.bias, self.rows, self.in_features)

    @property
    def nbytes(self) -> int:
        return self.packed.numel() + self.scales.numel() * 2 + (0 if self.bias is None else self.bias.numel() * 4)


def rope_from_rotary(rotary, max_len: int) -> Tensor:
    """[max_len, rope_dim/2, 2] (cos, sin) of one attention layer, computed by the reference's own
    ``Rotary.rotate`` on unit vectors (as StaticDecoder._prepare_attention does, decoder.py:177-181)."""

    dim = int(rotary.head_dim)
    unit = torch.zeros(1, max_len, 1, dim, dtype=torch.float32)
    unit[..., 0::2] = 1.0
    return rotary.rotate(unit, offset=0).reshape(max_len, dim // 2, 2).contiguous()
