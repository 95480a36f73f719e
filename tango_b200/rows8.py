"""Tensors held in 8 bits with one scale per group of neighbouring columns, and activations that keep their input that way.

A tensor is seen as a matrix [size(0), everything else] (1-D: one row) and cut into groups of columns.  A group keeps int8 codes
and one fp32 scale: scale = max|x| / 127, code = x / scale exactly rounded (ties to even), value = code * scale -- off by at most
half a step, 1/254 of the group's largest magnitude.  (`config.set_rounding` applies as it does to the other stand-alone
quantizers.)  A group that holds an infinity or a NaN comes back as NaN.  The reference keeps int8 copies with one scale per
tensor (ctx.backward_cache, cuda/QLinear.py:28-35) and its activations in fp32.
"""
from __future__ import annotations

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import _native

GROUP = 128


class Packed8:
    """A tensor in 8 bits: `codes` int8 [rows, row pitch], `scales` fp32 [rows, groups], and the shape, group and type it had."""
    __slots__ = ("codes", "scales", "shape", "group", "dtype")

    def __init__(self, codes, scales, shape, group, dtype):
        self.codes, self.scales, self.shape, self.group, self.dtype = codes, scales, shape, group, dtype

    @property
    def device(self):
        return self.codes.device

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + 4 * self.scales.numel()

    def to(self, device) -> "Packed8":
        return Packed8(self.codes.to(device), self.scales.to(device), self.shape, self.group, self.dtype)

    def unpack(self, dtype=None) -> torch.Tensor:
        return unpack8(self, dtype)

    def __repr__(self):
        return f"Packed8(shape={tuple(self.shape)}, group={self.group}, dtype={self.dtype}, device={self.device})"


def pack8(x: torch.Tensor, group: int = GROUP) -> Packed8:
    """The 8-bit form of x (fp32, bf16 or fp16, any strides) in groups of `group` columns, 1 to 1024.  Not differentiable."""
    codes, scales = _native.call(_native.ops.pack8, x if not x.requires_grad else x.detach(), group)
    return Packed8(codes, scales, x.shape, group, x.dtype)


def unpack8(packed: Packed8, dtype=None) -> torch.Tensor:
    """The values of a packed tensor, by default in the type it had."""
    return _native.call(_native.ops.unpack8, packed.codes, packed.scales, packed.shape, packed.group, dtype or packed.dtype)


_KINDS = {"elu": 0, "gelu": 1, "silu": 2}
_TORCH = {F.elu: "elu", torch.nn.functional.gelu: "gelu", F.silu: "silu"}


def activation8(x: torch.Tensor, kind: str = "elu", group: int = GROUP) -> torch.Tensor:
    """ELU (alpha = 1), GELU (erf) or SiLU of x, which keeps an 8-bit copy of x for its backward pass in place of x itself: a
    quarter of the memory in fp32, made in the same pass over x.  The output is that of the plain activation to fp32's
    rounding (GELU by a formula of the error function that is off by at most 1.5e-7); the gradient is dy * f'(copy of x).  The three are smooth, so that a copy off by half a step moves the slope by no more than that; a
    ReLU, whose slope hangs on the sign of small values, is not offered."""
    if kind not in _KINDS:
        raise ValueError(f"activation8: {kind!r} is not one of {', '.join(_KINDS)}")
    return _native.call(_native.ops.activation8, x, _KINDS[kind], group)


class Activation8(nn.Module):
    """activation8 as a module."""

    def __init__(self, kind: str = "elu", group: int = GROUP):
        super().__init__()
        if kind not in _KINDS:
            raise ValueError(f"Activation8: {kind!r} is not one of {', '.join(_KINDS)}")
        self.kind, self.group = kind, group

    def forward(self, x):
        return activation8(x, self.kind, self.group)

    def extra_repr(self):
        return f"{self.kind}, group={self.group}"


def in_8_bits(activation):
    """The form with an 8-bit checkpoint of one of PyTorch's activations, given as function or module."""
    kind = _TORCH.get(activation)
    if isinstance(activation, nn.ELU) and activation.alpha == 1:
        kind = "elu"
    elif isinstance(activation, nn.GELU) and activation.approximate == "none":
        kind = "gelu"
    elif isinstance(activation, nn.SiLU):
        kind = "silu"
    if kind is None:
        raise ValueError(f"{activation!r} has no form with an 8-bit checkpoint (ELU with alpha = 1, GELU by erf, SiLU)")
    return Activation8(kind)
