"""Activations kept in 8 bits between the forward and the backward pass.

Training holds every layer's inputs and pre-activations until the backward
pass has used them; in 16 bits they are most of a step's memory.  Here 32
neighbouring values along the last axis share a power of two ``2**e`` and each
is held as e4m3 (1 sign, 4 exponent, 3 mantissa bits) of ``value / 2**e``:
8.25 bits a value.  ``e`` is the smallest with ``max |value| / 2**e <= 448``,
e4m3's largest, so scaling is exact and the only rounding is e4m3's, to
nearest even: at most 2**-4 of a value, or 2**-10 times ``2**e`` where that
is more.  ``e`` is kept between -118 and 120.  (On the GPU float32 below
2**-126 counts as 0, so that such values come back as 0.)

The largest value of a group is taken over its finite ones; infinities and NaN
come back as NaN, so that a gradient that uses them shows them.  Values that
round up past the type's largest finite one come back as that one.

``linear_act`` and ``gated_linear`` keep their activations this way with
``checkpoint="8bit"``; ``pack_activation`` and ``unpack_activation`` do it for
any tensor.  HIP path: csrc/kernels/act8.hip; on the CPU the same values in
plain PyTorch.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from rocps.ops import hip_ext, require_hip_for

__all__ = ["PackedActivation", "pack_activation", "unpack_activation"]

_GROUP = 32
_TYPES = (torch.bfloat16, torch.float16, torch.float32)


class PackedActivation(NamedTuple):
    """A tensor in 8 bits.  ``codes``: e4m3 bytes, (rows, last axis filled
    with zeros to a multiple of 32); ``scales``: e + 127, one byte a group."""

    codes: torch.Tensor
    scales: torch.Tensor
    shape: torch.Size
    dtype: torch.dtype

    @property
    def nbytes(self) -> int:
        return self.codes.nbytes + self.scales.nbytes


def _pack_cpu(x: torch.Tensor):
    m, n = x.shape
    v = torch.nn.functional.pad(x.float(), (0, -n % _GROUP))
    wide = v.shape[1]
    v = v.reshape(m, wide // _GROUP, _GROUP)
    fine = v.isfinite()
    top = torch.where(fine, v.abs(), 0.0).amax(-1)
    frac, e = torch.frexp(top)
    # 448 is 0.875 * 2**9
    e = (e - 9 + (frac > 0.875).int()).clamp(-118, 120)
    e = torch.where(top > 0, e, -118)
    down = ((127 - e) << 23).view(torch.float32)
    v = torch.where(fine, v * down[..., None], float("nan"))
    codes = v.to(torch.float8_e4m3fn).view(torch.uint8).reshape(m, wide)
    return codes, (e + 127).to(torch.uint8)


def _unpack_cpu(codes, scales, n: int, dtype: torch.dtype) -> torch.Tensor:
    v = codes.view(torch.float8_e4m3fn).float()
    v = v.reshape(*scales.shape, _GROUP)
    v = v * (scales.int() << 23).view(torch.float32)[..., None]
    most = torch.finfo(dtype).max
    v = v.reshape(codes.shape)[:, :n].clamp(-most, most)
    return v.to(dtype).contiguous()


def pack_rows(x: torch.Tensor):
    """(..., n) -> codes, scales."""
    if require_hip_for(x):
        return hip_ext().act8_pack(x)
    if x.dtype not in _TYPES:
        raise TypeError(f"pack_activation: {x.dtype} is not one of {_TYPES}")
    if x.dim() == 0:
        raise ValueError("pack_activation: a scalar has no last axis")
    return _pack_cpu(x.detach().reshape(x.shape[:-1].numel(), x.shape[-1]))


def unpack_rows(codes, scales, shape, dtype: torch.dtype) -> torch.Tensor:
    if require_hip_for(codes):
        return hip_ext().act8_unpack(codes, scales, shape, dtype)
    if dtype not in _TYPES:
        raise TypeError(f"unpack_activation: {dtype} is not one of {_TYPES}")
    n = shape[-1]
    if (codes.shape != (shape[:-1].numel(), (n + 31) // 32 * 32)
            or scales.shape != (codes.shape[0], codes.shape[1] // 32)):
        raise ValueError("unpack_activation: codes and scales as "
                         "pack_activation gives them")
    return _unpack_cpu(codes, scales, n, dtype).reshape(shape)


def pack_activation(x: torch.Tensor) -> PackedActivation:
    """``x`` (any shape but a scalar's; bfloat16, float16 or float32) in 8
    bits, in groups of 32 along its last axis.  Nothing is differentiated
    through it: the values are those of ``x.detach()``."""
    codes, scales = pack_rows(x)
    return PackedActivation(codes, scales, x.shape, x.dtype)


def unpack_activation(packed: PackedActivation,
                      dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """The values that ``packed`` holds, in their own type or in ``dtype``."""
    codes, scales, shape, own = packed
    return unpack_rows(codes, scales, shape, own if dtype is None else dtype)
