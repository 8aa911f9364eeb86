"""Activations kept between forward and backward in 8 bits
(bdh_activations_save, bdh_activations_restore): e4m3 values with one power of
two for 32 neighbours of a row, 33/32 bytes a value.

A value is off by at most 2^-4 of its magnitude, or by 2^-17 of its block's
largest where it is far below that (by 2^-127 in a block of which nothing passes
2^-109).  ``gated_block(save=True)`` keeps its two
projections so, and ``gated_block_vjp(saved=...)`` reads them.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib
from .recurrent import _call_on, _dtype_code, _ptr, _stream_ptr, _supported

BLOCK = 32


class ActivationCheckpoint(NamedTuple):
    codes: torch.Tensor     # [..., C] uint8: e4m3
    scales: torch.Tensor    # [..., ceil(C / 32)] uint8: the power's exponent plus 127


def _scales_shape(shape) -> tuple:
    return (*shape[:-1], (shape[-1] + BLOCK - 1) // BLOCK)


def new_checkpoint(shape, device: torch.device) -> ActivationCheckpoint:
    """Room for values of ``shape``."""
    u8 = torch.uint8
    return ActivationCheckpoint(torch.empty(shape, device=device, dtype=u8),
                                torch.empty(_scales_shape(shape), device=device, dtype=u8))


def check_checkpoint(c: ActivationCheckpoint, shape, device: torch.device, name: str) -> None:
    """Raises ValueError where c does not hold values of ``shape``."""
    codes, scales = c
    u8 = torch.uint8
    if (codes.shape != shape or scales.shape != _scales_shape(shape) or codes.dtype is not u8 or scales.dtype is not u8
            or codes.device != device or scales.device != device or not codes.is_contiguous()
            or not scales.is_contiguous()):
        raise ValueError(f"{name} must hold contiguous uint8 tensors of {list(shape)} and "
                         f"{list(_scales_shape(shape))} on the other tensors' device")


def checkpoint_activations(x: torch.Tensor, *, out: Optional[ActivationCheckpoint] = None
                           ) -> Optional[ActivationCheckpoint]:
    """x [..., C] f32 or bf16 on the device in 8 bits, blocks of 32 along the
    last dimension.  A block's power of two is the least with which its largest
    finite magnitude is at most 448 (at least 2^-117); values round to nearest, ties to even;
    infinities and NaN are kept as NaN.  ``out``: a checkpoint to write over.
    None where the library does not support the input (no supported device,
    another dtype, an empty dimension)."""
    dev, shape, n = x.device, x.shape, x.numel()
    if not _supported(dev) or not shape or n == 0:
        return None
    code = _dtype_code(x)
    if code is None:
        return None
    x = x.contiguous()
    C = shape[-1]
    if out is None:
        u8 = torch.uint8
        out = ActivationCheckpoint(torch.empty_like(x, dtype=u8), torch.empty(_scales_shape(shape), device=dev, dtype=u8))
    else:
        check_checkpoint(out, shape, dev, "out")
    st = _call_on(dev, _lib.load().bdh_activations_save, _ptr(x), code, n // C, C, _ptr(out.codes),
                  _ptr(out.scales), _stream_ptr(dev))
    return out if _lib.check(st) else None


def restore_activations(saved: ActivationCheckpoint, *, dtype: torch.dtype = torch.bfloat16,
                        out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """The values of a checkpoint in ``dtype`` (f32 or bf16, which both hold
    them exactly) or in ``out``.  None where the library does not support the
    input."""
    codes = saved.codes
    dev, shape, n = codes.device, codes.shape, codes.numel()
    if out is not None:
        dtype = out.dtype
    code = _lib.BDH_BF16 if dtype is torch.bfloat16 else _lib.BDH_F32 if dtype is torch.float32 else None
    if not _supported(dev) or not shape or n == 0 or code is None:
        return None
    check_checkpoint(saved, shape, dev, "saved")
    if out is None:
        out = torch.empty(shape, device=dev, dtype=dtype)
    elif out.shape != shape or out.device != dev or not out.is_contiguous():
        raise ValueError("out must be a contiguous tensor like the saved values")
    C = shape[-1]
    st = _call_on(dev, _lib.load().bdh_activations_restore, _ptr(codes), _ptr(saved.scales), n // C, C, code,
                  _ptr(out), _stream_ptr(dev))
    return out if _lib.check(st) else None
