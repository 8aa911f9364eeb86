"""Activations kept between forward and backward in 8 bits
(bdh_activations_save, bdh_activations_restore): e4m3 values with one power of
two for 32 neighbours of a row, 33/32 bytes a value.

A value is off by at most 2^-4 of its magnitude, or by 2^-19 of its block's
largest where it is far below that.  ``gated_block(save=True)`` keeps its two
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


def new_checkpoint(shape, device: torch.device) -> ActivationCheckpoint:
    """Room for values of ``shape``."""
    codes = torch.empty(shape, device=device, dtype=torch.uint8)
    return ActivationCheckpoint(codes, torch.empty((*shape[:-1], -(-shape[-1] // BLOCK)), device=device,
                                                   dtype=torch.uint8))


def check_checkpoint(c: ActivationCheckpoint, shape, device: torch.device, name: str) -> None:
    """Raises ValueError where c does not hold values of ``shape``."""
    want = (tuple(shape), (*shape[:-1], -(-shape[-1] // BLOCK)))
    for t, s in zip(c, want):
        if tuple(t.shape) != s or t.dtype != torch.uint8 or t.device != device or not t.is_contiguous():
            raise ValueError(f"{name} must hold contiguous uint8 tensors of {list(want[0])} and {list(want[1])} "
                             "on the other tensors' device")


def checkpoint_activations(x: torch.Tensor, *, out: Optional[ActivationCheckpoint] = None
                           ) -> Optional[ActivationCheckpoint]:
    """x [..., C] f32 or bf16 on the device in 8 bits, blocks of 32 along the
    last dimension.  A block's power of two is the least with which its largest
    finite magnitude is at most 448 (at least 2^-117); values round to nearest, ties to even;
    infinities and NaN are kept as NaN.  ``out``: a checkpoint to write over.
    None where the library does not support the input (no supported device,
    another dtype, an empty dimension)."""
    dev = x.device
    if not _supported(dev) or x.dim() == 0 or x.numel() == 0:
        return None
    code = _dtype_code(x)
    if code is None:
        return None
    if out is None:
        out = new_checkpoint(x.shape, dev)
    else:
        check_checkpoint(out, x.shape, dev, "out")
    x = x.contiguous()
    C = x.shape[-1]
    st = _call_on(dev, _lib.load().bdh_activations_save, _ptr(x), code, x.numel() // C, C, _ptr(out.codes),
                  _ptr(out.scales), _stream_ptr(dev))
    return out if _lib.check(st) else None


def restore_activations(saved: ActivationCheckpoint, *, dtype: torch.dtype = torch.bfloat16,
                        out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """The values of a checkpoint in ``dtype`` (f32 or bf16, which both hold
    them exactly) or in ``out``.  None where the library does not support the
    input."""
    codes = saved.codes
    dev = codes.device
    if out is not None:
        dtype = out.dtype
    if not _supported(dev) or codes.dim() == 0 or codes.numel() == 0 or dtype not in (torch.float32, torch.bfloat16):
        return None
    check_checkpoint(saved, codes.shape, dev, "saved")
    if out is None:
        out = torch.empty(codes.shape, device=dev, dtype=dtype)
    elif out.shape != codes.shape or out.device != dev or not out.is_contiguous():
        raise ValueError("out must be a contiguous tensor like the saved values")
    C = codes.shape[-1]
    st = _call_on(dev, _lib.load().bdh_activations_restore, _ptr(codes), _ptr(saved.scales), codes.numel() // C, C,
                  _dtype_code(out), _ptr(out), _stream_ptr(dev))
    return out if _lib.check(st) else None
