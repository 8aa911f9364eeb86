"""Low-rank adapters of many requests beside a shared projection
(bdh_apply_adapters): the batch's sequences share the model's logits
projection, and each adds its own adapter's product to it,

    out[b] = base[b] + scale[id] * (hidden[b] A[id]^T) B[id]^T,   id = ids[b]

with all adapters of a set in one call.  ``model_forward_logits`` applies a
set to its logits (``adapters=``, ``adapter_ids=``).
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from . import _lib
from .recurrent import _call_on, _dtype_code, _ptr, _stream_ptr, _supported


class AdapterSet(NamedTuple):
    """n adapters of one rank (pad smaller ones with zeros)."""
    a: torch.Tensor       # [n, R, D] bf16: into the rank (a linear layer's [out, in] weight)
    b: torch.Tensor       # [n, V, R] bf16: out of it
    scale: torch.Tensor   # [n] f32 (alpha / R)


# What one call takes: in_dim, out_dim, adapters, batch, batch * time (time goes with the batch), rank.
_MOST_IN, _MOST_OUT, _MOST_ADAPTERS = 1 << 20, 1 << 22, 1 << 20
_MOST_BATCH, _MOST_TIME, _MOST_ROWS, _MOST_RANK = 65535, 65535 * 64, 1 << 23, 128


def _plan(base_shape, hidden_shape, device: torch.device, adapters: AdapterSet,
          ids: torch.Tensor) -> Optional[_lib.BdhAdapterPlan]:
    """adapter_plan without the limits of sizes, which the library checks."""
    B, T, V = base_shape
    Bh, Th, D = hidden_shape
    a, b, scale = adapters
    if a.dim() != 3 or b.dim() != 3 or a.dtype != torch.bfloat16 or b.dtype != torch.bfloat16:
        return None
    n, R, _ = a.shape
    if min(B, T, V, D, n, R) == 0:
        return None
    if (Bh != B or Th != T or a.shape != (n, R, D) or b.shape != (n, V, R)
            or scale.shape != (n,) or ids.shape != (B,)):
        raise ValueError("base, hidden, adapters and ids do not fit together")
    if scale.dtype != torch.float32 or ids.dtype != torch.int32:
        raise ValueError("scale must be f32 and ids int32")
    if not a.device == b.device == scale.device == ids.device == device:
        raise ValueError("base, hidden, adapters and ids must be on one device")
    return _lib.BdhAdapterPlan(B, T, D, V, R, n)


def adapter_plan(base_shape, hidden_shape, device: torch.device, adapters: AdapterSet,
                 ids: torch.Tensor) -> Optional[_lib.BdhAdapterPlan]:
    """The plan of a call on a base [B, T, V] and a hidden [B, T, D] of these
    shapes on ``device``: every check of the adapters and ids, before anything
    is computed.  None where the library does not support them; raises
    ValueError where they do not fit."""
    p = _plan(base_shape, hidden_shape, device, adapters, ids)
    if p is None or (p.rank > _MOST_RANK or p.in_dim > _MOST_IN or p.out_dim > _MOST_OUT
                     or p.adapters > _MOST_ADAPTERS or p.batch > _MOST_BATCH or p.time > _MOST_TIME
                     or p.batch * p.time > _MOST_ROWS):
        return None
    return p


def apply_adapters(base: torch.Tensor, hidden: torch.Tensor, adapters: AdapterSet, ids: torch.Tensor,
                   *, out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """base [B, T, V] and hidden [B, T, D] of one dtype (f32 or bf16), or [B,
    V] and [B, D] for a token a sequence; ids [B] int32 on the device, each
    sequence's adapter (outside [0, n): none).  Returns base plus the
    adapters' products, in a new tensor or in ``out`` (contiguous; ``base``
    itself for in place).  Sums are f32; scale * hidden A^T is held to 2^-24 of
    it in f32 calls, to 2^-16 in bf16 calls, and the result is rounded once.
    The form of a call goes by its sizes: the same call repeats bit for bit, a
    sequence in another batch within these bounds.  None where the library does
    not support the input (no supported device, another dtype, an empty
    dimension, a rank above 128, a scratch that would have to grow under
    capture)."""
    dev, shape = base.device, base.shape
    code = _dtype_code(base)
    if not _supported(dev) or code is None or hidden.dtype != base.dtype:
        return None
    if len(shape) not in (2, 3) or hidden.dim() != len(shape):
        return None
    hidden_shape = hidden.shape
    if len(shape) == 2:
        plan = _plan((shape[0], 1, shape[1]), (hidden_shape[0], 1, hidden_shape[1]), dev, adapters, ids)
    else:
        plan = _plan(shape, hidden_shape, dev, adapters, ids)
    if plan is None:
        return None
    if hidden.device != dev:
        raise ValueError("base, hidden, adapters and ids must be on one device")
    if out is None:
        out = torch.empty(shape, device=dev, dtype=base.dtype)
    elif out.shape != shape or out.dtype != base.dtype or out.device != dev or not out.is_contiguous():
        raise ValueError("out must be a contiguous tensor like base")
    # contiguous copies stay referenced until the launch is enqueued
    a, b, scale = adapters
    base, hidden, a, b = base.contiguous(), hidden.contiguous(), a.contiguous(), b.contiguous()
    scale, ids = scale.contiguous(), ids.contiguous()
    st = _call_on(dev, _lib.load().bdh_apply_adapters, ctypes.byref(plan), code, _ptr(base), _ptr(hidden),
                  _ptr(a), _ptr(b), _ptr(scale), _ptr(ids), _ptr(out), _stream_ptr(dev))
    return out if _lib.check(st) else None
