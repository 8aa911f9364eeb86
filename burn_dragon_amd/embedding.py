"""The token embedding and its table's gradient (bdh_embed_tokens,
bdh_embed_tokens_vjp): rows of a table times a scale, or through the model's
input norm (DragonModel's LN(embed[tokens]), dragon.rs:3352).  The gradient
sorts the tokens by id and sums each id's rows in the order of the tokens, so
it needs no atomics and repeats bit for bit.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from .recurrent import _call_on, _dtype_code, _ptr, _stream_ptr, _supported


def _table(tokens: torch.Tensor, table: torch.Tensor, device: torch.device) -> Optional[int]:
    """The table's dtype code; None where the library does not take it."""
    if len(table.shape) != 2 or not _supported(device):
        return None
    code = _dtype_code(table)
    if code is None or tokens.numel() == 0 or table.numel() == 0:
        return None
    if tokens.dtype is not torch.int32:
        raise ValueError("tokens must be int32")
    if tokens.device != device:
        raise ValueError("tokens and table must be on one device")
    return code


def embed_tokens(tokens: torch.Tensor, table: torch.Tensor, *, scale: float = 1.0, norm: bool = False,
                 out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """tokens [...] int32 on the device, table [V, D] f32 or bf16 -> [..., D]
    of the table's dtype: ``scale`` times the tokens' rows or, with ``norm``,
    times their LayerNorm (eps 1e-5, no weights), in f32, rounded once.  An id
    outside [0, V) gives a zero row.  ``out``: a contiguous tensor for the
    result.  None where the library does not support the input (no supported
    device, another dtype, an empty dimension, D above 2048, V or tokens
    above 2^24)."""
    dev = table.device
    code = _table(tokens, table, dev)
    if code is None:
        return None
    V, D = table.shape
    shape = (*tokens.shape, D)
    if out is None:
        out = torch.empty(shape, device=dev, dtype=table.dtype)
    elif tuple(out.shape) != shape or out.dtype != table.dtype or out.device != dev or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous {table.dtype} tensor of {list(shape)} on the table's device")
    # contiguous copies stay referenced until the launch is enqueued
    tokens, table = tokens.contiguous(), table.contiguous()
    st = _call_on(dev, _lib.load().bdh_embed_tokens, _ptr(tokens), tokens.numel(), _ptr(table), code, V, D,
                  float(scale), int(norm), _ptr(out), _stream_ptr(dev))
    return out if _lib.check(st) else None


def embed_tokens_vjp(grad: torch.Tensor, tokens: torch.Tensor, table: torch.Tensor, *, scale: float = 1.0,
                     norm: bool = False, out: Optional[torch.Tensor] = None, accumulate: bool = False
                     ) -> Optional[torch.Tensor]:
    """The table's gradient [V, D] from ``grad`` [..., D], the gradient of
    embed_tokens(tokens, table, ...), all of the table's dtype: written whole
    (zeros for ids that no token has), or with ``accumulate`` added to
    ``out``, whose other rows stay untouched.  Sums are f32, in the order of
    the tokens sorted by id; rounded once.  None where the library does not
    support the input (as embed_tokens; a scratch that would have to grow
    under capture)."""
    dev = table.device
    code = _table(tokens, table, dev)
    if code is None:
        return None
    V, D = table.shape
    if tuple(grad.shape) != (*tokens.shape, D) or grad.dtype != table.dtype or grad.device != dev:
        raise ValueError(f"grad must be {table.dtype} of {[*tokens.shape, D]} on the table's device")
    if accumulate and out is None:
        raise ValueError("accumulate adds to out")
    if out is None:
        out = torch.empty((V, D), device=dev, dtype=table.dtype)
    elif tuple(out.shape) != (V, D) or out.dtype != table.dtype or out.device != dev or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous {table.dtype} tensor of {[V, D]} on the table's device")
    tokens, table, grad = tokens.contiguous(), table.contiguous(), grad.contiguous()
    st = _call_on(dev, _lib.load().bdh_embed_tokens_vjp, _ptr(tokens), tokens.numel(), _ptr(table), code, V, D,
                  float(scale), int(norm), _ptr(grad), _ptr(out), int(accumulate), _stream_ptr(dev))
    return out if _lib.check(st) else None
