"""The gated block of latents and its backward pass (bdh_gated_block_fwd,
bdh_gated_block_vjp), bf16 with f32 sums:

    p   = current up_h - th,  q = context_h gate_h - th     a head h, [B, T, N]
    out = u(p) mask * act(q) mask                           [B, T, H * N]

``activation="relu"`` (u = act = ReLU) is the layer's y
(residual_stream.rs:440-505: up the encoder, gate the encoder_v, context the
normalised attention output); "silu" and "gelu" (u(p) = p) an ordinary gated
feed-forward block.  One kernel computes both projections, the activation and
the product; the backward takes the four products over the projections'
gradients, either from the projections computed again or from what the
forward kept of them in 8 bits.
"""
from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple, Optional

import torch

from . import _lib
from .activations import ActivationCheckpoint, check_checkpoint, new_checkpoint
from .recurrent import _call_on, _ptr, _stream_ptr, _supported

ACTIVATIONS = {"relu": _lib.BDH_RELU, "silu": _lib.BDH_SILU, "gelu": _lib.BDH_GELU}


class GatedWeights(NamedTuple):
    up: torch.Tensor      # [H, D, N] bf16 (the encoder's layout)
    gate: torch.Tensor    # [H, D, N] bf16 (the encoder_v's)


class GatedSaved(NamedTuple):
    """What the backward reads in place of the projections: p and q (with
    "relu" after the ReLU) in 8 bits, [B, T, H, N] each."""
    up: ActivationCheckpoint
    gate: ActivationCheckpoint


class GatedOutput(NamedTuple):
    out: torch.Tensor                  # [B, T, H * N] bf16
    saved: Optional[GatedSaved]


class GatedGrads(NamedTuple):
    current: torch.Tensor              # [B, T, D] bf16
    context: Optional[torch.Tensor]    # [B, H, T, D] bf16 (None without a context)
    up: torch.Tensor                   # [H, D, N] bf16
    gate: torch.Tensor                 # [H, D, N] bf16


@functools.lru_cache(maxsize=1024)
def _plan_of(B: int, H: int, T: int, N: int, D: int):
    """The library's plan of a shape, by reference (it reads it only)."""
    return ctypes.byref(_lib.BdhLayerPlan(B, H, T, N, D))


@functools.lru_cache(maxsize=1024)
def _options_of(activation: int, threshold: float):
    return ctypes.byref(_lib.BdhGatedOptions(activation, threshold, None))


def _call(current, weights, context, activation, relu_threshold, latent_mask):
    """(device, (B, H, T, N, D), plan, options, tensors) of a call; None where
    the library does not support it, ValueError where the arguments do not
    fit together."""
    kind = ACTIVATIONS.get(activation)
    if kind is None:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}")
    up, gate = weights
    dev, bf16 = current.device, torch.bfloat16
    x_shape, w_shape = current.shape, up.shape
    if not _supported(dev) or len(x_shape) != 3 or len(w_shape) != 3 or len(gate.shape) != 3:
        return None
    if (current.dtype is not bf16 or up.dtype is not bf16 or gate.dtype is not bf16
            or (context is not None and context.dtype is not bf16)):
        return None
    B, T, D = x_shape
    H, _, N = w_shape
    if 0 in (B, T, D, H, N):
        return None
    if w_shape[1] != D or gate.shape != w_shape:
        raise ValueError("up and gate must be [H, D, N] with current's D")
    if context is not None and context.shape != (B, H, T, D):
        raise ValueError(f"context must be {[B, H, T, D]}")
    mask = None
    if latent_mask is not None:
        mask = latent_mask.reshape(-1)
        if mask.numel() != N or mask.dtype is not torch.float32:
            raise ValueError(f"latent_mask must hold {N} f32 values")
    if (up.device != dev or gate.device != dev or (context is not None and context.device != dev)
            or (mask is not None and mask.device != dev)):
        raise ValueError("the tensors must be on one device")
    if kind != _lib.BDH_RELU and (relu_threshold != 0.0 or mask is not None):
        raise ValueError('relu_threshold and latent_mask go with activation="relu"')
    if N % 8 or D % 8:
        return None
    tensors = [_aligned(current), _aligned(context), _aligned(up), _aligned(gate)]
    if mask is None:
        options = _options_of(kind, float(relu_threshold))
    else:
        mask = _aligned(mask)
        tensors.append(mask)   # (held until the launch is enqueued)
        options = ctypes.byref(_lib.BdhGatedOptions(kind, float(relu_threshold), _ptr(mask)))
    return dev, (B, H, T, N, D), _plan_of(B, H, T, N, D), options, tensors


def _aligned(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """Contiguous, from a 16-byte boundary on."""
    if t is None:
        return None
    if not t.is_contiguous():
        t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def gated_block(current: torch.Tensor, weights: GatedWeights, context: Optional[torch.Tensor] = None, *,
                activation: str = "relu", relu_threshold: float = 0.0, latent_mask: Optional[torch.Tensor] = None,
                save: bool = False) -> Optional[GatedOutput]:
    """current [B, T, D] and context [B, H, T, D] (None: current for all
    heads) bf16 on the device -> out [B, T, H * N] bf16, the decoder's operand.
    ``save`` also keeps the projections in 8 bits for gated_block_vjp.
    ``relu_threshold`` and ``latent_mask`` ([N] f32) are the layer's projection
    options, with "relu" alone.  None where the library does not support the
    input (no supported device, another dtype, an empty dimension, D or N not
    a multiple of 8 or too large)."""
    call = _call(current, weights, context, activation, relu_threshold, latent_mask)
    if call is None:
        return None
    dev, (B, H, T, N, D), plan, options, t = call
    out = torch.empty((B, T, H * N), device=dev, dtype=torch.bfloat16)
    saved, parts = None, (None, None, None, None)
    if save:
        saved = GatedSaved(new_checkpoint((B, T, H, N), dev), new_checkpoint((B, T, H, N), dev))
        parts = [_ptr(p) for c in saved for p in c]
    st = _call_on(dev, _lib.load().bdh_gated_block_fwd, plan, _ptr(t[0]), _ptr(t[1]), _ptr(t[2]), _ptr(t[3]), options,
                  _ptr(out), *parts, _stream_ptr(dev))
    return GatedOutput(out, saved) if _lib.check(st) else None


def gated_block_vjp(grad: torch.Tensor, current: torch.Tensor, weights: GatedWeights,
                    context: Optional[torch.Tensor] = None, *, saved: Optional[GatedSaved] = None,
                    activation: str = "relu", relu_threshold: float = 0.0,
                    latent_mask: Optional[torch.Tensor] = None) -> Optional[GatedGrads]:
    """The gradients of gated_block's inputs from ``grad`` [B, T, H * N] bf16,
    the gradient of its out, with the forward's other arguments.  ``saved`` is
    what the forward kept: the gradient is then the block's at those values,
    and the projections are not computed again.  Without a context current's
    gradient has both parts.  None where the library does not support the
    input (as gated_block; a scratch that would have to grow under capture).
    Where the device has no memory for the scratch, the tokens go in groups."""
    call = _call(current, weights, context, activation, relu_threshold, latent_mask)
    if call is None or grad.dtype is not torch.bfloat16:
        return None
    dev, (B, H, T, N, D), plan, options, t = call
    if grad.shape != (B, T, H * N) or grad.device != dev:
        raise ValueError(f"grad must be {[B, T, H * N]} on the other tensors' device")
    parts, kept = (None, None, None, None), None
    if saved is not None:
        check_checkpoint(saved.up, (B, T, H, N), dev, "saved.up")
        check_checkpoint(saved.gate, (B, T, H, N), dev, "saved.gate")
        kept = [_aligned(saved.up.codes), saved.up.scales, _aligned(saved.gate.codes), saved.gate.scales]
        parts = [_ptr(p) for p in kept]
    grad = _aligned(grad)
    bf16 = torch.bfloat16
    d_current = torch.empty((B, T, D), device=dev, dtype=bf16)
    d_context = None if context is None else torch.empty((B, H, T, D), device=dev, dtype=bf16)
    d_up = torch.empty((H, D, N), device=dev, dtype=bf16)
    d_gate = torch.empty((H, D, N), device=dev, dtype=bf16)
    st = _call_on(dev, _lib.load().bdh_gated_block_vjp, plan, _ptr(t[0]), _ptr(t[1]), _ptr(t[2]), _ptr(t[3]), options,
                  _ptr(grad), *parts, _ptr(d_current), _ptr(d_context), _ptr(d_up), _ptr(d_gate), _stream_ptr(dev))
    return GatedGrads(d_current, d_context, d_up, d_gate) if _lib.check(st) else None
