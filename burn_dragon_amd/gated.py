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


def _plan(current, weights, context, activation, relu_threshold, latent_mask):
    """(plan, options, tensors) of a call; None where the library does not
    support it, ValueError where the arguments do not fit together."""
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}")
    up, gate = weights
    dev = current.device
    if not _supported(dev) or current.dim() != 3 or up.dim() != 3 or gate.dim() != 3:
        return None
    tensors = [t for t in (current, up, gate, context) if t is not None]
    if any(t.dtype != torch.bfloat16 for t in tensors):
        return None
    B, T, D = current.shape
    H, _, N = up.shape
    if min(B, T, D, H, N) == 0:
        return None
    if tuple(up.shape) != (H, D, N) or tuple(gate.shape) != (H, D, N):
        raise ValueError("up and gate must be [H, D, N] with current's D")
    if context is not None and tuple(context.shape) != (B, H, T, D):
        raise ValueError(f"context must be {[B, H, T, D]}")
    mask = None
    if latent_mask is not None:
        mask = latent_mask.reshape(-1)
        if mask.numel() != N or mask.dtype != torch.float32:
            raise ValueError(f"latent_mask must hold {N} f32 values")
        tensors.append(mask)
    if any(t.device != dev for t in tensors):
        raise ValueError("the tensors must be on one device")
    if activation != "relu" and (relu_threshold != 0.0 or mask is not None):
        raise ValueError('relu_threshold and latent_mask go with activation="relu"')
    current, up, gate, context, mask = (_aligned(t) for t in (current, up, gate, context, mask))
    plan = _lib.BdhLayerPlan(B, H, T, N, D)
    options = _lib.BdhGatedOptions(ACTIVATIONS[activation], float(relu_threshold), _ptr(mask))
    return plan, options, (current, context, up, gate, mask)


def _aligned(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """Contiguous, from a 16-byte boundary on."""
    if t is None:
        return None
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
    call = _plan(current, weights, context, activation, relu_threshold, latent_mask)
    if call is None:
        return None
    plan, options, (current, context, up, gate, _mask) = call
    B, H, T, N = plan.batch, plan.heads, plan.time, plan.latent
    dev = current.device
    if N % 8 or plan.embd % 8:
        return None
    out = torch.empty((B, T, H * N), device=dev, dtype=torch.bfloat16)
    saved, parts = None, (None,) * 4
    if save:
        saved = GatedSaved(new_checkpoint((B, T, H, N), dev), new_checkpoint((B, T, H, N), dev))
        parts = (*saved.up, *saved.gate)
    st = _call_on(dev, _lib.load().bdh_gated_block_fwd, ctypes.byref(plan), _ptr(current), _ptr(context), _ptr(up),
                  _ptr(gate), ctypes.byref(options), _ptr(out), *map(_ptr, parts), _stream_ptr(dev))
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
    input (as gated_block; a scratch that would have to grow under capture)."""
    call = _plan(current, weights, context, activation, relu_threshold, latent_mask)
    if call is None:
        return None
    plan, options, (current, context, up, gate, _mask) = call
    B, H, T, N, D = plan.batch, plan.heads, plan.time, plan.latent, plan.embd
    dev = current.device
    if grad.dtype != torch.bfloat16 or N % 8 or D % 8:
        return None
    if tuple(grad.shape) != (B, T, H * N) or grad.device != dev:
        raise ValueError(f"grad must be {[B, T, H * N]} on the other tensors' device")
    parts = (None,) * 4
    if saved is not None:
        for c, name in zip(saved, ("saved.up", "saved.gate")):
            check_checkpoint(c, (B, T, H, N), dev, name)
        parts = tuple(_aligned(t) for t in (*saved.up, *saved.gate))
    grad = _aligned(grad)
    bf16 = lambda *shape: torch.empty(shape, device=dev, dtype=torch.bfloat16)  # noqa: E731
    out = GatedGrads(bf16(B, T, D), None if context is None else bf16(B, H, T, D), bf16(H, D, N), bf16(H, D, N))
    st = _call_on(dev, _lib.load().bdh_gated_block_vjp, ctypes.byref(plan), _ptr(current), _ptr(context), _ptr(up),
                  _ptr(gate), ctypes.byref(options), _ptr(grad), *map(_ptr, parts), _ptr(out.current),
                  _ptr(out.context), _ptr(out.up), _ptr(out.gate), _stream_ptr(dev))
    return out if _lib.check(st) else None
