"""Streams' recurrent states moved between the slots of a batch.

A serving batch is a ``BdhModelState``: one rho [B, H, N, D] f32 a layer,
slot b holding stream b.  Requests come and go between steps: a prompt is
run once and its state forked into the slots of its samples, a search keeps
some candidates and doubles others, a batch closes up when requests end, a
slot is cleared for a new sequence.  Each call moves whole slots of every
layer in one launch (bdh_state_copy_streams), in place, as one assignment:
every source is read before any slot is written, whatever the pattern.

All calls take a BdhModelState, or a list of the layers' rho (a layer may be
None).  The slots are host integers: they are what the server's scheduler
decides.  A state has one position for all its streams, so streams may be
copied between states of the same position only; a cleared slot begins a new
sequence at whatever position its state is, since scores depend on
differences of positions.
"""
from __future__ import annotations

import ctypes
from typing import List, Optional, Sequence, Union

import torch

from . import _lib
from .model import BdhModelState
from .recurrent import _call_on, _stream_ptr, supports_backend

StreamStates = Union[BdhModelState, Sequence[Optional[torch.Tensor]]]


def _layers(state: StreamStates) -> List[Optional[torch.Tensor]]:
    return list(state.rho if isinstance(state, BdhModelState) else state)


class _Slots:
    """The layers of a state as the library takes them."""

    def __init__(self, rho):
        n = len(rho)
        self.descs = (_lib.BdhLayerStateDesc * n)()
        self.ptrs = (ctypes.c_void_p * n)()
        self.batch, self.device = 0, None
        for i, r in enumerate(rho):
            if r is None:
                continue
            if r.dtype != torch.float32 or not r.is_cuda or r.dim() != 4 or not r.is_contiguous():
                raise ValueError("rho must be a contiguous f32 [B,H,N,D] device tensor")
            if self.device is None:
                self.batch, self.device = r.shape[0], r.device
            elif r.shape[0] != self.batch or r.device != self.device:
                raise ValueError("the layers of a state have different batches or devices")
            d = self.descs[i]
            d.batch, d.heads, d.latent, d.embd = r.shape
            self.ptrs[i] = r.data_ptr()


def _check_slots(slots: List[int], batch: int, what: str, least: int = 0):
    if slots and (min(slots) < least or max(slots) >= batch):
        raise ValueError(f"{what} must lie in [{least}, {batch})")


def copy_streams(state: StreamStates, dst: Sequence[int], src: Sequence[int], *,
                 source: Optional[StreamStates] = None) -> Optional[StreamStates]:
    """Slot dst[i] of ``state`` takes the value of slot src[i] of ``source``
    (default: of ``state`` itself), or zeros where src[i] is -1, in every
    layer; the dst are distinct.  In place; returns ``state``, or None on an
    unsupported device.  Raises ValueError on slots outside their batch, a
    slot written twice, layers that do not match, or two states at different
    positions."""
    if not supports_backend():
        return None
    rho, dst, src = _layers(state), [int(d) for d in dst], [int(s) for s in src]
    slots = _Slots(rho)
    other, batch = None, slots.batch
    if source is not None and source is not state:
        from_ = _layers(source)
        if len(from_) != len(rho):
            raise ValueError("the states have different numbers of layers")
        if any(a is not b for a, b in zip(rho, from_)):
            other = _Slots(from_)
            batch = other.batch
            if any((a is None) != (b is None) or (a is not None and a.shape[1:] != b.shape[1:])
                   for a, b in zip(rho, from_)) or other.device != slots.device:
                raise ValueError("the states' layers have different shapes or devices")
            if (isinstance(state, BdhModelState) and isinstance(source, BdhModelState)
                    and state.position != source.position and any(s >= 0 for s in src)):
                raise ValueError(f"the states are at positions {state.position} and {source.position}")
    if len(dst) != len(src):
        raise ValueError("dst and src have different lengths")
    _check_slots(dst, slots.batch, "dst")
    _check_slots(src, batch, "src", -1)
    n = len(dst)
    if len(set(dst)) != n:
        raise ValueError("a slot is written twice")
    dev = slots.device
    if dev is None or n == 0:
        return state
    st = _call_on(dev, _lib.load().bdh_state_copy_streams, len(rho), slots.descs, slots.ptrs,
                  other.descs if other else None, other.ptrs if other else None, n,
                  (ctypes.c_int32 * n)(*dst), (ctypes.c_int32 * n)(*src), _stream_ptr(dev))
    return state if _lib.check(st) else None


def free_streams(state: StreamStates, streams: Sequence[int]) -> Optional[StreamStates]:
    """Clears slots: each then begins a new sequence."""
    streams = list(streams)
    return copy_streams(state, streams, [-1] * len(streams))


def compact_streams(state: StreamStates, keep: Sequence[int]) -> Optional[StreamStates]:
    """Slot i takes the stream keep[i], and the batch ends after len(keep)
    streams: returns a state (or list) of the same memory's first slots, at
    the same position.  ``keep`` in any order, a stream more than once if it
    is to go on as several (at most B entries).  None on an unsupported
    device."""
    keep = list(keep)
    if len(keep) == 0:
        raise ValueError("keep names no stream")
    if copy_streams(state, range(len(keep)), keep) is None:
        return None
    rho = [r if r is None else r[:len(keep)] for r in _layers(state)]
    if not isinstance(state, BdhModelState):
        return rho
    out = BdhModelState.__new__(BdhModelState)
    out.rho = rho
    out.position = state.position
    return out
