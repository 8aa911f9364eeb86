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
from .recurrent import _on_current_device, _stream_ptr, supports_backend

StreamStates = Union[BdhModelState, Sequence[Optional[torch.Tensor]]]


def _layers(state: StreamStates) -> List[Optional[torch.Tensor]]:
    rho = list(state.rho if isinstance(state, BdhModelState) else state)
    for r in rho:
        if r is not None and (r.dtype != torch.float32 or not r.is_cuda or r.dim() != 4
                              or not r.is_contiguous()):
            raise ValueError("rho must be a contiguous f32 [B,H,N,D] device tensor")
    if len({r.device for r in rho if r is not None}) > 1:
        raise ValueError("the layers' rho are on different devices")
    return rho


def _arrays(rho):
    n = len(rho)
    descs = (_lib.BdhLayerStateDesc * max(n, 1))()
    ptrs = (ctypes.c_void_p * max(n, 1))()
    for i, r in enumerate(rho):
        if r is not None:
            descs[i].batch, descs[i].heads, descs[i].latent, descs[i].embd = r.shape
            ptrs[i] = r.data_ptr()
    return descs, ptrs


def _slots(slots, batch: int, what: str, least: int = 0) -> List[int]:
    out = [int(s) for s in slots]
    if any(s < least or s >= batch for s in out):
        raise ValueError(f"{what} must lie in [{least}, {batch})")
    return out


def _batch(rho) -> int:
    sizes = {r.shape[0] for r in rho if r is not None}
    if len(sizes) > 1:
        raise ValueError("the layers of a state have different batches")
    return sizes.pop() if sizes else 0


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
    rho = _layers(state)
    from_ = None if source is None or source is state else _layers(source)
    if from_ is not None and all(a is b for a, b in zip(rho, from_)) and len(rho) == len(from_):
        from_ = None
    if from_ is not None:
        if len(from_) != len(rho):
            raise ValueError("the states have different numbers of layers")
        if any((a is None) != (b is None) or (a is not None and (a.shape[1:] != b.shape[1:]
               or a.device != b.device)) for a, b in zip(rho, from_)):
            raise ValueError("the states' layers have different shapes or devices")
        if (isinstance(state, BdhModelState) and isinstance(source, BdhModelState)
                and any(s >= 0 for s in src) and state.position != source.position):
            raise ValueError(f"the states are at positions {state.position} and {source.position}")
    batch = _batch(rho)
    dst = _slots(dst, batch, "dst")
    src = _slots(src, batch if from_ is None else _batch(from_), "src", -1)
    if len(dst) != len(src):
        raise ValueError("dst and src have different lengths")
    if len(set(dst)) != len(dst):
        raise ValueError("a slot is written twice")
    dev = next((r.device for r in rho if r is not None), None)
    if dev is None or not dst:
        return state
    descs, ptrs = _arrays(rho)
    src_descs, src_ptrs = _arrays(from_) if from_ is not None else (None, None)
    n = len(dst)
    with _on_current_device(dev):
        st = _lib.load().bdh_state_copy_streams(len(rho), descs, ptrs, src_descs, src_ptrs, n,
                                                (ctypes.c_int32 * n)(*dst), (ctypes.c_int32 * n)(*src),
                                                _stream_ptr(dev))
    if not _lib.check(st):
        return None
    return state


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
    if len(keep) > _batch(_layers(state)):
        raise ValueError("keep has more streams than the state has slots")
    if copy_streams(state, range(len(keep)), keep) is None:
        return None
    rho = [r if r is None else r[:len(keep)] for r in _layers(state)]
    if not isinstance(state, BdhModelState):
        return rho
    out = BdhModelState.__new__(BdhModelState)
    out.rho = rho
    out.position = state.position
    return out
