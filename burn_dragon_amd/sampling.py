"""The next token of every row from its logits and a given random number:
temperature, top-k, top-p and min-p on the device (bdh_sample_tokens), in
place of the reference's sampling on the host, which reads the logits back
each step (DragonModel::generate, dragon.rs:1749-1808).

Nothing waits for the device, so a generated token feeds the next forward
without a host round trip, and a step can be captured into a graph.  The
random numbers are an argument: the same numbers give the same tokens,
whatever the batch around a row.
"""
from __future__ import annotations

import ctypes
import math
from typing import NamedTuple, Optional, Union

import torch

from . import _lib
from .recurrent import _call_on, _dtype_code, _ptr, _stream_ptr, _supported

PerRow = Union[float, torch.Tensor]


class SampleOutput(NamedTuple):
    tokens: torch.Tensor                # [rows] int32
    logprob: Optional[torch.Tensor]     # [rows] f32 when requested


def _per_row(value, rows: int, dtype: torch.dtype, device, name: str):
    """(scalar, tensor or None): one setting for all rows, or one a row."""
    if not isinstance(value, torch.Tensor):
        return value, None
    if value.dtype != dtype or value.shape != (rows,) or value.device != device:
        raise ValueError(f"{name} must be a number or a {dtype} tensor of [{rows}] on the logits' device")
    return 0, value.contiguous()


def _options(rows: int, vocab: int, dev: torch.device, uniform: torch.Tensor, temperature: PerRow,
             top_k: Union[int, torch.Tensor], top_p: PerRow, min_p: PerRow):
    """The library's options and the tensors that they point to; raises
    ValueError where the random numbers or a setting a row do not fit."""
    if uniform.dtype != torch.float32 or uniform.shape != (rows,) or uniform.device != dev:
        raise ValueError(f"uniform must be a f32 tensor of [{rows}] on the logits' device")
    temp, temp_rows = _per_row(temperature, rows, torch.float32, dev, "temperature")
    p, p_rows = _per_row(top_p, rows, torch.float32, dev, "top_p")
    mp, mp_rows = _per_row(min_p, rows, torch.float32, dev, "min_p")
    k, k_rows = _per_row(top_k, rows, torch.int32, dev, "top_k")
    if k_rows is None:
        k = min(max(int(k), -1), vocab)  # (an int32 to the library)
    opts = _lib.BdhSampleOptions(float(temp), float(p), float(mp), k, _ptr(temp_rows), _ptr(p_rows),
                                 _ptr(mp_rows), _ptr(k_rows))
    return opts, (temp_rows, p_rows, mp_rows, k_rows)


def check_settings(rows: int, vocab: int, uniform: torch.Tensor, temperature: PerRow,
                   top_k: Union[int, torch.Tensor], top_p: PerRow, min_p: PerRow) -> bool:
    """What sample_tokens would say to [rows, vocab] logits on uniform's device
    with these arguments, before there are any: False where it returns None
    for their size, its errors where it raises."""
    o, _ = _options(rows, vocab, uniform.device, uniform, temperature, top_k, top_p, min_p)
    if not 0 < rows < 1 << 22 or not 0 < vocab <= 1 << 20:
        return False
    if not o.temperature_rows and not 0.0 <= o.temperature < math.inf:
        raise _lib.BdhError("temperature must be finite and not negative")
    if not o.top_p_rows and not 0.0 <= o.top_p <= 1.0:
        raise _lib.BdhError("top_p must lie in [0, 1]")
    if not o.min_p_rows and not 0.0 <= o.min_p <= 1.0:
        raise _lib.BdhError("min_p must lie in [0, 1]")
    if not o.top_k_rows and o.top_k < 0:
        raise _lib.BdhError("top_k must not be negative")
    return True


def sample_tokens(logits: torch.Tensor, uniform: torch.Tensor, *, temperature: PerRow = 1.0,
                  top_k: Union[int, torch.Tensor] = 0, top_p: PerRow = 1.0, min_p: PerRow = 0.0,
                  want_logprob: bool = False, out: Optional[torch.Tensor] = None
                  ) -> Optional[SampleOutput]:
    """logits [rows, V] f32 or bf16 on the device, V contiguous (a slice such
    as ``logits[:, -1]`` or an expanded row is read in place), uniform [rows]
    f32 in [0, 1).  Per row, with w = exp((x - max x) / temperature):
    ``top_k`` keeps the first k in descending order (ties by index; 0: all),
    ``top_p`` of these each before which the kept w sum to less than top_p
    of their sum, ``min_p`` of these each with w >= min_p; the token is the
    first index at which the running sum of kept w exceeds uniform times
    their sum.  temperature 0 is the argmax (first index).  NaN logits count
    as -inf; a row without a logit above -inf gives -1.  Each setting is a
    number or a tensor of [rows] (f32; top_k int32).  ``logprob`` is the log
    of the token's share of the kept w.  Returns None where the library does
    not support the input (no supported device, another dtype, an empty
    dimension, V above 2^20, a scratch too small for a single row under
    capture)."""
    dev = logits.device
    if not _supported(dev) or logits.dim() != 2:
        return None
    rows, vocab = logits.shape
    code = _dtype_code(logits)
    if code is None or rows == 0 or vocab == 0:
        return None
    row_stride, stride = logits.stride()
    if vocab > 1 and stride != 1:
        logits, row_stride = logits.contiguous(), vocab
    opts, rows_of = _options(rows, vocab, dev, uniform, temperature, top_k, top_p, min_p)
    uniform = uniform.contiguous()
    if out is None:
        tokens = torch.empty(rows, device=dev, dtype=torch.int32)
    elif (out.dtype != torch.int32 or out.shape != (rows,) or out.device != dev
          or not out.is_contiguous()):
        raise ValueError(f"out must be a contiguous int32 tensor of [{rows}] on the logits' device")
    else:
        tokens = out
    logprob = torch.empty(rows, device=dev, dtype=torch.float32) if want_logprob else None
    # (rows_of holds what opts points to until the launch is enqueued.)
    st = _call_on(dev, _lib.load().bdh_sample_tokens, _ptr(logits), code, rows, vocab,
                  row_stride if rows > 1 else 0, _ptr(uniform), ctypes.byref(opts), _ptr(tokens),
                  _ptr(logprob), _stream_ptr(dev))
    if not _lib.check(st):
        return None
    return SampleOutput(tokens, logprob)
