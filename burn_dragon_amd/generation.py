"""Generation of a batch of sequences on the device: the prompt, then one
forward and one draw a token (DragonModel::generate,
crates/burn_dragon_core/src/model/dragon.rs:1749-1808, generation.rs:458).
The reference reads each step's logits back to the host to sample; here the
drawn token feeds the next forward on the device.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Union

import torch

from .adapters import AdapterSet
from .model import BdhModelState, BdhModelWeights, model_forward_logits, new_model_state
from .recurrent import DEFAULT_ROPE_THETA
from .sampling import PerRow, check_settings, sample_tokens


class GenerateOutput(NamedTuple):
    tokens: torch.Tensor                # [B, steps] int32
    logprob: Optional[torch.Tensor]     # [B, steps] f32 when requested
    state: BdhModelState


def generate_tokens(prompt: torch.Tensor, weights: BdhModelWeights, uniform: torch.Tensor, *,
                    state: Optional[BdhModelState] = None, temperature: PerRow = 1.0,
                    top_k: Union[int, torch.Tensor] = 0, top_p: PerRow = 1.0, min_p: PerRow = 0.0,
                    theta: float = DEFAULT_ROPE_THETA, relu_threshold: float = 0.0,
                    latent_mask: Optional[torch.Tensor] = None,
                    adapters: Optional[AdapterSet] = None, adapter_ids: Optional[torch.Tensor] = None,
                    want_logprob: bool = False) -> Optional[GenerateOutput]:
    """prompt [B, T] int32 on the device, continued by ``uniform.shape[0]``
    tokens a sequence: uniform [steps, B] f32 in [0, 1) are the draws' random
    numbers.  ``state`` (default: a new one) is continued in place and holds
    the prompt and all drawn tokens but the last, which the next call's
    prompt begins with.  The cuts are sample_tokens', the other options
    model_forward_logits'.  Settings, random numbers and adapters that do not
    fit are refused with those calls' errors before the prompt runs.  Returns
    None where the library does not support a call: for the arguments' types
    and sizes, before the prompt runs; for want of scratch under capture, with
    what ran in the state."""
    if weights is None or prompt.dim() != 2 or not prompt.is_cuda:
        return None
    B = prompt.shape[0]
    if uniform.dim() != 2 or uniform.shape[0] == 0 or uniform.shape[1] != B:
        raise ValueError(f"uniform must be [steps, {B}]")
    steps = uniform.shape[0]
    if uniform.device != prompt.device:
        raise ValueError("uniform must be on the prompt's device")
    if not check_settings(B, weights.vocab, uniform[0], temperature, top_k, top_p, min_p):
        return None
    if state is None:
        state = new_model_state(weights, B, prompt.device)
    tokens = torch.empty((steps, B), device=prompt.device, dtype=torch.int32)
    logprob = torch.empty((steps, B), device=prompt.device, dtype=torch.float32) if want_logprob else None
    current = prompt
    for i in range(steps):
        logits = model_forward_logits(current, weights, theta=theta, state=state,
                                      relu_threshold=relu_threshold, latent_mask=latent_mask,
                                      adapters=adapters, adapter_ids=adapter_ids)
        if logits is None:
            return None
        drawn = sample_tokens(logits[:, -1], uniform[i], temperature=temperature, top_k=top_k,
                              top_p=top_p, min_p=min_p, want_logprob=want_logprob, out=tokens[i])
        if drawn is None:
            return None
        if logprob is not None:
            logprob[i] = drawn.logprob
        current = tokens[i].unsqueeze(1)
    return GenerateOutput(tokens.t(), logprob.t() if logprob is not None else None, state)
