"""Token generation over a ``VeraceV1Model`` (the loop of the reference's generator,
verace_v1/serving/hyper_generate.py:33-80, for a batch and with the usual controls): the prompt
once, then one token a step through ``layer_states``, its logits through ``process_logits`` and
``sample_logits``.  With ``quantize_model_int4(model)`` the projections and the LM head of
every step are products with 4-bit weights.
"""
from typing import Callable, Optional, Tuple, Union

import torch

from .sampling import PerRow, process_logits, sample_logits


@torch.no_grad()
def generate(model: torch.nn.Module, input_ids: torch.Tensor, max_new_tokens: int, *, temperature: PerRow = 0.0,
             top_k: Union[int, torch.Tensor] = 0, top_p: PerRow = 1.0, min_p: PerRow = 0.0,
             repetition_penalty: PerRow = 1.0, presence_penalty: PerRow = 0.0, frequency_penalty: PerRow = 0.0,
             bias_ids: Optional[torch.Tensor] = None, bias_values: Optional[torch.Tensor] = None,
             allowed: Union[None, torch.Tensor, Callable[[torch.Tensor], Optional[torch.Tensor]]] = None,
             eos_token_id: Optional[int] = None, generator: Optional[torch.Generator] = None
             ) -> Tuple[torch.Tensor, torch.Tensor]:
    """input_ids [b, s] -> (tokens [b, s + n], log-probabilities [b, n]) with n at most
    ``max_new_tokens``.  The controls are those of ``process_logits`` (the prompt counts for the
    repetition penalty, not for the other two) and ``sample_logits``; ``allowed`` may be a
    function of the tokens so far, [b, s + i], that returns the step's mask.  A row ends at
    ``eos_token_id`` or where the mask or the biases (of -inf) leave it nothing: its tokens from there on
    are ``eos_token_id`` (-1 without one) with log-probability 0, and the loop ends once every row has (a
    host read a step, only with an eos or a mask)."""
    if max_new_tokens < 0:
        raise ValueError(f"max_new_tokens {max_new_tokens}: expected at least 0")
    assert input_ids.is_cuda, "This kernel requires CUDA tensors"
    assert input_ids.dim() == 2 and input_ids.shape[1] > 0, "input_ids must be [b, s] with at least one token"
    b, s = input_ids.shape
    dev = input_ids.device
    end = -1 if eos_token_id is None else int(eos_token_id)
    tokens = torch.full((b, s + max_new_tokens), end, dtype=torch.int64, device=dev)
    tokens[:, :s] = input_ids
    logprobs = torch.zeros(b, max_new_tokens, device=dev)
    prompt = torch.full((b,), s, dtype=torch.int32, device=dev)
    done = torch.zeros(b, dtype=torch.bool, device=dev)
    ends = eos_token_id is not None or allowed is not None
    sampled = isinstance(temperature, torch.Tensor) or temperature > 0
    ids, states, n = input_ids, None, 0
    for i in range(max_new_tokens):
        logits, _, states = model(ids, layer_states=states, return_layer_states=True)
        row = logits[:, -1]
        so_far = tokens[:, :s + i]
        mask = allowed(so_far) if callable(allowed) else allowed
        row = process_logits(row, so_far, None, prompt, repetition_penalty=repetition_penalty,
                             presence_penalty=presence_penalty, frequency_penalty=frequency_penalty,
                             bias_ids=bias_ids, bias_values=bias_values, allowed=mask, out_dtype=torch.float32)
        noise = torch.empty_like(row).exponential_(generator=generator) if sampled else None
        token, lp = sample_logits(row, noise, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
        if ends or bias_ids is not None:
            done = done | (token < 0)
            token = torch.where(done, end, token)
            lp = torch.where(done, 0.0, lp)
            done = done | (token == end)
        tokens[:, s + i] = token
        logprobs[:, i] = lp
        n = i + 1
        if ends and bool(done.all()):
            break
        ids = token.clamp_min(0)[:, None]
    return tokens[:, :s + n], logprobs[:, :n]
