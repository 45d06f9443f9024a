"""What a row of logits says about tokens, computed on the GPU.

The reference's samplers return tokens only (tinyvllm/core/sampling.py); the greedy one is part of the
decode step (``llama.DecodeGraph``).  ``token_logprobs`` scores tokens that are already known: a prompt's
own, or the ones a step sampled.
"""

from typing import NamedTuple

import torch

from . import _lib

_lib.load()


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor       # [...] float32
    entropy: torch.Tensor        # [...] float32, natural logarithm
    top_ids: torch.Tensor        # [..., top_k] int32
    top_logprobs: torch.Tensor   # [..., top_k] float32


def token_logprobs(logits, tokens, top_k=0):
    """Log-probabilities of ``tokens`` [...] (int32) under ``logits`` [..., V] (float32, float16 or
    bfloat16), the rows' entropy, and the ``top_k`` (0 to 64) most likely tokens of each row with their
    log-probabilities, most likely first and equal logits by lowest id.

    Rows may be strided (``logits[:, :-1]`` of a prompt pass against ``tokens[1:]``); the vocabulary must be
    contiguous.  A logit of -inf has probability 0; a token outside the vocabulary (padding) gives NaN; a
    row with a NaN, with +inf or without a finite logit gives NaN, and its ``top_ids`` rank NaN first.
    """
    index = logits.get_device()
    if index < 0 or tokens.get_device() != index:
        raise ValueError(f"logits and tokens must be on one HIP device (got {logits.device}, {tokens.device})")
    shape = logits.shape[:-1]
    if logits.dim() < 1 or tokens.shape != shape:
        raise ValueError(f"tokens must be {tuple(shape)}, got {tuple(tokens.shape)}")
    if tokens.dtype != torch.int32:
        raise ValueError("tokens must be int32")
    v = logits.shape[-1]
    top_k = int(top_k)
    if v < 1 or not 0 <= top_k <= min(64, v):
        raise ValueError(f"top_k must be between 0 and min(64, {v}), got {top_k}")
    code = _lib.dtype_code(logits.dtype)
    if logits.stride(-1) != 1 and v > 1:
        raise ValueError("the vocabulary must be contiguous")
    rows = logits
    if logits.dim() != 2:
        try:
            rows = logits.view(-1, v)
        except RuntimeError:
            raise ValueError("the rows of logits must be evenly spaced") from None
    m = rows.shape[0]
    dev = logits.device
    flat = tokens.reshape(-1).contiguous()
    lp = torch.empty(shape, dtype=torch.float32, device=dev)
    entropy = torch.empty_like(lp)
    ids = torch.empty((*shape, top_k), dtype=torch.int32, device=dev)
    top = torch.empty_like(ids, dtype=torch.float32)
    need = _lib.device_size("tv_token_logprobs_workspace_bytes", index, m, v, top_k, code)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    _lib.call("token_logprobs", index, _lib.load().tv_token_logprobs,
              lp.data_ptr(), entropy.data_ptr(), ids.data_ptr(), top.data_ptr(), rows.data_ptr(), flat.data_ptr(), m,
              v, rows.stride(0) if m > 1 else v, top_k, code, ws.data_ptr() if ws is not None else None, need)
    return TokenLogprobs(lp, entropy, ids, top)
