"""What a row of logits says about tokens, computed on the GPU.

The reference's samplers return tokens only (tinyvllm/core/sampling.py); the greedy one is part of the
decode step (``llama.DecodeGraph``).  ``token_logprobs`` scores tokens that are already known: a prompt's
own, or the ones a step sampled.  ``verify_draft_tree`` decides which drafted tokens a step keeps.
"""

from typing import NamedTuple

import torch

from . import _lib
from .draft_tree import MAX_NODES, check_int32

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


class DraftVerdict(NamedTuple):
    path: torch.Tensor          # [B, T] int32: accepted nodes from node 0 on, -1 behind them
    counts: torch.Tensor        # [B] int32
    next_tokens: torch.Tensor   # [B] int32


def verify_draft_tree(logits, tokens, parents, tree_lens, *, temperatures=None, uniforms=None):
    """The path through each sequence's draft tree that the model's logits accept, and the token after it (no
    reference counterpart).

    logits [B, T, V] (float32, float16 or bfloat16; rows evenly spaced) follow the nodes' ``tokens`` [B, T];
    ``parents`` [B, T] and ``tree_lens`` [B] as for ``draft_tree.draft_tree_layout``, all int32.  Node 0 is
    accepted.  Greedy (no ``temperatures``, or an entry below 2^-126): the path goes on to the child whose token is the
    first maximum of the node's logits; the maximum of its last node is the next token.  Sampled, by ``temperatures`` [B]
    and ``uniforms`` [B, T] float32, the latter independent draws from [0, 1): tokens follow softmax(logits /
    temperature) exactly, child or not.  With u of the path's node it goes on to the first child at which the
    children's probabilities sum, in the order of their indexes, to more than u; without one the next token is the first at
    which the probabilities of the other tokens sum to more than (u - c) / (1 - c) of theirs, c being the children's.

    Of siblings with one token the first counts; a token outside the vocabulary is never accepted.  A logit of -inf has
    probability 0.  A node whose logits have a NaN, nothing above -inf or (sampled) +inf ends its path with -1 for the
    next token; an empty tree has count 0 and -1.
    """
    index = logits.get_device()
    if index < 0:
        raise ValueError(f"tensors must live on a HIP device (got {logits.device})")
    if logits.dim() != 3 or not 1 <= logits.shape[1] <= MAX_NODES or logits.shape[2] < 1:
        raise ValueError(f"logits must be [B, T, V] with T of 1 to {MAX_NODES}, got {list(logits.shape)}")
    b, t, v = logits.shape
    code = _lib.dtype_code(logits.dtype)
    check_int32(index, (b, t), ("tokens", tokens), ("parents", parents))
    check_int32(index, (b,), ("tree_lens", tree_lens))
    if logits.stride(2) != 1 and v > 1:
        raise ValueError("the vocabulary must be contiguous")
    try:
        rows = logits.view(-1, v) if b else logits.new_empty((0, v))
    except RuntimeError:
        raise ValueError("the rows of logits must be evenly spaced") from None
    if (temperatures is None) != (uniforms is None):
        raise ValueError("temperatures and uniforms are given together")
    if temperatures is not None:
        for x, name, shape in ((temperatures, "temperatures", (b,)), (uniforms, "uniforms", (b, t))):
            if x.dtype != torch.float32 or tuple(x.shape) != shape or not x.is_contiguous() or x.get_device() != index:
                raise ValueError(f"{name} must be contiguous float32 {list(shape)} on the logits' device")
    path, counts, following = torch.empty_like(tokens), torch.empty_like(tree_lens), torch.empty_like(tree_lens)
    need = _lib.device_size("tv_verify_draft_tree_workspace_bytes", index, b, t, v, code)
    ws = torch.empty(need, dtype=torch.uint8, device=logits.device) if need else None
    _lib.call("verify_draft_tree", index, _lib.load().tv_verify_draft_tree,
              path.data_ptr(), counts.data_ptr(), following.data_ptr(), logits.data_ptr(), tokens.data_ptr(),
              parents.data_ptr(), tree_lens.data_ptr(), temperatures.data_ptr() if temperatures is not None else None,
              uniforms.data_ptr() if uniforms is not None else None, b, t, v, rows.stride(0) if b * t > 1 else v, code,
              ws.data_ptr() if ws is not None else None, need)
    return DraftVerdict(path, counts, following)
