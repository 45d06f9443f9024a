"""Trees of drafted tokens: what each node sees, where it stands and where its K/V go.

The reference decodes one token a step and has no counterpart.  A verified step over a tree, all on the
device (and so in a captured graph):

    layout = draft_tree_layout(parents, tree_lens, context_lens, block_tables, block_size, num_blocks)
    for every layer:                     # q, k, v of all nodes from the layer's projection
        q = kv_cache.write_rope_slots(layer, layout.slots, layout.positions, rope, q, k, v)
        out = paged_tree_attention(q.view(B, T, Hq, D), k_cache, v_cache, block_tables, context_lens,
                                   tree_lens, layout.mask, Hq, Hkv, D, block_size)
    verdict = verify_draft_tree(logits, tokens, parents, tree_lens)
    kv_cache.keep_draft_path(verdict.path, verdict.counts, context_lens, block_tables)
    context_lens += verdict.counts       # verdict.next_tokens are the next trees' node 0

``kv_cache.KVCache.write_rope_slots`` / ``keep_draft_path``, ``attention.paged_tree_attention`` and
``sampling.verify_draft_tree`` are the other parts.  The block tables must list the blocks of positions
up to context + nodes - 1 before the step.
"""

from typing import NamedTuple

import torch

from . import _lib

_lib.load()

MAX_NODES = 256


class DraftTreeLayout(NamedTuple):
    mask: torch.Tensor        # [B, T, ceil(T / 64)] int64
    positions: torch.Tensor   # [B, T] int32
    slots: torch.Tensor       # [B, T] int32


def check_int32(index, shape, *named):
    """Raises ValueError unless each (name, tensor) is dense int32 of ``shape`` on device ``index``."""
    for name, x in named:
        if x.dtype is not torch.int32 or x.shape != shape or not x.is_contiguous():
            raise ValueError(f"{name} must be contiguous int32 {list(shape)}, got {x.dtype} {list(x.shape)}")
        if x.get_device() != index:
            raise ValueError("all tensors must be on one HIP device")


def check_block_tables(index, b, block_tables):
    """Raises ValueError unless block_tables is dense int32 [B, columns] on device ``index``; the columns."""
    shape = block_tables.shape
    if block_tables.dtype is not torch.int32 or len(shape) != 2 or shape[0] != b or shape[1] < 1 or \
            not block_tables.is_contiguous():
        raise ValueError(f"block_tables must be contiguous int32 [{b}, columns], got {block_tables.dtype} {list(shape)}")
    if block_tables.get_device() != index:
        raise ValueError("all tensors must be on one HIP device")
    return shape[1]


def draft_tree_layout(parents, tree_lens, context_lens, block_tables, block_size, num_blocks):
    """Mask, positions and cache slots of every node, from ``parents`` [B, T] int32 (T at most 256).

    A parent is a lower index of the same tree; anything else stands for none (node 0 has none).
    ``tree_lens`` [B] nodes of a tree are in use, ``context_lens`` [B] tokens of the sequence cached before
    it.  ``mask`` has bit t % 64 of word t // 64 set for a node and all its ancestors; ``positions`` are
    context + depth; ``slots`` the places of cache positions context + i by ``block_tables``, -1
    where the table does not reach them or names a block outside 0 .. num_blocks - 1.  Nodes at
    ``tree_lens`` and beyond have mask 0, position 0 and slot -1.
    """
    index = parents.get_device()
    if index < 0:
        raise ValueError(f"tensors must live on a HIP device (got {parents.device})")
    shape = parents.shape
    if len(shape) != 2 or not 1 <= shape[1] <= MAX_NODES:
        raise ValueError(f"parents must be [B, T] with T of 1 to {MAX_NODES}, got {list(shape)}")
    b, t = shape
    check_int32(index, shape, ("parents", parents))
    check_int32(index, shape[:1], ("tree_lens", tree_lens), ("context_lens", context_lens))
    columns = check_block_tables(index, b, block_tables)
    mask = parents.new_empty((b, t, (t + 63) // 64), dtype=torch.int64)
    positions, slots = torch.empty_like(parents), torch.empty_like(parents)
    _lib.call("draft_tree_layout", index, _lib.load().tv_draft_tree_layout,
              mask.data_ptr(), positions.data_ptr(), slots.data_ptr(), parents.data_ptr(), tree_lens.data_ptr(),
              context_lens.data_ptr(), block_tables.data_ptr(), b, t, columns, int(block_size), int(num_blocks))
    return DraftTreeLayout(mask, positions, slots)
