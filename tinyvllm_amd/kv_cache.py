"""Paged KV cache with the reference's interface (tinyvllm/core/kv_cache.py:13-61).

Storage per layer: one K and one V tensor [num_blocks, block_size, n_kv_heads,
head_dim], zero-initialised, dense, on a HIP device.  Element (blk, t, h, d)
sits at ((blk*bs + t)*Hkv + h)*D + d, the layout paged_decode_attention reads.
All writes and reads go through libtvattn.so kernels.
"""

import ctypes

import numpy as np
import torch

from . import _lib
from .draft_tree import check_block_tables, check_int32

_lib.load()

_DTYPES = {
    "float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16,
    "half": torch.float16, "float": torch.float32,
}


def as_torch_dtype(dtype):
    """Accept a torch dtype, a numpy dtype or a name ('float16', ...)."""
    if isinstance(dtype, torch.dtype):
        return dtype
    if isinstance(dtype, str):
        return _DTYPES[dtype]
    name = getattr(dtype, "name", None) or np.dtype(dtype).name
    return _DTYPES[name]


class KVCache:
    """Block-based KV cache.  Shape per layer: [num_blocks, block_size, n_kv_heads, head_dim]."""

    def __init__(self, num_layers, num_blocks, block_size, n_kv_heads, head_dim, dtype, device="cuda"):
        self.num_layers = num_layers
        self.num_blocks = num_blocks
        self.block_size = block_size
        self.n_kv_heads = n_kv_heads
        self.head_dim = head_dim
        self.dtype = as_torch_dtype(dtype)
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise ValueError("KVCache storage must be on a HIP device")
        shape = (num_blocks, block_size, n_kv_heads, head_dim)
        self.k_cache = [torch.zeros(shape, dtype=self.dtype, device=self.device) for _ in range(num_layers)]
        self.v_cache = [torch.zeros(shape, dtype=self.dtype, device=self.device) for _ in range(num_layers)]

    # -- helpers -------------------------------------------------------------
    def _rows(self, x, name):
        """View ``x`` as [T, Hkv*D] rows with a token stride; validates layout."""
        if x.dim() == 2:          # a single token [Hkv, D]
            x = x.unsqueeze(0)
        if x.dim() != 3 or tuple(x.shape[1:]) != (self.n_kv_heads, self.head_dim):
            raise ValueError(f"{name} must be [T, {self.n_kv_heads}, {self.head_dim}], got {tuple(x.shape)}")
        if x.dtype != self.dtype:
            raise ValueError(f"{name} dtype {x.dtype} differs from cache dtype {self.dtype}")
        if x.device != self.k_cache[0].device:
            raise ValueError(f"{name} must be on {self.k_cache[0].device}")
        stride = x.stride()         # a dimension of size 1 may have any
        if x.shape[0] and ((stride[2] != 1 and self.head_dim > 1) or
                           (stride[1] != self.head_dim and self.n_kv_heads > 1)):
            raise ValueError(f"{name}: heads and head_dim must be contiguous")
        return x, stride[0] if x.shape[0] > 1 else self.n_kv_heads * self.head_dim

    # -- reference API -------------------------------------------------------
    def write_kv(self, layer_idx, block_id, start_offset, k, v):
        """Write k/v [T, Hkv, D] to [block_id, start_offset:start_offset+T] (kv_cache.py:34-38)."""
        k, ks = self._rows(k, "k")
        v, vs = self._rows(v, "v")
        if k.shape[0] != v.shape[0]:
            raise ValueError("k and v must hold the same number of tokens")
        lib = _lib.load()
        rc = lib.tv_write_kv(
            self.k_cache[layer_idx].data_ptr(), self.v_cache[layer_idx].data_ptr(),
            k.data_ptr(), v.data_ptr(), int(block_id), int(start_offset), k.shape[0],
            self.n_kv_heads, self.head_dim, self.block_size, self.num_blocks, ks, vs,
            _lib.dtype_code(self.dtype), _lib.stream_ptr(self.device))
        _lib.check(rc, "KVCache.write_kv")

    def read_kv_blocks(self, layer_idx, block_ids, context_len):
        """Return (k, v) [context_len, Hkv, D] gathered from ``block_ids`` (kv_cache.py:40-55)."""
        shape = (0, self.n_kv_heads, self.head_dim)
        if not block_ids:
            return (torch.zeros(shape, dtype=self.dtype, device=self.device),
                    torch.zeros(shape, dtype=self.dtype, device=self.device))
        n = min(int(context_len), len(block_ids) * self.block_size)
        if n < 0:
            raise ValueError("context_len must be >= 0")
        k_out = torch.empty((n, self.n_kv_heads, self.head_dim), dtype=self.dtype, device=self.device)
        v_out = torch.empty_like(k_out)
        if n == 0:
            return k_out, v_out
        ids = torch.tensor(list(block_ids), dtype=torch.int32).to(self.device)
        lib = _lib.load()
        rc = lib.tv_read_kv_blocks(
            k_out.data_ptr(), v_out.data_ptr(),
            self.k_cache[layer_idx].data_ptr(), self.v_cache[layer_idx].data_ptr(),
            ids.data_ptr(), len(block_ids), n, self.n_kv_heads, self.head_dim, self.block_size,
            self.num_blocks, _lib.dtype_code(self.dtype), _lib.stream_ptr(self.device))
        _lib.check(rc, "KVCache.read_kv_blocks")
        return k_out, v_out

    def get_memory_bytes(self):
        """Total bytes of K and V storage over all layers (kv_cache.py:57-61)."""
        return (self.num_layers * self.num_blocks * self.block_size *
                self.n_kv_heads * self.head_dim * 2) * self.dtype.itemsize

    # -- fused path (no reference counterpart) --------------------------------
    def write_kv_slots(self, layer_idx, slot_mapping, k, v, err_count=None):
        """Write token t of k/v [T, Hkv, D] to flat slot ``slot_mapping[t]`` in one launch.

        Replaces the per-chunk ``write_kv`` loop of llama.py:199-209 and the
        per-token loop of llama.py:381-386.  ``slot_mapping`` is an int32 device
        tensor [T]; negative slots are skipped.  ``err_count`` (uint32/int32
        device scalar) counts tokens whose slot is past the cache.
        """
        return reshape_and_cache(self.k_cache[layer_idx], self.v_cache[layer_idx], k, v,
                                 slot_mapping, err_count=err_count)

    def write_rope_slots(self, layer_idx, slot_mapping, positions, rope, q, k, v, *, pairs="adjacent", out=None,
                         err_count=None):
        """``write_kv_slots`` of keys that are rotated on the way; returns the rotated queries.  See
        ``rope_and_cache``."""
        return rope_and_cache(self.k_cache[layer_idx], self.v_cache[layer_idx], q, k, v, slot_mapping, positions, rope,
                              pairs=pairs, out=out, err_count=err_count)

    def keep_draft_path(self, path, counts, context_lens, block_tables):
        """Moves an accepted path's K/V to where the sequences go on, in all layers; see ``keep_draft_rows``."""
        keep_draft_rows(self.k_cache, self.v_cache, path, counts, context_lens, block_tables)


class FP8KVCache:
    """Block-based K/V cache held in 8 bits, with ``KVCache``'s interface (no reference counterpart).

    ``k_cache`` / ``v_cache`` hold e4m3 numbers [num_blocks, n_kv_heads, block_size, head_dim] per layer
    and ``k_scale`` / ``v_scale`` a power of two for each block and KV head [num_blocks, n_kv_heads]
    (float32); an element stands for number * scale.  ``dtype`` is the model's: rows are written from it
    and read back in it.  A block's scale fits the rows written so far: writing its row 0 starts it
    anew (rows that the call does not write become zero), and a later row that needs a larger scale has
    the rows before it rounded again.  (A ``KVCache`` takes a block's rows in any order; here row 0 comes
    first.)  NaN and infinite elements are stored as NaN; values read back are limited to ``dtype``'s largest
    finite number.  head_dim 64, 128 or 256, block_size at most 1024.
    """

    def __init__(self, num_layers, num_blocks, block_size, n_kv_heads, head_dim, dtype, device="cuda"):
        self.num_layers = num_layers
        self.num_blocks = num_blocks
        self.block_size = block_size
        self.n_kv_heads = n_kv_heads
        self.head_dim = head_dim
        self.dtype = as_torch_dtype(dtype)
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise ValueError("FP8KVCache storage must be on a HIP device")
        if head_dim not in (64, 128, 256):
            raise ValueError(f"FP8KVCache: head_dim {head_dim} not supported (64, 128, 256)")
        if not 1 <= block_size <= 1024:
            raise ValueError(f"FP8KVCache: block_size {block_size} not in 1..1024")
        shape = (num_blocks, n_kv_heads, block_size, head_dim)

        def zeros():
            return [torch.zeros(shape, dtype=torch.uint8, device=self.device).view(torch.float8_e4m3fn)
                    for _ in range(num_layers)]

        def scales():      # the least scale: any row raises it
            return [torch.full(shape[:2], 2.0 ** -100, dtype=torch.float32, device=self.device)
                    for _ in range(num_layers)]

        self.k_cache, self.v_cache = zeros(), zeros()
        self.k_scale, self.v_scale = scales(), scales()

    _rows = KVCache._rows

    def write_kv(self, layer_idx, block_id, start_offset, k, v):
        """Write k/v [T, Hkv, D] to rows start_offset .. start_offset + T - 1 of a block."""
        k, ks = self._rows(k, "k")
        v, vs = self._rows(v, "v")
        if k.shape[0] != v.shape[0]:
            raise ValueError("k and v must hold the same number of tokens")
        kc = self.k_cache[layer_idx]
        _lib.call("FP8KVCache.write_kv", kc.get_device(), _lib.load().tv_write_kv_fp8,
                  kc.data_ptr(), self.v_cache[layer_idx].data_ptr(), self.k_scale[layer_idx].data_ptr(),
                  self.v_scale[layer_idx].data_ptr(), k.data_ptr(), v.data_ptr(), int(block_id), int(start_offset),
                  k.shape[0], self.n_kv_heads, self.head_dim, self.block_size, self.num_blocks, ks, vs,
                  _lib.dtype_code(self.dtype))

    def write_kv_slots(self, layer_idx, slot_mapping, k, v, err_count=None):
        """Write token t of k/v [T, Hkv, D] to flat slot ``slot_mapping[t]`` (int32 device tensor) in one
        launch; negative slots are skipped, of equal slots the last token is written, and ``err_count``
        counts tokens whose slot is past the cache."""
        return reshape_and_cache_fp8(self.k_cache[layer_idx], self.v_cache[layer_idx], self.k_scale[layer_idx],
                                     self.v_scale[layer_idx], k, v, slot_mapping, err_count=err_count)

    def read_kv_blocks(self, layer_idx, block_ids, context_len):
        """(k, v) [context_len, Hkv, D] of ``dtype``: the rows of ``block_ids`` (a list, or an int32 tensor
        on the device, which is read without a host copy) as values."""
        kc = self.k_cache[layer_idx]
        if isinstance(block_ids, torch.Tensor):
            if block_ids.dtype != torch.int32 or block_ids.get_device() != kc.get_device() or \
                    not block_ids.is_contiguous():
                raise ValueError("block_ids must be a contiguous int32 tensor on the cache's device")
            count = block_ids.numel()
        else:
            count = len(block_ids)
        n = min(int(context_len), count * self.block_size)
        if n < 0:
            raise ValueError("context_len must be >= 0")
        k_out = torch.empty((n, self.n_kv_heads, self.head_dim), dtype=self.dtype, device=kc.device)
        v_out = torch.empty_like(k_out)
        if n == 0:
            return k_out, v_out
        ids = block_ids if isinstance(block_ids, torch.Tensor) else \
            torch.tensor(list(block_ids), dtype=torch.int32).to(kc.device)
        _lib.call("FP8KVCache.read_kv_blocks", kc.get_device(), _lib.load().tv_read_kv_blocks_fp8,
                  k_out.data_ptr(), v_out.data_ptr(), kc.data_ptr(), self.v_cache[layer_idx].data_ptr(),
                  self.k_scale[layer_idx].data_ptr(), self.v_scale[layer_idx].data_ptr(), ids.data_ptr(), count, n,
                  self.n_kv_heads, self.head_dim, self.block_size, self.num_blocks, _lib.dtype_code(self.dtype))
        return k_out, v_out

    def get_memory_bytes(self):
        """Total bytes of the numbers and scales over all layers."""
        return self.num_layers * self.num_blocks * self.n_kv_heads * 2 * (self.block_size * self.head_dim + 4)


def check_fp8_cache(k_cache, v_cache, k_scale, v_scale):
    """Shape [NB, Hkv, bs, D] and device index of one layer's 8-bit cache; raises ValueError."""
    shape = k_cache.shape
    if len(shape) != 4 or v_cache.shape != shape or not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("k_cache / v_cache must be dense [NB, Hkv, bs, D] tensors of one shape")
    if k_cache.dtype != torch.float8_e4m3fn or v_cache.dtype != torch.float8_e4m3fn:
        raise ValueError("k_cache / v_cache must be float8_e4m3fn")
    for t in (k_scale, v_scale):
        if t.dtype != torch.float32 or t.shape != shape[:2] or not t.is_contiguous():
            raise ValueError(f"k_scale / v_scale must be dense float32 [{shape[0]}, {shape[1]}]")
    index = k_cache.get_device()
    check_devices(index, v_cache, k_scale, v_scale)
    return (*shape, index)


def check_devices(index, *tensors):
    """Raises ValueError for a tensor that is not on device ``index`` (-1: the CPU)."""
    for t in tensors:
        if t.get_device() != index:
            raise ValueError("all tensors must be on the cache's device")


def reshape_and_cache_fp8(k_cache, v_cache, k_scale, v_scale, k, v, slot_mapping, err_count=None):
    """``reshape_and_cache`` into an 8-bit cache (one layer's tensors of ``FP8KVCache``)."""
    nb, hkv, bs, d, index = check_fp8_cache(k_cache, v_cache, k_scale, v_scale)
    if k.dim() != 3 or k.shape[1] != hkv or k.shape[2] != d or v.shape != k.shape:
        raise ValueError(f"k/v must be [T, {hkv}, {d}]")
    t = k.shape[0]
    ks, vs = k.stride(), v.stride()
    if ks[2] != 1 or ks[1] != d or vs[2] != 1 or vs[1] != d:
        raise ValueError("k/v heads and head_dim must be contiguous")
    if k.dtype != v.dtype:
        raise ValueError("k and v must share a dtype")
    if slot_mapping.dtype != torch.int32 or slot_mapping.numel() != t or not slot_mapping.is_contiguous():
        raise ValueError("slot_mapping must be contiguous int32 with one entry per token")
    check_devices(index, k, v, slot_mapping)
    if index < 0:
        raise ValueError("the cache must be on a HIP device")
    if err_count is not None and (err_count.get_device() != index or
                                  err_count.dtype not in (torch.int32, torch.uint32)):
        raise ValueError("err_count must be an int32/uint32 tensor on the cache's device")
    _lib.call("reshape_and_cache_fp8", index, _lib.load().tv_reshape_and_cache_fp8,
              k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), k.data_ptr(),
              v.data_ptr(), slot_mapping.data_ptr(), t, hkv, d, bs, nb, ks[0] if t > 1 else hkv * d,
              vs[0] if t > 1 else hkv * d, _lib.dtype_code(k.dtype),
              err_count.data_ptr() if err_count is not None else None)


def reshape_and_cache(k_cache, v_cache, k, v, slot_mapping, err_count=None):
    """Fused cache write: ``cache[slot // bs, slot % bs] = row`` for every token."""
    nb, bs, hkv, d = k_cache.shape
    if tuple(v_cache.shape) != (nb, bs, hkv, d) or not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("k_cache / v_cache must be dense [NB, bs, Hkv, D] tensors of one shape")
    if k.dim() != 3 or tuple(k.shape[1:]) != (hkv, d) or tuple(v.shape) != tuple(k.shape):
        raise ValueError(f"k/v must be [T, {hkv}, {d}]")
    if not (k.stride(2) == 1 and k.stride(1) == d and v.stride(2) == 1 and v.stride(1) == d):
        raise ValueError("k/v heads and head_dim must be contiguous")
    if k.dtype != k_cache.dtype or v.dtype != k_cache.dtype:
        raise ValueError("k/v dtype must match the cache dtype")
    if slot_mapping.dtype != torch.int32 or slot_mapping.numel() != k.shape[0]:
        raise ValueError("slot_mapping must be int32 with one entry per token")
    if not slot_mapping.is_contiguous():
        raise ValueError("slot_mapping must be contiguous")
    dev = k_cache.device
    for t in (v_cache, k, v, slot_mapping):
        if t.device != dev:
            raise ValueError("all tensors must be on the cache's device")
    if err_count is not None and (err_count.device != dev or err_count.dtype not in (torch.int32, torch.uint32)):
        raise ValueError("err_count must be an int32/uint32 tensor on the cache's device")
    lib = _lib.load()
    t = k.shape[0]
    rc = lib.tv_reshape_and_cache(
        k_cache.data_ptr(), v_cache.data_ptr(), k.data_ptr(), v.data_ptr(), slot_mapping.data_ptr(),
        t, hkv, d, bs, nb, k.stride(0) if t > 1 else hkv * d, v.stride(0) if t > 1 else hkv * d,
        _lib.dtype_code(k_cache.dtype), err_count.data_ptr() if err_count is not None else None,
        _lib.stream_ptr(dev))
    _lib.check(rc, "reshape_and_cache")


def _token_stride(x, shape, name):
    """Elements between the tokens of x, which has to be of ``shape`` [N, heads, d] with dense heads."""
    if x.shape != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {list(x.shape)}")
    n, heads, d = shape
    s0, s1, s2 = x.stride()             # a dimension of size 1 may have any
    if (s2 != 1 and d > 1) or (s1 != d and heads > 1):
        raise ValueError(f"{name}: heads and head_dim must be contiguous")
    if n <= 1:
        return heads * d
    if s0 < heads * d:
        raise ValueError(f"{name}: tokens overlap")
    return s0


def rope_and_cache(k_cache, v_cache, q, k, v, slot_mapping, positions, rope, *, pairs="adjacent", out=None,
                   err_count=None):
    """Rotates queries and keys to their positions and writes keys and values into the cache, in one launch
    (no reference counterpart as one call: apply_rope, llama.py:34-55, then the writes of llama.py:188-209).

    q [N, Hq, D], k / v [N, Hkv, D] of the cache's dtype, rows possibly strided (views of one projection);
    slot_mapping and positions [N] int32 (or [B, T] with B * T = N); rope [P, R / 2, 2] float32, cos and sin of
    each pair by position (``Llama.rope``).  The first R elements of a head are rotated, pairs (2i, 2i + 1), or with
    ``pairs="halves"`` (i, i + R / 2); the others stay as they are.  Returns the rotated queries [N, Hq, D], in
    ``out`` where it is given (which may be q).

    A negative slot is padding: its K/V are not written.  A slot past the cache is not written and counted
    in ``err_count`` (int32/uint32 device scalar); nor is a token whose position the table does not hold,
    whose queries become NaN.  The slots of a call differ from each other.
    """
    index = k_cache.get_device()
    if index < 0:
        raise ValueError(f"the cache must be on a HIP device (got {k_cache.device})")
    shape = k_cache.shape
    if len(shape) != 4 or v_cache.shape != shape or not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("k_cache / v_cache must be dense [NB, bs, Hkv, D] tensors of one shape")
    nb, bs, hkv, d = shape
    if q.dim() != 3:
        raise ValueError(f"q must be [N, Hq, {d}], got {list(q.shape)}")
    n, hq, _ = q.shape
    if len(k) != n or len(v) != n:
        raise ValueError("q, k and v must hold the same number of tokens")
    q_stride = _token_stride(q, (n, hq, d), "q")
    k_stride, v_stride = _token_stride(k, (n, hkv, d), "k"), _token_stride(v, (n, hkv, d), "v")
    dtype = k_cache.dtype
    if not (v_cache.dtype is dtype and q.dtype is dtype and k.dtype is dtype and v.dtype is dtype):
        raise ValueError("q, k, v and the caches must share a dtype")
    if slot_mapping.dtype is not torch.int32 or slot_mapping.numel() != n or not slot_mapping.is_contiguous():
        raise ValueError("slot_mapping must be contiguous int32 with one entry per token")
    if positions.dtype is not torch.int32 or positions.numel() != n or not positions.is_contiguous():
        raise ValueError("positions must be contiguous int32 with one entry per token")
    if rope.dtype is not torch.float32 or rope.dim() != 3 or rope.shape[2] != 2 or not rope.is_contiguous():
        raise ValueError("rope must be contiguous float32 [positions, pairs, 2]")
    rope_len, half, _ = rope.shape
    if not 1 <= 2 * half <= d or rope_len < 1:
        raise ValueError(f"rope of {half} pairs does not fit head_dim {d}")
    if pairs not in ("adjacent", "halves"):
        raise ValueError(f"pairs must be 'adjacent' or 'halves', got {pairs!r}")
    check_devices(index, v_cache, q, k, v, slot_mapping, positions, rope)
    if out is None:
        out = q.new_empty((n, hq, d))
        out_stride = hq * d
    else:
        if out.dtype is not dtype or out.shape != q.shape or out.get_device() != index:
            raise ValueError("out must be like q")
        out_stride = _token_stride(out, (n, hq, d), "out")
    if err_count is not None and (err_count.get_device() != index or
                                  err_count.dtype not in (torch.int32, torch.uint32)):
        raise ValueError("err_count must be an int32/uint32 tensor on the cache's device")
    _lib.call("rope_and_cache", index, _lib.load().tv_rope_and_cache,
              out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(),
              slot_mapping.data_ptr(), positions.data_ptr(), rope.data_ptr(), rope_len, 2 * half,
              1 if pairs == "halves" else 0, n, hq, hkv, d, bs, nb, out_stride, q_stride, k_stride, v_stride,
              _lib.dtype_code(dtype), err_count.data_ptr() if err_count is not None else None)
    return out


def keep_draft_rows(k_caches, v_caches, path, counts, context_lens, block_tables):
    """Moves the K/V of a verified tree's accepted nodes to where their sequences go on, in every layer's cache
    [NB, bs, Hkv, D]: position context + path[j] -> context + j for j < count, in one launch per 64 layers (no
    reference counterpart).

    path [B, T], counts and context_lens [B] int32 (``sampling.verify_draft_tree``; the context before the
    tree), block_tables [B, columns] int32.  ``path`` rises from node to node.  Entries outside j .. T - 1 and
    positions that the table does not reach, or whose block is outside the cache, are not moved.  Other rows stay as
    they are.
    """
    n = len(k_caches)
    if n == 0 or len(v_caches) != n:
        raise ValueError("k_caches and v_caches must hold one tensor per layer each")
    first = k_caches[0]
    shape, dtype, index = first.shape, first.dtype, first.get_device()
    if index < 0:
        raise ValueError(f"the caches must be on a HIP device (got {first.device})")
    if len(shape) != 4:
        raise ValueError("caches must be dense [NB, bs, Hkv, D] tensors")
    for c in (*k_caches, *v_caches):
        if c.shape != shape or c.dtype is not dtype or not c.is_contiguous():
            raise ValueError("caches must be dense tensors of one shape and dtype")
        if c.get_device() != index:
            raise ValueError("all tensors must be on the cache's device")
    tree = path.shape
    if len(tree) != 2 or tree[1] < 1:
        raise ValueError(f"path must be [B, T], got {list(tree)}")
    check_int32(index, tree, ("path", path))
    check_int32(index, tree[:1], ("counts", counts), ("context_lens", context_lens))
    columns = check_block_tables(index, tree[0], block_tables)
    nb, bs, hkv, d = shape
    array = ctypes.c_void_p * n
    _lib.call("keep_draft_rows", index, _lib.load().tv_keep_draft_rows, array(*[c.data_ptr() for c in k_caches]),
              array(*[c.data_ptr() for c in v_caches]), n, path.data_ptr(), counts.data_ptr(), context_lens.data_ptr(),
              block_tables.data_ptr(), *tree, columns, hkv, d, bs, nb, _lib.dtype_code(dtype))
