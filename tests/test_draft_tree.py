"""The layout of draft trees and the rows that are kept of them."""

import ctypes

import numpy as np
import pytest
import torch

from oracle import draft_tree as ref
from tests.random_cases import case_count, case_seed

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
gpu = pytest.mark.gpu


def rng_of(seed):
    return np.random.Generator(np.random.PCG64(seed))


def cuda(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def random_tree(rng, b, t):
    """Parents of every kind: chains, stars, several roots, and values that are no parent."""
    parents = np.empty((b, t), np.int32)
    for i in range(b):
        kind = rng.integers(4)
        for j in range(t):
            parents[i, j] = {0: j - 1, 1: 0 if j else -1, 2: rng.integers(0, j) if j else -1,
                             3: rng.integers(-2, t + 3)}[int(kind)]
    return parents


def random_tables(rng, rows, block, spare=3):
    """(tables [B, columns] of sequences of `rows` positions, blocks of the pool)."""
    need = -(-np.asarray(rows) // block)
    pool = int(need.sum()) + spare
    perm = rng.permutation(pool).astype(np.int32)
    table = np.zeros((len(need), max(1, int(need.max()))), np.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = perm[at:at + n]
        at += n
    return table, pool


# ---- the oracle, on the CPU -----------------------------------------------------------

def test_oracle_layout_of_a_small_tree():
    parents = np.array([[-1, 0, 0, 1, 3, 9]], np.int32)
    mask, pos, slots = ref.layout_ref(parents, [6], [5], np.array([[7, 2, 9]], np.int32), 4, 9)
    assert mask[0, :, 0].tolist() == [1, 3, 5, 11, 27, 32]
    assert pos[0].tolist() == [5, 6, 6, 7, 8, 5]
    assert slots[0].tolist() == [9, 10, 11, -1, -1, -1]          # block 9 is outside the cache


def test_oracle_words_of_more_than_64_nodes():
    seen = ref.ancestors_ref(np.arange(-1, 69), 70)
    words = ref.words_of(seen, 70)
    assert words.shape == (70, 2) and words[69].tolist() == [-1, 63] and words[63].tolist() == [-1, 0]


# ---- refusals: nothing is launched ----------------------------------------------------

def test_entry_points_validate_on_the_host():
    from tinyvllm_amd import _lib
    lib, p = _lib.load(), ctypes.c_void_p(256)
    base = [p] * 7 + [4, 8, 3, 16, 20, None]

    def layout(**kw):
        a = list(base)
        for i, v in kw.items():
            a[int(i[1:])] = v
        return lib.tv_draft_tree_layout(*a)

    for i in range(7):
        assert layout(**{f"_{i}": None}) == _lib.TV_EINVAL and b"null pointer" in lib.tv_last_error()
    assert layout(_0=ctypes.c_void_p(260)) == _lib.TV_EINVAL and b"misaligned" in lib.tv_last_error()
    assert layout(_7=-1) == _lib.TV_EINVAL and layout(_7=65536) == _lib.TV_EINVAL
    assert layout(_7=0) == _lib.TV_OK
    assert layout(_8=0) == _lib.TV_EINVAL and layout(_8=257) == _lib.TV_EINVAL and b"nodes" in lib.tv_last_error()
    for i in (9, 10, 11):
        assert layout(**{f"_{i}": 0}) == _lib.TV_EINVAL and b"block table" in lib.tv_last_error()
    assert layout(_10=1 << 16, _11=1 << 16) == _lib.TV_EINVAL and b"32 bits" in lib.tv_last_error()

    two = (ctypes.c_void_p * 2)(256, 512)
    hole = (ctypes.c_void_p * 2)(256, None)
    odd = (ctypes.c_void_p * 2)(256, 513)
    base2 = [two, two, 2, p, p, p, p, 4, 8, 3, 2, 64, 16, 20, 1, None]

    def keep(**kw):
        a = list(base2)
        for i, v in kw.items():
            a[int(i[1:])] = v
        return lib.tv_keep_draft_rows(*a)

    for i in (3, 4, 5, 6):
        assert keep(**{f"_{i}": None}) == _lib.TV_EINVAL and b"null pointer" in lib.tv_last_error()
    assert keep(_0=hole) == _lib.TV_EINVAL and b"layer 1" in lib.tv_last_error()
    assert keep(_1=odd) == _lib.TV_EINVAL and b"misaligned" in lib.tv_last_error()
    assert keep(_2=-1) == _lib.TV_EINVAL and keep(_2=0) == _lib.TV_OK and keep(_7=0) == _lib.TV_OK
    assert keep(_8=300) == _lib.TV_EINVAL and keep(_10=0) == _lib.TV_EINVAL and keep(_14=3) == _lib.TV_EINVAL


def test_python_refuses_tensors_on_the_cpu():
    from tinyvllm_amd.draft_tree import draft_tree_layout
    from tinyvllm_amd.kv_cache import keep_draft_rows
    i = torch.zeros((2, 4), dtype=torch.int32)
    with pytest.raises(ValueError, match="HIP device"):
        draft_tree_layout(i, i[:, 0], i[:, 0], i, 16, 8)
    c = torch.zeros((4, 16, 2, 64))
    with pytest.raises(ValueError, match="HIP device"):
        keep_draft_rows([c], [c], i, i[:, 0], i[:, 0], i)
    with pytest.raises(ValueError, match="per layer"):
        keep_draft_rows([], [], i, i[:, 0], i[:, 0], i)


@gpu
def test_python_refusals_on_the_gpu():
    from tinyvllm_amd.draft_tree import draft_tree_layout
    from tinyvllm_amd.kv_cache import keep_draft_rows
    i = torch.zeros((2, 4), dtype=torch.int32, device="cuda")
    one = torch.zeros(2, dtype=torch.int32, device="cuda")
    for args, what in (((i.long(), one, one, i), "parents"), ((i, one[:1], one, i), "tree_lens"),
                       ((i, one, one.cpu(), i), "one HIP device"), ((i, one, one, i[:1]), "block_tables"),
                       ((i.t().contiguous().t(), one, one, i), "parents"), ((i, one, one, i[:, :0]), "block_tables"),
                       ((i.new_zeros((2, 257)), one, one, i), "256"), ((i[:, :0], one, one, i), "256")):
        with pytest.raises(ValueError, match=what):
            draft_tree_layout(*args, 16, 8)
    with pytest.raises(ValueError, match="block_size"):
        draft_tree_layout(i, one, one, i, 0, 8)
    c = torch.zeros((4, 16, 2, 64), device="cuda")
    for args, what in ((([c], [c.half()], i, one, one, i), "one shape and dtype"), (([c], [c, c], i, one, one, i), "per layer"),
                       (([c[0]], [c[0]], i, one, one, i), "dense"), (([c.transpose(1, 2)], [c], i, one, one, i), "dense"),
                       (([c], [c], i.long(), one, one, i), "path"), (([c], [c], i, one[:1], one, i), "counts"),
                       (([c.double()], [c.double()], i, one, one, i), "dtype")):
        with pytest.raises(ValueError, match=what):
            keep_draft_rows(*args)


# ---- layout -------------------------------------------------------------------------------

def check_layout(parents, lens, ctx, table, block, pool):
    from tinyvllm_amd.draft_tree import draft_tree_layout
    got = draft_tree_layout(cuda(parents), cuda(lens), cuda(ctx), cuda(table), block, pool)
    for a, want in zip(got, ref.layout_ref(parents, lens, ctx, table, block, pool)):
        assert np.array_equal(a.cpu().numpy(), want)


@gpu
@pytest.mark.parametrize("t", [1, 2, 7, 63, 64, 65, 128, 129, 192, 193, 256])
def test_layout(t):
    rng = rng_of(t)
    b = 9
    parents = random_tree(rng, b, t)
    parents[0] = np.arange(-1, t - 1)                            # one long chain
    lens = rng.integers(0, t + 1, b).astype(np.int32)
    lens[:3] = t, 0, 1
    ctx = rng.integers(0, 70, b).astype(np.int32)
    ctx[3] = 0
    table, pool = random_tables(rng, ctx + t, 16)
    check_layout(parents, lens, ctx, table, 16, pool)


@gpu
def test_layout_with_lengths_out_of_range_and_short_tables():
    """Lengths are clamped; positions past the table or in a block outside the cache have no slot."""
    rng = rng_of(5)
    parents = random_tree(rng, 4, 20)
    lens = np.array([25, -3, 20, 20], np.int32)
    ctx = np.array([10, 4, -7, 30], np.int32)
    table = rng.permutation(12).astype(np.int32).reshape(4, 3)
    table[2, 1] = -1
    check_layout(parents, lens, ctx, table, 11, 9)


@gpu
def test_contexts_next_to_32_bits():
    """No table reaches these positions; the lengths are only counted."""
    from tinyvllm_amd.draft_tree import draft_tree_layout
    ctx = cuda(np.array([2 ** 31 - 6, 2 ** 31 - 1], np.int32))
    parents = cuda(np.tile(np.arange(-1, 4, dtype=np.int32), (2, 1)))
    lens, table = cuda(np.array([5, 1], np.int32)), cuda(np.arange(8, dtype=np.int32).reshape(2, 4))
    out = draft_tree_layout(parents, lens, ctx, table, 16, 8)
    assert out.positions.tolist() == [[2 ** 31 - 6 + i for i in range(5)], [2 ** 31 - 1, 0, 0, 0, 0]]
    assert (out.slots == -1).all()
    k = torch.randn((8, 16, 2, 8), device="cuda")
    before = k.clone()
    path = cuda(np.array([[0, 2, 4, -1, -1], [0, -1, -1, -1, -1]], np.int32))
    from tinyvllm_amd.kv_cache import keep_draft_rows
    keep_draft_rows([k], [k], path, cuda(np.array([3, 1], np.int32)), ctx, table)
    assert torch.equal(k, before)


@gpu
def test_layout_of_no_sequences():
    from tinyvllm_amd.draft_tree import draft_tree_layout
    none = torch.zeros((0,), dtype=torch.int32, device="cuda")
    out = draft_tree_layout(none.view(0, 5), none, none, none.view(0, 2), 16, 4)
    assert out.mask.shape == (0, 5, 1)


# ---- kept rows --------------------------------------------------------------------------------

def keep_ref(caches, path, counts, ctx, table, block):
    out = caches.copy()
    nb, t = caches.shape[1], path.shape[1]
    for b in range(len(counts)):
        def slot(pos):
            col = pos // block
            ok = col < table.shape[1] and 0 <= table[b, col] < nb
            return (int(table[b, col]), pos % block) if ok else None
        for j in range(min(max(int(counts[b]), 0), t)):
            if j < path[b, j] < t:
                a, z = slot(int(ctx[b] + path[b, j])), slot(int(ctx[b]) + j)
                if a and z:
                    out[:, z[0], z[1]] = caches[:, a[0], a[1]]
    return out


def check_keep(rng, layers, heads, d, block, dtype, path, counts, ctx, table, pool):
    from tinyvllm_amd.kv_cache import keep_draft_rows
    shape = (2 * layers, pool, block, heads, d)
    old = torch.from_numpy(rng.standard_normal(shape)).to("cuda", DTYPES[dtype])
    new = [c.clone() for c in old]
    keep_draft_rows(new[:layers], new[layers:], cuda(path), cuda(counts), cuda(ctx), cuda(table))
    want = keep_ref(old.double().cpu().numpy(), path, counts, ctx, table, block)
    assert np.array_equal(torch.stack(new).double().cpu().numpy(), want)


def rising_paths(rng, b, t):
    path, counts = np.full((b, t), -1, np.int32), np.zeros(b, np.int32)
    for i in range(b):
        n = int(rng.integers(0, t + 1))
        path[i, :n] = np.sort(rng.choice(t, n, replace=False))
        counts[i] = n
    return path, counts


@gpu
@pytest.mark.parametrize("dtype,heads,d", [("float32", 2, 64), ("bfloat16", 8, 128), ("float16", 1, 3), ("float32", 3, 5),
                                           ("bfloat16", 5, 6)])
@pytest.mark.parametrize("t,block", [(1, 16), (8, 16), (21, 5), (64, 1), (256, 32)])
def test_kept_rows(dtype, heads, d, t, block):
    """Paths that overlap their own places, in vectors of every width; other rows stay."""
    rng = rng_of(t + d)
    path, counts = rising_paths(rng, 6, t)
    ctx = rng.integers(0, 40, 6).astype(np.int32)
    table, pool = random_tables(rng, ctx + t, block)
    check_keep(rng, 2, heads, d, block, dtype, path, counts, ctx, table, pool)


@gpu
def test_kept_rows_of_many_layers():
    """More layers than one launch has pointers for."""
    rng = rng_of(3)
    path, counts = rising_paths(rng, 3, 12)
    ctx = np.array([0, 5, 17], np.int32)
    table, pool = random_tables(rng, ctx + 12, 8)
    check_keep(rng, 131, 2, 8, 8, "float16", path, counts, ctx, table, pool)


@gpu
def test_kept_rows_of_odd_paths():
    """Counts out of range are clamped; entries that are no later node, and positions without a block, stay."""
    rng = rng_of(4)
    path = np.array([[0, 3, 2, 9, 12, -1], [5, 5, 5, 5, 5, 5], [0, 1, 2, 3, 4, 5], [1, 2, 3, 4, 5, 6]], np.int32)
    counts = np.array([9, 1, -2, 6], np.int32)
    ctx = np.array([2, 0, 3, 6], np.int32)
    table = rng.permutation(12).astype(np.int32).reshape(4, 3)
    table[0, 2] = 99
    check_keep(rng, 1, 2, 64, 4, "float32", path, counts, ctx, table, 12)


@gpu
def test_kept_rows_through_the_cache():
    from tinyvllm_amd.kv_cache import KVCache
    rng = rng_of(6)
    cache = KVCache(3, 9, 4, 2, 16, "float16")
    for c in (*cache.k_cache, *cache.v_cache):
        c.copy_(torch.from_numpy(rng.standard_normal(c.shape)))
    old = np.stack([c.double().cpu().numpy() for c in (*cache.k_cache, *cache.v_cache)])
    path, counts = np.array([[0, 2, 5, -1, -1, -1]], np.int32), np.array([3], np.int32)
    table = np.array([[3, 8, 1]], np.int32)
    cache.keep_draft_path(cuda(path), cuda(counts), cuda(np.array([3], np.int32)), cuda(table))
    got = np.stack([c.double().cpu().numpy() for c in (*cache.k_cache, *cache.v_cache)])
    assert np.array_equal(got, keep_ref(old, path, counts, [3], table, 4))


@gpu
def test_layout_and_kept_rows_in_a_graph():
    """Replays follow their inputs, with eager work between them."""
    from tinyvllm_amd.draft_tree import draft_tree_layout
    from tinyvllm_amd.kv_cache import keep_draft_rows
    rng = rng_of(8)
    b, t, block = 5, 30, 8
    bufs = [torch.zeros(s, dtype=torch.int32, device="cuda") for s in ((b, t), (b,), (b,), (b, 12), (b, t), (b,))]
    parents, lens, ctx, table, path, counts = bufs
    k, v = (torch.zeros((b * 12, block, 2, 16), device="cuda") for _ in range(2))
    draft_tree_layout(parents, lens, ctx, table, block, b * 12)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        out = draft_tree_layout(parents, lens, ctx, table, block, b * 12)
        keep_draft_rows([k], [v], path, counts, ctx, table)
    for _ in range(4):
        new = [random_tree(rng, b, t), rng.integers(0, t + 1, b), rng.integers(0, 60, b),
               rng.permutation(b * 12).reshape(b, 12), *rising_paths(rng, b, t)]
        new = [np.asarray(x, np.int32) for x in new]
        for buf, x in zip(bufs, new):
            buf.copy_(cuda(x))
        rows = torch.from_numpy(rng.standard_normal((2, *k.shape))).float().cuda()
        k.copy_(rows[0])
        v.copy_(rows[1])
        graph.replay()
        torch.cuda.synchronize()
        for a, want in zip(out, ref.layout_ref(*new[:4], block, b * 12)):
            assert np.array_equal(a.cpu().numpy(), want)
        want = keep_ref(rows.double().cpu().numpy(), new[4], new[5], new[2], new[3], block)
        assert np.array_equal(torch.stack([k, v]).double().cpu().numpy(), want)


@gpu
@pytest.mark.parametrize("case", range(case_count(6)))
def test_random_layouts(case):
    rng = rng_of(case_seed(900) + case)
    b, t, block = int(rng.integers(1, 40)), int(rng.integers(1, 257)), int(rng.integers(1, 40))
    ctx = rng.integers(0, 500, b).astype(np.int32)
    table, pool = random_tables(rng, ctx + t, block)
    check_layout(random_tree(rng, b, t), rng.integers(0, t + 1, b).astype(np.int32), ctx, table, block, pool)
