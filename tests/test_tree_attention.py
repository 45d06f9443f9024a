"""Attention of draft trees over the paged cache."""

import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import draft_tree as ref
from tests.fp8_tolerance import rounded_weights_bound
from tests.random_cases import case_count, case_seed
from tests.test_draft_tree import DTYPES, cuda, gpu, random_tables, random_tree, rng_of


def test_entry_point_validates_on_the_host():
    from tinyvllm_amd import _lib
    lib, p = _lib.load(), ctypes.c_void_p(256)
    base = [p] * 8 + [0, 4, 8, 8, 2, 64, 16, 20, 8, 8, 4096, 512, 0.1, 1, 1, 0, None, 0, None]

    def call(**kw):
        a = list(base)
        for i, v in kw.items():
            a[int(i[1:])] = v
        return lib.tv_paged_tree(*a)

    for i in range(8):
        assert call(**{f"_{i}": None}) == _lib.TV_EINVAL and b"null pointer" in lib.tv_last_error()
    for i in (0, 1, 2, 3):
        assert call(**{f"_{i}": ctypes.c_void_p(264)}) == _lib.TV_EINVAL and b"aligned" in lib.tv_last_error()
    assert call(_7=ctypes.c_void_p(260)) == _lib.TV_EINVAL and b"aligned" in lib.tv_last_error()
    assert call(_9=-1) == _lib.TV_EINVAL and call(_9=0) == _lib.TV_OK
    assert call(_10=0) == _lib.TV_EINVAL and call(_10=257) == _lib.TV_EINVAL
    assert call(_11=7) == _lib.TV_EINVAL and b"head counts" in lib.tv_last_error()
    assert call(_13=96) == _lib.TV_EUNSUPPORTED and b"head_dim 96" in lib.tv_last_error()
    assert call(_14=0) == _lib.TV_EINVAL and call(_15=0) == _lib.TV_EINVAL
    assert call(_16=4) == _lib.TV_EINVAL and call(_17=0) == _lib.TV_EINVAL and b"block table" in lib.tv_last_error()
    assert call(_14=1 << 10, _15=1 << 11, _16=1 << 21, _17=1 << 21) == _lib.TV_EINVAL and b"too large" in lib.tv_last_error()
    assert call(_18=4097) == _lib.TV_EINVAL and call(_19=504) == _lib.TV_EINVAL and b"strides" in lib.tv_last_error()
    assert call(_21=3) == _lib.TV_EINVAL and call(_22=2) == _lib.TV_EINVAL and b"dtype" in lib.tv_last_error()
    for n in (-1, (1 << 16) + 1):
        assert call(_23=n) == _lib.TV_EINVAL and b"work_groups" in lib.tv_last_error()
    assert call(_23=64) == _lib.TV_EINVAL and b"workspace" in lib.tv_last_error()
    assert call(_23=64, _24=ctypes.c_void_p(264), _25=1 << 30) == _lib.TV_EINVAL and b"16-byte" in lib.tv_last_error()
    assert call(_9=65535, _10=256, _11=256, _19=16384) == _lib.TV_EINVAL and b"grid" in lib.tv_last_error()
    assert lib.tv_paged_tree_workspace_bytes(4, 8, 8, 2, 64, 1, 0) == 0
    need = lib.tv_paged_tree_workspace_bytes(4, 8, 8, 2, 64, 1, 64)
    assert need > 0 and call(_23=64, _24=p, _25=need - 1) == _lib.TV_EINVAL and b"workspace" in lib.tv_last_error()
    assert lib.tv_paged_tree_work_groups(4, 8, 7, 2, 64, 8, 16, 1) < 0


def test_python_refuses_tensors_on_the_cpu():
    from tinyvllm_amd.attention import paged_tree_attention
    i = torch.zeros((2, 4), dtype=torch.int32)
    c = torch.zeros((4, 16, 2, 64))
    with pytest.raises(ValueError, match="HIP device"):
        paged_tree_attention(torch.zeros((2, 4, 4, 64)), c, c, i, i[:, 0], i[:, 0], torch.zeros((2, 4, 1)), 4, 2, 64, 16)


class Case:
    """A batch of trees over a cache, on the host in float64 and on the device."""

    def __init__(self, rng, dtype, hq, hkv, d, block, lens, ctx, nodes, trees=True, scale=1.0, spare=3):
        b = len(lens)
        self.dtype, self.heads, self.block, self.nodes = dtype, (hq, hkv, d), block, nodes
        self.lens, self.ctx = np.asarray(lens, np.int32), np.asarray(ctx, np.int32)
        self.table, self.pool = random_tables(rng, np.maximum(self.ctx, 0) + nodes, block, spare)
        t = DTYPES[dtype]
        self.q = torch.from_numpy(rng.standard_normal((b, nodes, hq, d)) * scale).to("cuda", t)
        self.k, self.v = (torch.from_numpy(rng.standard_normal((self.pool, block, hkv, d))).to("cuda", t) for _ in range(2))
        if trees:
            parents = random_tree(rng, b, nodes)
            self.seen = np.stack([ref.ancestors_ref(p, nodes) for p in parents])
        else:
            self.seen = rng.random((b, nodes, nodes)) < 0.3       # any mask, empty rows among them
            self.seen[:, ::5] = False
        self.mask = np.stack([ref.words_of(s, nodes) for s in self.seen])

    def args(self, mask=None):
        return (self.q, self.k, self.v, cuda(self.table), cuda(self.ctx), cuda(self.lens),
                cuda(self.mask if mask is None else mask), *self.heads, self.block)

    def run(self, **kw):
        from tinyvllm_amd.attention import paged_tree_attention
        return paged_tree_attention(*self.args(), **kw)

    def want(self, b, width=None):
        """(out, bound, dev) of sequence b and its number of keys; at most `width` keys exist."""
        hq, hkv, d = self.heads
        width = self.table.shape[1] * self.block if width is None else width
        c, n = min(max(int(self.ctx[b]), 0), width), min(max(int(self.lens[b]), 0), self.nodes)
        keys = min(c + n, width)
        ids = self.table[b, :-(-keys // self.block)].astype(np.int64)
        ok = (ids >= 0) & (ids < self.pool)
        rows = [np.where(ok[:, None, None, None], x[cuda(np.where(ok, ids, 0))].double().cpu().numpy(), np.nan)
                .reshape(-1, hkv, d)[:keys] for x in (self.k, self.v)]
        seen = np.zeros((self.nodes, keys), bool)
        seen[:n, :c] = True
        seen[:n, c:] = self.seen[b, :n, :keys - c]
        return ref.attend_ref(self.q[b].double().cpu().numpy(), *rows, seen, 1 / math.sqrt(d)), rows, keys

    def check(self, got, out_dtype=None, width=None, rows=None):
        got = got.double().cpu().numpy()
        for b in range(len(self.lens)):
            (want, bound, dev), kv, keys = self.want(b, width)
            vmax = float(np.abs(kv[1]).max()) if keys else 0.0
            tol = rounded_weights_bound(want, bound, dev, vmax, keys, self.heads[2], self.dtype, out_dtype or self.dtype)
            # nothing seen: exactly zero
            n = min(max(int(self.lens[b]), 0), self.nodes)
            diff = np.abs(got[b] - want)
            assert np.all(diff <= tol), (b, float(np.nanmax(diff)), float(np.nanmax(diff / tol)), np.argwhere(diff > tol)[:3])
            empty = np.arange(self.nodes) >= n
            if self.ctx[b] <= 0:
                empty = empty | ~self.seen[b, :, :n].any(1)
            assert np.all(got[b][empty] == 0)


HEADS = [(8, 2, 128), (8, 1, 64), (3, 3, 64), (10, 2, 128), (2, 1, 256), (33, 1, 64)]


@gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("hq,hkv,d", HEADS)
@pytest.mark.parametrize("nodes,block", [(1, 16), (5, 32), (17, 16), (64, 5), (65, 16), (130, 8), (9, 256), (16, 1)])
def test_shapes(dtype, hq, hkv, d, nodes, block):
    """One node to several row tiles, empty and short contexts, ragged trees; blocks of every kind."""
    rng = rng_of(nodes + d)
    lens = [nodes, max(0, nodes - 3), nodes // 2, 0, nodes]
    case = Case(rng, dtype, hq, hkv, d, block, lens, [0, 1, 63, 70, 201], nodes)
    got = case.run()
    assert got.shape == case.q.shape and got.dtype == case.q.dtype
    case.check(got)


@gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("d", [64, 128, 256])
def test_any_mask(dtype, d):
    """Masks that are no trees: nodes that do not see themselves, see later ones, or see nothing."""
    rng = rng_of(d)
    case = Case(rng, dtype, 4, 2, d, 16, [70, 70, 41, 3], [0, 129, 0, 64], 70, trees=False)
    case.check(case.run())
    case.check(case.run(work_groups=11))
    case.check(case.run(out_dtype=torch.float32), out_dtype="float32")


@gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("size", [1, 2, 7, 8, 33, 64, 500])
def test_work_groups(dtype, size):
    """Sequences of no, one and many parts in one launch; work-groups with many units, with a part of one and with
    nothing; parts that hold only keys some nodes do not see."""
    rng = rng_of(size + 100)
    case = Case(rng, dtype, 8, 2, 128, 16, [40, 40, 40, 0, 7], [0, 64, 500, 300, 1100], 40)
    case.check(case.run(work_groups=size))


@gpu
@pytest.mark.parametrize("size", [0, 5, 300, None])
def test_many_sequences(size):
    """More sequences than a work-group has threads, long runs of empty ones among them, at the ends too."""
    rng = rng_of(600)
    lens, ctx = rng.integers(0, 4, 700), rng.integers(0, 90, 700)
    lens[:5] = lens[100:480] = lens[-300:] = 0
    case = Case(rng, "float16", 4, 2, 64, 16, lens, ctx, 3)
    case.check(case.run(work_groups=size))


@gpu
def test_sequences_that_share_blocks():
    """A prompt's blocks in several sequences' tables, each with its own after them."""
    rng = rng_of(601)
    case = Case(rng, "bfloat16", 8, 2, 128, 16, [9, 9, 5], [100, 71, 96], 9)
    case.table[1:, :4] = case.table[0, :4]
    case.check(case.run())
    case.check(case.run(work_groups=9))


@gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_long_context(dtype):
    rng = rng_of(77)
    case = Case(rng, dtype, 8, 2, 64, 16, [12, 9], [20011, 3000], 12)
    case.check(case.run())
    case.check(case.run(work_groups=0))


@gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_large_scores(dtype):
    """Scores of some hundreds: a maximum that keeps rising, weights that vanish."""
    rng = rng_of(78)
    case = Case(rng, dtype, 4, 2, 128, 16, [20, 20], [700, 50], 20, scale=40.0)
    case.check(case.run())
    case.check(case.run(work_groups=10))


@gpu
def test_query_strides_and_shared_mask():
    """Queries out of a wider projection, sequences in another order of strides; one mask for all."""
    from tinyvllm_amd.attention import paged_tree_attention
    rng = rng_of(79)
    case = Case(rng, "bfloat16", 8, 2, 64, 16, [9, 9, 4], [100, 0, 33], 9)
    case.seen[:] = case.seen[0]
    case.mask[:] = case.mask[0]
    want = case.run()
    case.check(want)
    wide = torch.zeros((9, 3, 8 * 64 + 256), dtype=torch.bfloat16, device="cuda")        # node, sequence
    wide[..., :512] = case.q.transpose(0, 1).reshape(9, 3, 512)
    view = torch.as_strided(wide, (3, 9, 8, 64), (wide.stride(1), wide.stride(0), 64, 1))
    args = list(case.args(case.mask[0]))
    args[0] = view
    assert torch.equal(paged_tree_attention(*args), want)
    args[0] = case.q[:1].expand(3, 9, 8, 64)                                             # stride 0 between sequences
    assert torch.equal(paged_tree_attention(*args)[0], want[0])


@gpu
def test_one_token_is_paged_decode():
    """A tree of node 0 alone is a decode step over context + 1."""
    from tinyvllm_amd.attention import paged_decode_attention
    rng = rng_of(80)
    case = Case(rng, "float32", 8, 2, 128, 16, [1] * 6, [0, 1, 15, 16, 90, 300], 1)
    got = case.run()
    case.check(got)
    other = paged_decode_attention(case.q, case.k, case.v, cuda(case.table), cuda(case.ctx + 1), 8, 2, 128, 16)
    assert float((got - other).abs().max()) < 1e-5      # both are within 5e-6 of float64 at these sizes


@gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("size", [0, 9])
def test_tables_that_end_before_the_sequence(dtype, size):
    """Positions past the table, or past max_context_len's columns, do not exist."""
    rng = rng_of(81)
    case = Case(rng, dtype, 4, 2, 64, 16, [20, 20, 20], [30, 200, 85], 20)
    case.table = np.ascontiguousarray(case.table[:, :6])
    case.check(case.run(work_groups=size))
    case.check(case.run(work_groups=size, max_context_len=50), width=64)


@gpu
def test_lengths_out_of_range_are_clamped():
    rng = rng_of(82)
    case = Case(rng, "float16", 4, 2, 64, 16, [25, -4, 7], [40, 10, -5], 12)
    case.check(case.run())


@gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("size", [0, 9])
def test_values_that_are_not_finite(dtype, value, where, size):
    """Behind the tree and in other sequences' rows they reach nothing; in a drafted token's row the nodes that see
    it, in a context row every node.  An infinite key element times a query element of the other sign is a score of
    -inf, whose weight is 0 by the definition: those rows stay finite."""
    rng = rng_of(83)
    case = Case(rng, dtype, 8, 2, 64, 16, [11, 20], [70, 10], 20)
    clean = case.run(work_groups=size)
    cache = case.k if where == "k" else case.v

    def row(b, pos):
        return cache[int(case.table[b, pos // 16]), pos % 16]

    row(0, 70 + 11)[:] = value                        # past the tree, in its tile
    row(0, 70 + 19)[:] = value
    assert torch.equal(case.run(work_groups=size), clean)
    row(0, 70 + 3)[1, 5] = value                      # node 3, KV head 1
    got = case.run(work_groups=size)
    sees = torch.from_numpy(case.seen[0][:, 3].copy()).cuda() & (torch.arange(20, device="cuda") < 11)
    assert torch.equal(got[1], clean[1]) and torch.equal(got[0][:, :4], clean[0][:, :4])
    assert torch.equal(got[0][~sees], clean[0][~sees])

    def spoilt(q):                                    # by the element of the query that meets it
        return torch.ones_like(q, dtype=torch.bool) if where == "v" or value != value else q * value > 0

    assert torch.equal(got[0][sees][:, 4:].isnan().any(2), spoilt(case.q[0][sees][:, 4:, 5]))
    row(0, 40)[0, 9] = value                          # context, KV head 0
    got = case.run(work_groups=size)
    assert torch.equal((~got[0, :11, :4].isfinite()).any(2), spoilt(case.q[0, :11, :4, 9])) and torch.equal(got[1], clean[1])


@gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("size", [0, 9])
def test_block_ids_outside_the_cache(dtype, size):
    """NaN in the nodes that see the block, and nowhere else."""
    rng = rng_of(84)
    case = Case(rng, dtype, 4, 2, 128, 16, [20, 20, 20], [70, 60, 5], 20)
    clean = case.run(work_groups=size)
    case.table[0, 1] = case.pool                      # context
    case.table[1, 4] = -1                             # positions 64 .. 79: nodes 4 .. 19
    got = case.run(work_groups=size)
    assert got[0].isnan().all() and torch.equal(got[2], clean[2])
    sees = torch.from_numpy(case.seen[1][:, 4:].any(1)).cuda()
    assert got[1][sees].isnan().all() and torch.equal(got[1][~sees], clean[1][~sees])


@gpu
def test_queries_of_padding_are_not_looked_at():
    rng = rng_of(85)
    case = Case(rng, "bfloat16", 4, 2, 64, 16, [5, 9], [70, 100], 20)
    clean = case.run()
    case.q[0, 5:] = float("nan")
    case.q[1, 9:] = float("inf")
    assert torch.equal(case.run(), clean)
    case.q[0, 2, 1] = float("nan")
    got = case.run()
    assert got[0, 2, 1].isnan().all()
    got[0, 2, 1] = clean[0, 2, 1]
    assert torch.equal(got, clean)


@gpu
def test_results_repeat_and_do_not_depend_on_the_batch():
    rng = rng_of(86)
    case = Case(rng, "bfloat16", 8, 2, 128, 16, [16] * 5, [900, 40, 333, 0, 1200], 16)
    for size in (0, 24):
        a = case.run(work_groups=size)
        for _ in range(3):
            assert torch.equal(case.run(work_groups=size), a)
    a = case.run(work_groups=0)
    one = Case.__new__(Case)
    one.__dict__ = dict(case.__dict__)
    for name in ("lens", "ctx", "table", "mask"):
        setattr(one, name, getattr(case, name)[2:3])
    one.q = case.q[2:3]
    assert torch.equal(one.run(work_groups=0), a[2:3])


@gpu
def test_plans_in_graphs_follow_their_inputs():
    """Two captured plans, eager work between their replays: trees, lengths, tables and cache change."""
    from tinyvllm_amd.attention import PagedTreePlan
    rng = rng_of(87)
    case = Case(rng, "float16", 8, 2, 64, 16, [20] * 4, [600] * 4, 20)
    bufs = list(case.args())
    plans = [PagedTreePlan(*bufs, work_groups=size) for size in (20, 0)]
    for p in plans:
        p.run()
    torch.cuda.synchronize()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        for p in plans:
            p.run()
    for step in range(4):
        case.ctx = rng.integers(0, 600, 4).astype(np.int32)
        case.lens = rng.integers(0, 21, 4).astype(np.int32)
        case.seen = np.stack([ref.ancestors_ref(p, 20) for p in random_tree(rng, 4, 20)])
        case.mask = np.stack([ref.words_of(s, 20) for s in case.seen])
        case.table = case.table[rng.permutation(4)]
        for i, x in ((3, case.table), (4, case.ctx), (5, case.lens), (6, case.mask)):
            bufs[i].copy_(cuda(x))
        case.q.copy_(torch.from_numpy(rng.standard_normal(tuple(case.q.shape))))
        graph.replay()
        torch.cuda.synchronize()
        for p in plans:
            case.check(p.out)


@gpu
def test_two_streams_at_once():
    rng = rng_of(88)
    cases = [Case(rng, "bfloat16", 8, 2, 128, 16, [30, 12], [900, 2000], 30) for _ in range(2)]
    want = [c.run(work_groups=40) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(5):
        for i, c in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                got[i].append(c.run(work_groups=40))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


@gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_cache_of_more_than_4_gib(dtype):
    """Blocks beyond 2^32 bytes and 2^31 elements."""
    rng = rng_of(89)
    case = Case(rng, dtype, 8, 2, 128, 16, [9, 9], [100, 45], 9)
    first = (1 << 31) // (16 * 2 * 128)
    for name in ("k", "v"):
        large = torch.empty((first + case.pool, 16, 2, 128), dtype=case.k.dtype, device="cuda")
        large[first:] = getattr(case, name)
        setattr(case, name, large)
    case.table, case.pool = case.table + np.int32(first), first + case.pool
    case.check(case.run())
    case.check(case.run(work_groups=0))


@gpu
def test_python_refusals_on_the_gpu():
    from tinyvllm_amd.attention import paged_tree_attention
    rng = rng_of(90)
    case = Case(rng, "float16", 4, 2, 64, 16, [5, 5], [40, 20], 5)
    good = list(case.args())
    for at, bad, what in ((0, good[0][0], "queries must be"), (0, good[0].float(), "share a dtype"), (0, good[0].cpu(), "device"),
                          (0, good[0].transpose(1, 2).contiguous().transpose(1, 2), "contiguous"),
                          (0, good[0][:, :0], "T must be"), (1, good[1][:-1], "one shape"), (2, good[2].transpose(1, 2), "dense"),
                          (3, good[3].long(), "block_tables"), (3, good[3][:1], "block_tables"),
                          (4, good[4][:1], "context_lens"), (5, good[5].long(), "tree_lens"),
                          (6, good[6].int(), "tree_mask"), (6, good[6][:, :, 0], "tree_mask"), (6, good[6].cpu(), "device"),
                          (7, 8, "n_heads"), (8, 4, "cache shape"), (10, 8, "cache shape")):
        args = list(good)
        args[at] = bad
        with pytest.raises(ValueError, match=what):
            paged_tree_attention(*args)
    for kw, what in (({"work_groups": -1}, "work_groups"), ({"max_context_len": 0}, "columns"),
                     ({"out_dtype": torch.bfloat16}, "dtype")):
        with pytest.raises(ValueError, match=what):
            paged_tree_attention(*good, **kw)
    assert paged_tree_attention(case.q[:0], case.k, case.v, *(x[:0] for x in good[3:7]), 4, 2, 64, 16).shape == (0, 5, 4, 64)
    odd = Case(rng, "float16", 4, 2, 96, 16, [5], [40], 5)
    with pytest.raises(ValueError, match="head_dim 96"):
        odd.run()


@gpu
@pytest.mark.parametrize("case", range(case_count(24)))
def test_random_trees(case):
    rng = rng_of(case_seed(3300) + case)
    hkv = int(rng.integers(1, 5))
    hq, d = hkv * int(rng.integers(1, 10)), int(rng.choice([64, 64, 128, 256]))
    nodes, b = int(np.exp(rng.uniform(0, np.log(120)))), int(rng.integers(1, 7))
    block = int(rng.choice([1, 3, 8, 16, 16, 32, 64, 100]))
    c = Case(rng, str(rng.choice(sorted(DTYPES))), hq, hkv, d, block, rng.integers(0, nodes + 1, b),
             rng.integers(0, int(rng.choice([2, 80, 700])), b), nodes, trees=bool(rng.integers(2)))
    size = rng.choice([-1, 0, 3, 37])
    c.check(c.run(work_groups=None if size < 0 else int(size)))
