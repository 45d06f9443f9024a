"""The path through a draft tree that logits accept, and the token after it."""

import ctypes

import numpy as np
import pytest
import torch

from oracle import draft_tree as ref
from tests.random_cases import case_count, case_seed
from tests.test_draft_tree import DTYPES, cuda, gpu, random_tree, rng_of

# u is within this of a bound: fp64 sums of up to 2^18 terms, each off by 2^-50, may fall on either side
NEAR = 2.0 ** -32


def test_oracle_walks_and_draws():
    x = np.log(np.array([[[0.1, 0.2, 0.3, 0.4], [0.7, 0.1, 0.1, 0.1], [0.25, 0.25, 0.25, 0.25]]]))
    tokens, parents = np.array([[0, 3, 2]], np.int32), np.array([[-1, 0, 0]], np.int32)
    path, counts, follow, _ = ref.verify_ref(x, tokens, parents, [3])
    assert path.tolist() == [[0, 1, -1]] and counts[0] == 2 and follow[0] == 0
    temps = np.ones(1, np.float32)
    for u, want in ((0.39, ([0, 1, -1], 0)), (0.41, ([0, 2, -1], 1)), (0.75, ([0, -1, -1], 0)), (0.85, ([0, -1, -1], 1))):
        path, counts, follow, _ = ref.verify_ref(x, tokens, parents, [3], temps, np.full((1, 3), u, np.float32) * [1, 0.5, 0.5])
        # child 3 up to 0.4, child 2 up to 0.7, then tokens 0 and 1
        assert path[0].tolist() == want[0]
        if counts[0] == 1:
            assert follow[0] == want[1]


def test_entry_point_validates_on_the_host():
    from tinyvllm_amd import _lib
    lib, p = _lib.load(), ctypes.c_void_p(256)
    base = [p] * 9 + [4, 8, 1000, 1000, 0, p, 1 << 40, None]

    def call(**kw):
        a = list(base)
        for i, v in kw.items():
            a[int(i[1:])] = v
        return lib.tv_verify_draft_tree(*a)

    for i in range(7):
        assert call(**{f"_{i}": None}) == _lib.TV_EINVAL and b"null pointer" in lib.tv_last_error()
    assert call(_8=None) == _lib.TV_EINVAL and b"uniforms" in lib.tv_last_error()
    for i in (0, 3, 7, 8):
        assert call(**{f"_{i}": ctypes.c_void_p(257)}) == _lib.TV_EINVAL and b"misaligned" in lib.tv_last_error()
    assert call(_9=-1) == _lib.TV_EINVAL and call(_9=0) == _lib.TV_OK
    assert call(_10=0) == _lib.TV_EINVAL and call(_10=257) == _lib.TV_EINVAL
    assert call(_11=0) == _lib.TV_EINVAL and call(_12=999) == _lib.TV_EINVAL and b"bad shape" in lib.tv_last_error()
    assert call(_11=(1 << 24) + 1, _12=1 << 25) == _lib.TV_EINVAL
    assert call(_13=3) == _lib.TV_EINVAL and b"dtype" in lib.tv_last_error()
    need = lib.tv_verify_draft_tree_workspace_bytes(4, 8, 1000, 0)
    assert need > 0 and call(_15=need - 1) == _lib.TV_EINVAL and b"workspace" in lib.tv_last_error()
    assert call(_14=ctypes.c_void_p(264)) == _lib.TV_EINVAL and call(_14=None) == _lib.TV_EINVAL
    assert lib.tv_verify_draft_tree_workspace_bytes(0, 8, 1000, 0) == 0


def test_python_refuses_tensors_on_the_cpu():
    from tinyvllm_amd.sampling import verify_draft_tree
    i = torch.zeros((2, 4), dtype=torch.int32)
    with pytest.raises(ValueError, match="HIP device"):
        verify_draft_tree(torch.zeros((2, 4, 9)), i, i, i[:, 0])


@gpu
def test_python_refusals_on_the_gpu():
    from tinyvllm_amd.sampling import verify_draft_tree
    i = torch.zeros((2, 4), dtype=torch.int32, device="cuda")
    x, one, f = torch.zeros((2, 4, 9), device="cuda"), i[:, 0].contiguous(), torch.zeros(2, device="cuda")
    for args, kw, what in (((x[0], i, i, one), {}, "logits must be"), ((x.double(), i, i, one), {}, "dtype"),
                           ((x, i.long(), i, one), {}, "tokens"), ((x, i, i[:1], one), {}, "parents"),
                           ((x, i, i, one.cpu()), {}, "one HIP device"), ((x, i, i, i), {}, "tree_lens"),
                           ((x.transpose(1, 2).contiguous().transpose(1, 2), i, i, one), {}, "vocabulary"),
                           ((x.transpose(0, 1).contiguous().transpose(0, 1), i, i, one), {}, "evenly"),
                           ((x, i, i, one), {"temperatures": f}, "together"), ((x, i, i, one), {"uniforms": f}, "together"),
                           ((x, i, i, one), {"temperatures": f, "uniforms": f}, "uniforms must"),
                           ((x, i, i, one), {"temperatures": f.double(), "uniforms": x[:, :, 0].contiguous()}, "temperatures must"),
                           ((x[:, :0], i[:, :0], i[:, :0], one), {}, "logits must be"),
                           ((x.new_zeros((1, 257, 4)), i, i, one), {}, "256")):
        with pytest.raises(ValueError, match=what):
            verify_draft_tree(*args, **kw)
    out = verify_draft_tree(x[:0], i[:0], i[:0], one[:0])
    assert out.path.shape == (0, 4) and out.counts.shape == (0,)


def make(rng, b, t, v, dtype, spread=2.5, hits=0.7):
    """(logits float64 as the dtype holds them, tokens, parents, lens) with children among the likely tokens."""
    parents = random_tree(rng, b, t)
    lens = rng.integers(0, t + 1, b).astype(np.int32)
    lens[0] = t
    tokens = rng.integers(0, v, (b, t)).astype(np.int32)
    x = rng.standard_normal((b, t, v)) * spread
    for i in range(b):
        for j in range(1, t):
            if 0 <= parents[i, j] < j and rng.random() < hits:
                x[i, parents[i, j], tokens[i, j]] = x[i, parents[i, j]].max() + rng.normal()
    return torch.from_numpy(x).to("cuda", DTYPES[dtype]), tokens, parents, lens


def check(logits, tokens, parents, lens, temps=None, u=None, whole=True):
    from tinyvllm_amd.sampling import verify_draft_tree
    out = verify_draft_tree(logits, cuda(tokens), cuda(parents), cuda(lens), temperatures=None if temps is None else cuda(temps),
                            uniforms=None if u is None else cuda(u))
    path, counts, follow, near = ref.verify_ref(logits.double().cpu().numpy(), tokens, parents, lens, temps, u)
    clear = near > NEAR
    assert clear.mean() > 0.9 or not whole
    for got, want in zip(out, (path, counts, follow)):
        assert got.dtype == torch.int32
        assert np.array_equal(got.cpu().numpy()[clear], want[clear])
    return out


SHAPES = [(1, 1, 1), (3, 2, 2), (5, 7, 63), (4, 64, 1000), (2, 65, 257), (3, 130, 300), (2, 256, 70), (6, 9, 8193), (2, 5, 32000),
          (1, 3, 128256), (2, 3, 70001)]


@gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("b,t,v", SHAPES)
def test_greedy(dtype, b, t, v):
    rng = rng_of(v + t)
    check(*make(rng, b, t, v, dtype))


@gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("b,t,v", SHAPES)
def test_sampled(dtype, b, t, v):
    rng = rng_of(v + 2 * t)
    logits, tokens, parents, lens = make(rng, b, t, v, dtype)
    for _ in range(3):
        temps = rng.choice([0.3, 0.8, 1.0, 1.7], b).astype(np.float32)
        check(logits, tokens, parents, lens, temps, rng.random((b, t)).astype(np.float32), whole=False)


@gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_many_logits_are_read_by_path(dtype):
    """More logits than are read beforehand: the walk reads its rows itself."""
    rng = rng_of(4)
    b, t, v = 40, 24, 32003                    # rows start at any multiple of 2 or 4 bytes
    logits, tokens, parents, lens = make(rng, b, t, v, dtype)
    check(logits, tokens, parents, lens)
    temps = np.where(np.arange(b) % 3 == 0, 0.0, 0.7).astype(np.float32)
    check(logits, tokens, parents, lens, temps, rng.random((b, t)).astype(np.float32))


@gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_many_sequences_are_read_by_path(dtype):
    """So many short rows that the walk reads its own, greedy ones too; bf16 logits tie often."""
    rng = rng_of(14)
    b, t, v = 9000, 9, 100
    logits, tokens, parents, lens = make(rng, b, t, v, dtype)
    check(logits, tokens, parents, lens)
    temps = np.where(np.arange(b) % 2 == 0, 0.0, 0.7).astype(np.float32)
    check(logits, tokens, parents, lens, temps, rng.random((b, t)).astype(np.float32))


@gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("v", [60, 9000])
def test_long_greedy_paths_past_likely_siblings(dtype, v):
    """Paths of up to 128 nodes, whose every node has siblings of the same logit (a higher token, or the same one later), of a
    higher logit than other children's but no maximum, outside the vocabulary, or with NaN."""
    rng = rng_of(v + 15)
    b, t = 5, 256
    x = rng.standard_normal((b, t, v)) * 0.5
    tokens, parents = rng.integers(0, v, (b, t)).astype(np.int32), np.zeros((b, t), np.int32)
    parents[:, 0] = -1
    for i in range(b):
        end = 0                                             # of the path
        for j in range(1, t):
            parents[i, j] = end
            kind = rng.integers(0, 5)
            if j % 2 == 0 or kind == 0:                     # the path goes on (to this node, or to an earlier one of its kind)
                best = int(rng.integers(0, v - 1))
                x[i, end, best] = 4.0
                tokens[i, j] = best
                end = j
                continue
            parents[i, j] = rng.integers(0, j) if kind == 1 else end
            up, best = parents[i, j], int(x[i, parents[i, j]].argmax())
            if kind == 2:
                tokens[i, j] = v + 3
            elif kind == 3:
                x[i, up, min(best + 1, v - 1)] = x[i, up, best]
                tokens[i, j] = min(best + 1, v - 1)
            elif kind == 4:
                tokens[i, j] = best
    x[2, 60:, 5] = np.nan
    x[3, 100:, 7] = np.inf
    logits = torch.from_numpy(x).to("cuda", DTYPES[dtype])
    out = check(logits, tokens, parents, np.array([t, t - 1, t, t, 40], np.int32))
    assert int(out.counts.max()) > 16                       # more than any group of work-groups takes at a time


@gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("rows", [0, 60])
def test_ties_go_to_the_lowest_index(dtype, rows):
    """Equal maxima at every distance, -0 beside +0, siblings of one token."""
    rng = rng_of(5)
    b, t, v = 8 + rows, 12, 40000
    x = np.zeros((b, t, v))
    for i in range(b):
        for j in range(t):
            x[i, j, rng.integers(0, v, 5)] = 3.0
            if j % 3 == 0:
                x[i, j] = -np.abs(x[i, j])     # the maxima are 0, some of them -0
    logits = torch.from_numpy(x).to("cuda", DTYPES[dtype])
    best = x.argmax(2)
    parents = np.repeat(np.array([[-1, 0, 0, 0, 1, 2, 3, 4, 4, 5, 5, 6]], np.int32), b, 0)
    tokens = rng.integers(0, v, (b, t)).astype(np.int32)
    for i in range(b):
        for j in range(1, t):
            if rng.random() < 0.7:
                tokens[i, j] = best[i, parents[i, j]]
    check(logits, tokens, parents, np.full(b, t, np.int32))


@gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_rows_without_a_verdict(dtype):
    """NaN anywhere, nothing above -inf, and for a draw +inf: the path ends there and the next token is -1."""
    rng = rng_of(6)
    b, t, v = 9, 6, 5000
    logits, tokens, parents, lens = make(rng, b, t, v, dtype, hits=0.0)
    parents[:] = np.arange(-1, t - 1)
    lens[:] = t
    for i in range(b):
        for j in range(t - 1):
            logits[i, j, int(tokens[i, j + 1])] = 60.0             # the whole chain would be accepted
    logits[1, 2, 4999] = float("nan")
    logits[2, 0, 0] = -float("nan")
    logits[3, 3] = -float("inf")
    logits[4, 1, int(tokens[4, 2])] = float("inf")
    logits[5, :, 100:] = -float("inf")
    tokens[5] = np.arange(t)
    logits[6, 5] = float("nan")
    out = check(logits, tokens, parents, lens)
    assert out.counts.tolist()[1:5] == [3, 1, 4, 6] and out.next_tokens.tolist()[1:4] == [-1, -1, -1]
    temps = np.full(b, 0.9, np.float32)
    out = check(logits, tokens, parents, lens, temps, rng.random((b, t)).astype(np.float32))
    assert out.counts.tolist()[1:5] == [3, 1, 4, 2] and out.next_tokens.tolist()[1:5] == [-1] * 4


@gpu
def test_tokens_outside_the_vocabulary_and_odd_trees():
    """They are never taken; parents that are no lower index, and empty trees."""
    rng = rng_of(7)
    logits, tokens, parents, lens = make(rng, 12, 30, 500, "float32")
    tokens[:, 3::4] = rng.choice([-1, 500, 2 ** 31 - 1, -2 ** 31], tokens[:, 3::4].shape)
    lens[1:4] = 0, -5, 99
    check(logits, tokens, parents, lens)
    out = check(logits, tokens, parents, lens, np.ones(12, np.float32), rng.random((12, 30)).astype(np.float32))
    assert out.counts[1] == 0 and out.next_tokens[1] == -1 and (out.path[1] == -1).all()


@gpu
@pytest.mark.parametrize("rows", [0, 60])
def test_draws_next_to_a_child_s_bound(rows):
    """u on both sides of a child's bound, closer than fp32 sums can tell."""
    rng = rng_of(8)
    b, t, v = 16 + rows, 4, 40000
    parents = np.repeat(np.array([[-1, 0, 0, 0]], np.int32), b, 0)
    tokens = np.stack([rng.choice(v, t, replace=False) for _ in range(b)]).astype(np.int32)
    x = rng.standard_normal((b, t, v)) * 2
    for j in (1, 2, 3):
        x[np.arange(b), 0, tokens[:, j]] = 13.0
    logits = torch.from_numpy(x).float().cuda()
    y = logits.double().cpu().numpy()[:, 0]
    p = np.exp(y - y.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    c = np.cumsum(p[np.arange(b)[:, None], tokens[:, 1:]], 1)
    u = np.zeros((b, t), np.float32)
    u[:, 0] = c[np.arange(b), np.arange(b) % 3].astype(np.float32)
    for step in (-2, -1, 0, 1, 2):
        near = u.copy()
        near[:, 0] += np.float32(step * 2.0 ** -24)
        check(logits, tokens, parents, np.full(b, t, np.int32), np.ones(b, np.float32), near, whole=False)


@gpu
def test_children_that_have_nearly_all_of_it():
    """The rest of the vocabulary is summed for itself: it keeps its digits beside a child of 1 - 1e-6."""
    rng = rng_of(9)
    b, t, v = 6, 2, 30000
    logits = torch.from_numpy(rng.standard_normal((b, t, v))).float().cuda()
    tokens = rng.integers(0, v, (b, t)).astype(np.int32)
    for i in range(b):
        logits[i, 0, int(tokens[i, 1])] = 25.0
    u = np.full((b, t), 1 - 2.0 ** -23, np.float32)
    u[:, 0] -= np.arange(b).astype(np.float32) * 2.0 ** -22
    check(logits, tokens, np.repeat(np.array([[-1, 0]], np.int32), b, 0), np.full(b, 2, np.int32), np.ones(b, np.float32), u,
          whole=False)
    logits[:, 0] = -float("inf")                       # the child alone
    for i in range(b):
        logits[i, 0, int(tokens[i, 1])] = 0.0
    out = check(logits, tokens, np.repeat(np.array([[-1, 0]], np.int32), b, 0), np.full(b, 2, np.int32),
                np.ones(b, np.float32), u, whole=False)
    assert out.counts.tolist() == [2] * b


@gpu
def test_draws_follow_the_distribution():
    """Child or not, a token is drawn with its probability: 2^16 draws of five tokens, two of them children."""
    from tinyvllm_amd.sampling import verify_draft_tree
    n = 1 << 12
    p = np.array([0.1, 0.3, 0.05, 0.35, 0.2])
    logits = torch.from_numpy(np.log(p)).float().cuda().expand(n, 3, 5).contiguous()
    tokens = cuda(np.repeat(np.array([[0, 3, 0]], np.int32), n, 0))
    parents = cuda(np.repeat(np.array([[-1, 0, 0]], np.int32), n, 0))
    lens, temps = torch.full((n,), 3, dtype=torch.int32, device="cuda"), torch.ones(n, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(1)
    seen = torch.zeros(5, dtype=torch.int64, device="cuda")
    for _ in range(16):
        out = verify_draft_tree(logits, tokens, parents, lens, temperatures=temps,
                                uniforms=torch.rand((n, 3), generator=gen, device="cuda"))
        first = torch.where(out.counts > 1, tokens.gather(1, out.path[:, 1:2].clamp_min(0).long())[:, 0], out.next_tokens)
        seen += torch.bincount(first.long(), minlength=5)
    got = seen.double().cpu().numpy() / (16 * n)
    # five standard deviations of a share
    assert np.all(np.abs(got - p) < 5 * np.sqrt(p * (1 - p) / (16 * n)))


@gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_small_and_odd_temperatures(dtype):
    """Below 2^-126 greedy; a tiny one is nearly so; a large one flattens; logits far from 0."""
    rng = rng_of(10)
    logits, tokens, parents, lens = make(rng, 8, 9, 3000, dtype)
    temps = np.array([0.0, -1.0, 1e-40, 1e-30, 1e-3, 50.0, np.nan, 1e6], np.float32)
    u = rng.random((8, 9)).astype(np.float32)
    check(logits, tokens, parents, lens, temps, u)
    if dtype != "float16":
        check(logits + 4096, tokens, parents, lens, temps, u, whole=False)


@gpu
def test_strided_rows():
    """Rows of a wider buffer, not at multiples of 16 bytes."""
    rng = rng_of(11)
    logits, tokens, parents, lens = make(rng, 3, 6, 1001, "bfloat16")
    wide = torch.full((3, 6, 1007), float("nan"), dtype=torch.bfloat16, device="cuda")
    wide[:, :, 3:1004] = logits
    u, temps = rng.random((3, 6)).astype(np.float32), np.ones(3, np.float32)
    check(wide[:, :, 3:1004], tokens, parents, lens, temps, u)
    check(wide[:, :, 3:1004], tokens, parents, lens)


@gpu
@pytest.mark.parametrize("rows", [2, 48])
def test_in_a_graph(rows):
    """Replays follow their inputs, with eager work between them; both ways of reading rows."""
    from tinyvllm_amd.sampling import verify_draft_tree
    rng = rng_of(12)
    t, v = 12, 32000
    first = make(rng, rows, t, v, "float32")
    u, temps = rng.random((rows, t)).astype(np.float32), np.where(np.arange(rows) % 2, 0.8, 0.0).astype(np.float32)
    bufs = [first[0].clone(), *(cuda(x) for x in (*first[1:], temps, u))]
    verify_draft_tree(*bufs[:4], temperatures=bufs[4], uniforms=bufs[5])
    torch.cuda.synchronize()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = verify_draft_tree(*bufs[:4], temperatures=bufs[4], uniforms=bufs[5])
    for step in range(3):
        new = make(rng, rows, t, v, "float32")
        u = rng.random((rows, t)).astype(np.float32)
        for buf, x in zip(bufs, (new[0], *(cuda(x) for x in (*new[1:], temps, u)))):
            buf.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        want = check(*new, temps, u, whole=False)
        for a, b in zip(out, want):
            assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("case", range(case_count(12)))
def test_random_verdicts(case):
    rng = rng_of(case_seed(5100) + case)
    b, t = int(rng.integers(1, 30)), int(rng.integers(1, 40))
    v = int(np.exp(rng.uniform(0, np.log(20000))))
    logits, tokens, parents, lens = make(rng, b, t, v, str(rng.choice(sorted(DTYPES))))
    check(logits, tokens, parents, lens)
    check(logits, tokens, parents, lens, rng.uniform(0, 2, b).astype(np.float32), rng.random((b, t)).astype(np.float32),
          whole=False)
