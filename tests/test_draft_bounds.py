"""Sampled verdicts whose u lies next to a child's bound, where fp32 sums do not decide."""

import numpy as np
import pytest
import torch

from oracle import draft_tree as ref
from tests.test_draft_tree import DTYPES, cuda, gpu, rng_of
from tests.test_draft_verify import NEAR

NODES = 4                                    # live nodes of a tree: the root and three children


def trees(logits, rows):
    """A batch whose rows are read first, or by a walk: of `rows` rows, all but the first of a sequence unused."""
    b, v = logits.shape
    t = max(NODES, -(-rows // b))
    assert t <= 256
    x = torch.zeros((b, t, v), dtype=logits.dtype, device="cuda")
    x[:, 0] = logits
    return x


def rows_for_a_walk(v, dtype):
    """Rows of v logits that take longer to read than seven steps of a walk (5.2 GB/ms; 0.9 us and 36 ns for a KiB)."""
    row = v * DTYPES[dtype].itemsize
    return int((7 * (0.9 + row / 1024 * 0.036) - 4) * 5.2e6 / row) + 64


def bounds(logits, tokens, temp):
    """The children's cumulated probabilities after each, in fp64."""
    y = logits.double().cpu().numpy() / np.float64(temp)
    p = np.exp(y - y.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    return np.cumsum(p[np.arange(len(y))[:, None], tokens[:, 1:NODES]], 1)


def check(x, tokens, temp, u):
    from tinyvllm_amd.sampling import verify_draft_tree
    b, t, _ = x.shape
    parents = np.full((b, t), -1, np.int32)
    parents[:, 1:NODES] = 0
    lens, temps = np.full(b, NODES, np.int32), np.full(b, temp, np.float32)
    every = np.zeros((b, t), np.int32)
    every[:, :NODES] = tokens
    uniforms = np.zeros((b, t), np.float32)
    uniforms[:, 0] = u
    out = verify_draft_tree(x, cuda(every), cuda(parents), cuda(lens), temperatures=cuda(temps), uniforms=cuda(uniforms))
    path, counts, _, near = ref.verify_ref(x[:, :NODES].double().cpu().numpy(), tokens, parents[:, :NODES], lens, temps,
                                           uniforms[:, :NODES])
    clear = near > NEAR
    assert np.array_equal(out.path[:, 1].cpu().numpy()[clear], path[clear, 1])
    assert np.array_equal((out.counts > 1).cpu().numpy()[clear], (counts > 1)[clear])
    return clear


# u is a sum's distance from the bound: 2^-25 to 2^-12, on both sides of the margin of the fp32 sums
OFFSETS = np.array([s * 2.0 ** -k for k in range(12, 26) for s in (-1, 1)])


@gpu
@pytest.mark.parametrize("walk", [False, True])
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("v", [2003, 32000, 128256])
def test_the_fp32_sums_margin(v, dtype, walk):
    """Rows whose fp32 exponentials are all off in the same direction: one value, whose exponent is log2(v) below the
    maximum's, beside a child of about half the sum."""
    rng = rng_of(v)
    b, temp = len(OFFSETS), 0.7
    tokens = np.stack([rng.choice(v, NODES, replace=False) for _ in range(b)]).astype(np.int32)
    low = -np.log(v) * temp * rng.uniform(0.95, 1.05, (b, 1))
    logits = torch.from_numpy(np.broadcast_to(low, (b, v)).copy())
    logits[np.arange(b), tokens[:, 2]] = 0.0
    logits = logits.to("cuda", DTYPES[dtype])
    x = trees(logits, rows_for_a_walk(v, dtype) if walk else 0)
    c = bounds(logits, tokens, np.float32(temp))
    clear = 0
    for child in range(NODES - 1):
        clear += check(x, tokens, temp, np.clip(c[:, child] + OFFSETS, 0, 1 - 2.0 ** -24).astype(np.float32)).sum()
    assert clear > 2 * b


@gpu
@pytest.mark.parametrize("walk", [False, True])
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("v", [2, 5, 7, 9, 63, 517, 4099, 16384, 40001])
def test_the_fp64_sum_of_any_row(v, dtype, walk):
    """Rows at every alignment, shorter than a vector, with -inf among them: u is next to a bound in all of them."""
    rng = rng_of(3 * v + 1)
    b, nodes = 16, min(NODES, v)
    tokens = np.zeros((b, NODES), np.int32)
    tokens[:, 1:] = -1                                     # of two or three tokens the last nodes have none
    for i in range(b):
        tokens[i, 1:nodes] = rng.choice(v, nodes - 1, replace=False)
    x = rng.standard_normal((b, v)) * 2
    for j in range(1, nodes):
        x[np.arange(b), tokens[:, j]] = np.log(v) + rng.uniform(1, 2, b)
    x[rng.random((b, v)) < 0.1] = -np.inf
    x[:, tokens[0, 1]] = 9.0
    logits = torch.from_numpy(x).to("cuda", DTYPES[dtype])
    rows = rows_for_a_walk(v, dtype) if walk else 0
    batch = trees(logits, min(rows, 256 * b))
    y = logits.double().cpu().numpy()
    p = np.exp(y - y.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    have = np.where(tokens[:, 1:] >= 0, np.take_along_axis(p, np.maximum(tokens[:, 1:], 0), 1), 0)
    c = np.cumsum(have, 1)
    for child in range(nodes - 1):
        for offset in (-2.0 ** -22, 2.0 ** -22):
            check(batch, tokens, 1.0, np.clip(c[:, child] + offset, 0, 1 - 2.0 ** -24).astype(np.float32))


@gpu
@pytest.mark.parametrize("b,t,v,dtype", [(2, 32, 128256, "bfloat16"), (2, 8, 32000, "float32"), (64, 16, 128256, "bfloat16")])
def test_u_on_a_bound_is_no_stall(b, t, v, dtype):
    """The sum in fp64 takes its time, but not a multiple of the call's: up to 1.9 times the call where it was 4 to 12."""
    from tinyvllm_amd.sampling import verify_draft_tree
    torch.manual_seed(1)
    logits = (torch.randn((b, t, v), device="cuda") * 2).to(DTYPES[dtype])
    tokens = torch.randint(0, v, (b, t), device="cuda", dtype=torch.int32)
    parents = torch.zeros((b, t), device="cuda", dtype=torch.int32)
    parents[:, 0] = -1
    lens, temps = torch.full((b,), t, device="cuda", dtype=torch.int32), torch.ones(b, device="cuda")
    child = int(tokens[0, 1])
    logits[0, 0, child] = torch.logsumexp(logits[0, 0].double(), 0).to(logits.dtype)
    far = torch.full((b, t), 0.9, device="cuda")
    near = far.clone()
    near[0, 0] = torch.softmax(logits[0, 0].double(), 0)[child].float()

    def best_time(u):
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        graph = torch.cuda.CUDAGraph()
        verify_draft_tree(logits, tokens, parents, lens, temperatures=temps, uniforms=u)
        with torch.cuda.graph(graph):
            verify_draft_tree(logits, tokens, parents, lens, temperatures=temps, uniforms=u)
        times = []
        for _ in range(12):
            start.record()
            graph.replay()
            end.record()
            end.synchronize()
            times.append(start.elapsed_time(end))
        return min(times)

    assert best_time(near) < 3 * best_time(far)
