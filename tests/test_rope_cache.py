"""Rotation on the way into the paged cache."""

import ctypes

import numpy as np
import pytest
import torch

from oracle.draft_tree import rope_ref
from tests.fp8_tolerance import HALF_STEP
from tests.random_cases import case_count, case_seed
from tests.test_draft_tree import DTYPES, cuda, gpu, rng_of


def table_of(rows, dim, theta=10000.0):
    angle = np.arange(rows)[:, None] * theta ** (-np.arange(0, dim, 2) / dim)
    return np.stack([np.cos(angle), np.sin(angle)], 2).astype(np.float32)


def tolerance(want, x, dim, pairs, dtype):
    """Both products and their sum are rounded to fp32 (2^-24 each, of at most |a| + |b|), then once to the dtype."""
    half = dim // 2
    size = np.zeros_like(want)
    if pairs == "adjacent":
        both = np.abs(x[..., 0:dim:2]) + np.abs(x[..., 1:dim:2])
        size[..., 0:dim:2] = size[..., 1:dim:2] = both
    else:
        both = np.abs(x[..., :half]) + np.abs(x[..., half:dim])
        size[..., :half] = size[..., half:dim] = both
    off = 2.0 ** -23 * size
    return HALF_STEP[dtype] * (np.abs(want) + off) * (np.arange(want.shape[-1]) < dim) + off + \
        (2.0 ** -25 if dtype == "float16" else 0.0) * (size > 0)


def check(rng, dtype, n, hq, hkv, d, dim, pairs, block=16, extra=0, slots=None, positions=None, in_place=False, shift=0):
    from tinyvllm_amd.kv_cache import rope_and_cache
    t = DTYPES[dtype]
    nb = -(-n // block) + 3
    width = (hq + 2 * hkv) * d + extra
    buf = torch.from_numpy(rng.standard_normal(n * width + shift)).to("cuda", t)[shift:].view(n, width)
    q, k, v = (x.unflatten(1, (-1, d)) for x in buf[:, :width - extra].split([hq * d, hkv * d, hkv * d], 1))
    caches = [torch.from_numpy(rng.standard_normal((nb, block, hkv, d))).to("cuda", t) for _ in range(2)]
    rope = table_of(100, dim)
    positions = rng.integers(0, 100, n).astype(np.int32) if positions is None else positions
    slots = rng.permutation(nb * block)[:n].astype(np.int32) if slots is None else slots
    xq, xk, xv = (x.double().cpu().numpy() for x in (q, k, v))
    old = [c.double().cpu().numpy() for c in caches]
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = rope_and_cache(*caches, q, k, v, cuda(slots), cuda(positions), cuda(rope), pairs=pairs,
                         out=q if in_place else None, err_count=err)
    known = (positions >= 0) & (positions < 100)
    write = known & (slots >= 0) & (slots < nb * block)
    at = np.where(known, positions, 0)
    got = out.double().cpu().numpy()
    want = rope_ref(xq, at, rope, pairs)
    assert np.all(np.abs(got - want)[known] <= tolerance(want, xq, dim, pairs, dtype)[known])
    assert np.isnan(got[~known]).all()
    assert int(err) == int((~known | (slots >= nb * block)).sum())
    wk, wv, tol = old[0].reshape(-1, hkv, d), old[1].reshape(-1, hkv, d), np.zeros((nb * block, hkv, d))
    turned = rope_ref(xk, at, rope, pairs)
    for i in np.flatnonzero(write):
        wk[slots[i]], wv[slots[i]] = turned[i], xv[i]
        tol[slots[i]] = tolerance(turned[i], xk[i], dim, pairs, dtype)
    assert np.all(np.abs(caches[0].double().cpu().numpy().reshape(wk.shape) - wk) <= tol)
    assert np.array_equal(caches[1].double().cpu().numpy().reshape(wv.shape), wv)
    return out


def test_oracle_turns_a_pair():
    x = np.array([[[1.0, 0.0, 7.0, 2.0]]])
    rope = np.array([[[0.0, 1.0]]], np.float32)                   # a quarter turn
    assert rope_ref(x, [0], rope, "adjacent").tolist() == [[[0.0, 1.0, 7.0, 2.0]]]
    assert rope_ref(x, [0], np.tile(rope, (1, 2, 1)), "halves").tolist() == [[[-7.0, -2.0, 1.0, 0.0]]]


def test_entry_point_validates_on_the_host():
    from tinyvllm_amd import _lib
    lib, p = _lib.load(), ctypes.c_void_p(256)
    base = [p] * 9 + [100, 64, 0, 4, 8, 2, 64, 16, 20, 512, 512, 128, 128, 1, None, None]

    def call(**kw):
        a = list(base)
        for i, v in kw.items():
            a[int(i[1:])] = v
        return lib.tv_rope_and_cache(*a)

    for i in range(9):
        assert call(**{f"_{i}": None}) == _lib.TV_EINVAL and b"null pointer" in lib.tv_last_error()
    for i in (0, 3, 5):
        assert call(**{f"_{i}": ctypes.c_void_p(257)}) == _lib.TV_EINVAL and b"misaligned" in lib.tv_last_error()
    assert call(_8=ctypes.c_void_p(260)) == _lib.TV_EINVAL and b"misaligned" in lib.tv_last_error()
    for rope_len, dim in ((0, 64), (100, 0), (100, 63), (100, 66)):
        assert call(_9=rope_len, _10=dim) == _lib.TV_EINVAL and b"rope table" in lib.tv_last_error()
    assert call(_12=-1) == _lib.TV_EINVAL and call(_12=0) == _lib.TV_OK
    assert call(_12=1 << 24) == _lib.TV_EINVAL and b"grid" in lib.tv_last_error()
    for i in (13, 14, 15):
        assert call(**{f"_{i}": 0}) == _lib.TV_EINVAL and b"heads" in lib.tv_last_error()
    for i in (18, 19, 20, 21):
        assert call(**{f"_{i}": 127}) == _lib.TV_EINVAL and b"stride" in lib.tv_last_error()
    assert call(_22=3) == _lib.TV_EINVAL and b"dtype" in lib.tv_last_error()
    assert call(_10=62, _15=63) == _lib.TV_EUNSUPPORTED and b"adjacent" in lib.tv_last_error()


def test_python_refuses_tensors_on_the_cpu():
    from tinyvllm_amd.kv_cache import rope_and_cache
    c, x = torch.zeros((4, 16, 2, 64)), torch.zeros((3, 2, 64))
    i = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="HIP device"):
        rope_and_cache(c, c, x, x, x, i, i, torch.zeros((9, 32, 2)))


@gpu
def test_python_refusals_on_the_gpu():
    from tinyvllm_amd.kv_cache import FP8KVCache, rope_and_cache
    c, x = torch.zeros((4, 16, 2, 64), device="cuda"), torch.zeros((3, 2, 64), device="cuda")
    i = torch.zeros(3, dtype=torch.int32, device="cuda")
    r = torch.zeros((9, 32, 2), device="cuda")
    good = [c, c.clone(), x, x, x, i, i, r]
    for at, bad, what in ((1, c.half(), "share a dtype"), (1, c[:2], "one shape"), (0, c.transpose(1, 2), "dense"),
                          (2, x.half(), "share a dtype"), (2, x[:2], "same number"), (3, x[:, :1], "k must be"),
                          (4, x.transpose(1, 2).contiguous().transpose(1, 2), "contiguous"),
                          (3, x[:1].expand(3, 2, 64), "overlap"), (5, i[:2], "slot_mapping"), (6, i.long(), "positions"),
                          (5, i.cpu(), "cache's device"), (7, r.half(), "rope must"), (7, r[:, :, :1], "rope must"),
                          (7, r.new_zeros((9, 33, 2)), "fit"), (7, r[:0], "fit")):
        args = list(good)
        args[at] = bad
        with pytest.raises(ValueError, match=what):
            rope_and_cache(*args)
    with pytest.raises(ValueError, match="pairs"):
        rope_and_cache(*good, pairs="both")
    with pytest.raises(ValueError, match="like q"):
        rope_and_cache(*good, out=x[:2])
    with pytest.raises(ValueError, match="err_count"):
        rope_and_cache(*good, err_count=r)
    fp8 = FP8KVCache(1, 4, 16, 2, 64, "float32")
    with pytest.raises(ValueError):
        rope_and_cache(fp8.k_cache[0], fp8.v_cache[0], x, x, x, i, i, r)
    assert rope_and_cache(c, c.clone(), x[:0], x[:0], x[:0], i[:0], i[:0], r).shape == (0, 2, 64)


@gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("pairs", ["adjacent", "halves"])
@pytest.mark.parametrize("n,hq,hkv,d,dim", [(1, 32, 4, 64, 64), (37, 8, 2, 128, 128), (5, 3, 3, 64, 32), (3, 40, 8, 128, 64),
                                            (9, 2, 1, 256, 256), (4, 5, 1, 80, 80), (2, 3, 2, 10, 6), (600, 4, 2, 64, 64)])
def test_rotated_write(dtype, pairs, n, hq, hkv, d, dim):
    check(rng_of(n + d), dtype, n, hq, hkv, d, dim, pairs)


@gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("pairs", ["adjacent", "halves"])
def test_rows_of_a_wider_buffer(dtype, pairs):
    """Token strides that are, and are not, multiples of 16 bytes; a base that is not; in place."""
    check(rng_of(1), dtype, 11, 4, 2, 64, 64, pairs, extra=64)
    check(rng_of(2), dtype, 11, 4, 2, 64, 64, pairs, extra=3)
    check(rng_of(3), dtype, 11, 4, 2, 64, 64, pairs, shift=1)
    check(rng_of(4), dtype, 11, 4, 2, 64, 64, pairs, block=5, in_place=True)
    check(rng_of(5), dtype, 11, 4, 2, 64, 64, pairs, extra=1, in_place=True)


@gpu
def test_odd_heads_with_halves():
    check(rng_of(6), "bfloat16", 7, 3, 1, 65, 64, "halves")


@gpu
@pytest.mark.parametrize("pairs", ["adjacent", "halves"])
def test_padding_and_bad_tokens(pairs):
    """Negative slots are skipped; slots past the cache, and positions outside the table, are counted and not
    written, the latter's queries NaN."""
    slots = np.array([3, -1, 500, 7, -9, 2 ** 31 - 1, 12, 63], np.int32)
    positions = np.array([0, 99, 5, 100, -1, 50, -2 ** 31, 98], np.int32)
    check(rng_of(7), "float16", 8, 4, 2, 64, 64, pairs, slots=slots, positions=positions)


@gpu
def test_agrees_with_the_model_s_table_and_the_cache_s_write():
    """Llama.rope's table; without rotation (position 0) the cache's plain write, bit for bit."""
    from tinyvllm_amd.kv_cache import KVCache
    from tinyvllm_amd.llama import Llama, LlamaConfig
    model = Llama(LlamaConfig(dim=128, n_layers=1, n_heads=2, n_kv_heads=1, vocab_size=64, hidden_dim=96,
                              max_seq_len=32, dtype="float16"))
    rng = rng_of(8)
    a, b = (KVCache(1, 4, 16, 1, 64, "float16") for _ in range(2))
    q, k, v = (torch.from_numpy(rng.standard_normal((9, h, 64))).to("cuda", torch.float16) for h in (2, 1, 1))
    slots = cuda(rng.permutation(64)[:9].astype(np.int32))
    out = a.write_rope_slots(0, slots, torch.zeros(9, dtype=torch.int32, device="cuda"), model.rope, q, k, v)
    b.write_kv_slots(0, slots, k, v)
    assert torch.equal(a.k_cache[0], b.k_cache[0]) and torch.equal(a.v_cache[0], b.v_cache[0]) and torch.equal(out, q)
    pos = np.arange(40, 49).astype(np.int32)
    got = a.write_rope_slots(0, slots, cuda(pos), model.rope, q, k, v).double().cpu().numpy()
    x = q.double().cpu().numpy()
    want = rope_ref(x, pos, model.rope.cpu().numpy(), "adjacent")
    assert np.all(np.abs(got - want) <= tolerance(want, x, 64, "adjacent", "float16"))


@gpu
def test_on_another_stream_and_in_a_graph():
    from tinyvllm_amd.kv_cache import rope_and_cache
    rng = rng_of(9)
    q, k, v = (torch.from_numpy(rng.standard_normal((20, h, 64))).float().cuda() for h in (4, 2, 2))
    rope = cuda(table_of(64, 64))
    slots, positions = cuda(rng.permutation(64)[:20].astype(np.int32)), cuda(rng.integers(0, 64, 20).astype(np.int32))
    caches = [torch.zeros((4, 16, 2, 64), device="cuda") for _ in range(4)]
    want = rope_and_cache(*caches[:2], q, k, v, slots, positions, rope)
    torch.cuda.synchronize()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = rope_and_cache(*caches[2:], q, k, v, slots, positions, rope)
    for step in range(3):
        q.mul_(-1.0 if step else 1.0)
        k.add_(0.25 * step)
        want = rope_and_cache(*caches[:2], q, k, v, slots, positions, rope)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(caches[0], caches[2]) and torch.equal(caches[1], caches[3])


@gpu
@pytest.mark.parametrize("case", range(case_count(10)))
def test_random_rotated_writes(case):
    rng = rng_of(case_seed(1200) + case)
    d = int(rng.choice([16, 64, 96, 128, 256]))
    hkv = int(rng.integers(1, 9))
    check(rng, str(rng.choice(sorted(DTYPES))), int(rng.integers(1, 300)), hkv * int(rng.integers(1, 6)), hkv, d,
          2 * int(rng.integers(1, d // 2 + 1)), str(rng.choice(["adjacent", "halves"])), block=int(rng.integers(1, 40)),
          extra=int(rng.integers(0, 20)))
