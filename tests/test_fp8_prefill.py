"""Attention of a prompt's chunk over the 8-bit paged cache."""

import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import fp8_cache as ref
from tests.fp8_tolerance import rounded_weights_bound
from tests.random_cases import case_count, case_seed
from tests.test_fp8_cache import DTYPES, fill, gpu, make_cache, rng_of


def test_entry_point_validates_on_the_host():
    from tinyvllm_amd import _lib
    lib, p = _lib.load(), ctypes.c_void_p(256)
    base = [p] * 7 + [8, 16, 4, 0, 8, 2, 64, 512, 512, 1, 0.1, 1, 1, None, 0, None]

    def call(**kw):
        a = list(base)
        for i, v in kw.items():
            a[int(i[1:])] = v
        return lib.tv_flash_prefill_paged_fp8(*a)

    assert call(_1=None) == _lib.TV_EINVAL and b"null pointer" in lib.tv_last_error()
    assert call(_4=None) == _lib.TV_EINVAL and b"null pointer" in lib.tv_last_error()
    assert call(_9=0) == _lib.TV_EINVAL and b"bad sizes" in lib.tv_last_error()
    assert call(_10=-1) == _lib.TV_EINVAL and b"bad sizes" in lib.tv_last_error()
    assert call(_10=1 << 30) == _lib.TV_EINVAL
    assert call(_11=7) == _lib.TV_EINVAL and b"head counts" in lib.tv_last_error()
    assert call(_13=80) == _lib.TV_EUNSUPPORTED
    assert call(_14=511) == _lib.TV_EINVAL and b"stride" in lib.tv_last_error()
    assert call(_14=516) == _lib.TV_EINVAL and b"aligned" in lib.tv_last_error()
    assert call(_18=0, _19=0) == _lib.TV_EUNSUPPORTED and b"fp16 / bf16" in lib.tv_last_error()
    assert call(_19=2) == _lib.TV_EINVAL and b"out_dtype" in lib.tv_last_error()
    assert call(_20=ctypes.c_void_p(260), _21=1 << 30) == _lib.TV_EINVAL and b"workspace" in lib.tv_last_error()
    assert lib.tv_flash_prefill_paged_fp8_workspace_bytes(0, 0, 8, 2, 64) == 0


def chunk_case(rng, n, start, hq, hkv, d, bs, dtype, scales=1.0):
    cols = -(-(start + n) // bs)
    nb = cols + 3
    table = rng.permutation(nb)[:cols].astype(np.int32)
    cache = make_cache(nb, bs, hkv, d, dtype)
    held = fill(cache, rng)
    q = torch.from_numpy(rng.standard_normal((1, n, hq, d)) * scales).to("cuda", DTYPES[dtype])
    return cache, held, q, table


def run_chunk(cache, q, table, start, causal=True, **kw):
    from tinyvllm_amd.attention import flash_prefill_paged_fp8
    return flash_prefill_paged_fp8(q, cache.k_cache[0], cache.v_cache[0], cache.k_scale[0], cache.v_scale[0],
                                   torch.from_numpy(table).cuda(), start, causal, **kw)


def check_chunk(got, held, q, table, start, dtype, causal=True, rows=None, out_dtype=None):
    k8, v8, ks, vs = held
    n, d = q.shape[1], q.shape[3]
    k, v = ref.rows_ref(k8, ks, table, start + n), ref.rows_ref(v8, vs, table, start + n)
    want, bound, dev = ref.attend_ref(q[0].double().cpu().numpy(), k, v, start, 1 / math.sqrt(d), causal, spread=True)
    tol = rounded_weights_bound(want, bound, dev, float(np.abs(v).max()), start + n, d, dtype, out_dtype or dtype)
    diff = np.abs(got[0].double().cpu().numpy() - want)
    if rows is not None:
        diff, tol = diff[rows], tol[rows]
    assert np.all(diff <= tol), (float(np.nanmax(diff)), float(np.nanmax(diff / tol)))


@gpu
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (8, 1, 64), (3, 3, 64), (10, 2, 128), (2, 1, 256), (33, 1, 64)])
@pytest.mark.parametrize("n,start,bs", [(1, 0, 16), (1, 70, 16), (17, 0, 16), (64, 64, 32), (37, 300, 16), (130, 3, 5),
                                        (65, 63, 48)])
def test_chunk_shapes(dtype, hq, hkv, d, n, start, bs):
    """One row to several tiles, with and without a prefix; row tiles that end inside a position's heads."""
    rng = rng_of(31)
    cache, held, q, table = chunk_case(rng, n, start, hq, hkv, d, bs, dtype)
    got = run_chunk(cache, q, table, start)
    assert got.shape == q.shape and got.dtype == DTYPES[dtype]
    check_chunk(got, held, q, table, start, dtype)


@gpu
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_chunk_without_mask_and_in_fp32(dtype):
    rng = rng_of(32)
    cache, held, q, table = chunk_case(rng, 70, 200, 8, 2, 128, 16, dtype)
    check_chunk(run_chunk(cache, q, table, 200, False), held, q, table, 200, dtype, causal=False)
    got = run_chunk(cache, q, table, 200, out_dtype=torch.float32)
    assert got.dtype == torch.float32
    check_chunk(got, held, q, table, 200, dtype, out_dtype="float32")


@gpu
def test_chunk_split_and_unsplit_agree():
    """A few rows over a long prefix: split keys with a workspace, one pass without; rows that are a
    projection's."""
    from tinyvllm_amd import _lib
    lib = _lib.load()
    rng = rng_of(33)
    n, start, hq, hkv, d, bs = 9, 2100, 8, 2, 64, 16
    cache, held, q, table = chunk_case(rng, n, start, hq, hkv, d, bs, "bfloat16")
    wide = torch.zeros((n, hq * d + 64), dtype=torch.bfloat16, device="cuda")
    wide[:, :hq * d] = q[0].reshape(n, -1)
    view = torch.as_strided(wide, (n, hq, d), (wide.stride(0), d, 1))
    assert lib.tv_flash_prefill_paged_fp8_workspace_bytes(n, start, hq, hkv, d) > 0
    got = run_chunk(cache, view, table, start)
    check_chunk(got, held, q, table, start, "bfloat16")
    out = torch.full((1, n, hq, d), float("nan"), dtype=torch.bfloat16, device="cuda")
    rc = lib.tv_flash_prefill_paged_fp8(
        out.data_ptr(), q.data_ptr(), cache.k_cache[0].data_ptr(), cache.v_cache[0].data_ptr(),
        cache.k_scale[0].data_ptr(), cache.v_scale[0].data_ptr(), torch.from_numpy(table).cuda().data_ptr(),
        cache.num_blocks, bs, n, start, hq, hkv, d, hq * d, hq * d, 1, 1 / math.sqrt(d), _lib.TV_BF16, _lib.TV_BF16,
        None, 0, _lib.stream_ptr(q.device))
    _lib.check(rc, "unsplit")
    check_chunk(out, held, q, table, start, "bfloat16")


@gpu
def test_chunk_peaked_softmax():
    rng = rng_of(34)
    for dtype in ("float16", "bfloat16"):
        cache, held, q, table = chunk_case(rng, 40, 500, 4, 2, 128, 16, dtype, scales=16)
        check_chunk(run_chunk(cache, q, table, 500), held, q, table, 500, dtype)


@gpu
def test_chunk_fp16_values_near_its_largest():
    """Values that round past 65504 are limited to it; scales of any size enter exactly."""
    rng = rng_of(35)
    cache, held, q, table = chunk_case(rng, 20, 44, 4, 2, 64, 16, "float16")
    k8, v8, ks, vs = held
    vs[:] = 256.0
    cache.v_scale[0].fill_(256.0)
    v8[:] = np.clip(v8, -256, 256)
    v8[:, :, 3, :] = 256.0                       # 65536
    cache.v_cache[0].copy_(torch.from_numpy(v8.astype(np.float32)).cuda().to(torch.float8_e4m3fn))
    got = run_chunk(cache, q, table, 44, out_dtype=torch.float32)
    limited = np.clip(v8 * 256.0, -65504, 65504) / 256.0
    check_chunk(got, (k8, limited, ks, vs), q, table, 44, "float16", out_dtype="float32")


@gpu
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("bs", [16, 10])
def test_chunk_nan_and_bad_blocks_stay_with_the_rows_that_attend_them(dtype, bs):
    rng = rng_of(36)
    n, start, hq, hkv, d = 150, 90, 4, 2, 64
    cache, held, q, table = chunk_case(rng, n, start, hq, hkv, d, bs, dtype)
    last = table[(start + n - 1) // bs]
    for c in (cache.k_cache[0], cache.v_cache[0]):                # past the end of the sequence
        c.view(torch.uint8)[int(last), :, (start + n - 1) % bs + 1:] = 0x7F
    cache.v_cache[0].view(torch.uint8)[int(table[(start + 60) // bs]), 0, (start + 60) % bs, 7] = 0xFF
    cache.k_cache[0].view(torch.uint8)[int(table[(start + 100) // bs]), 1, (start + 100) % bs, 63] = 0x7F
    got = run_chunk(cache, q, table, start)
    bad = torch.isnan(got[0]).all(-1)
    fine = torch.isfinite(got[0]).all(-1)
    assert fine[:60, :2].all() and bad[60:, :2].all()
    assert fine[:100, 2:].all() and bad[100:, 2:].all()
    check_chunk(got, held, q, table, start, dtype, rows=slice(0, 60))
    broken = table.copy()
    col = (start + 120) // bs
    broken[col] = -1
    got = run_chunk(cache, q, broken, start)
    first = max(0, col * bs - start)
    assert torch.isnan(got[0, first:]).all() and torch.isfinite(got[0, :60]).all()
    broken[0] = cache.num_blocks
    assert torch.isnan(run_chunk(cache, q, broken, start)).all()


@gpu
def test_chunk_in_a_graph():
    """Split keys and their merge, replayed between eager calls on other inputs."""
    rng = rng_of(37)
    start, n = 1500, 12
    cache, held, q, table = chunk_case(rng, n, start, 8, 2, 128, 16, "float16")
    run_chunk(cache, q, table, start)
    from tinyvllm_amd.attention import flash_prefill_paged_fp8
    tb = torch.from_numpy(table).cuda()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = flash_prefill_paged_fp8(q, cache.k_cache[0], cache.v_cache[0], cache.k_scale[0], cache.v_scale[0], tb, start)
    for step in range(3):
        q.copy_(torch.from_numpy(rng.standard_normal(tuple(q.shape))).to("cuda", torch.float16))
        g.replay()
        eager = run_chunk(cache, q, table, start)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        check_chunk(out, held, q, table, start, "float16")


@gpu
def test_chunk_random_shapes():
    rng = rng_of(case_seed(50))
    for i in range(case_count(12)):
        dtype = ["float16", "bfloat16"][rng.integers(2)]
        d = int(rng.choice([64, 128, 256]))
        hkv = int(rng.integers(1, 4))
        hq = hkv * int(rng.integers(1, 9))
        bs = int(rng.choice([16, 16, 32, 1, 7, 24, 100]))
        n, start = int(rng.integers(1, 200)), int(rng.choice([0, rng.integers(1, 900)]))
        print("chunk", i, dtype, d, hkv, hq, bs, n, start, flush=True)
        cache, held, q, table = chunk_case(rng, n, start, hq, hkv, d, bs, dtype)
        check_chunk(run_chunk(cache, q, table, start), held, q, table, start, dtype)
