"""The 8-bit cache at the edges of its number range and of its callers' contracts."""

import pytest
import torch

from tests.test_fp8_cache import DTYPES, gpu, make_cache, rng_of
from tests.test_fp8_prefill import check_chunk, chunk_case, run_chunk


@gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_largest_finite_elements_are_read_back_finite(dtype):
    """The dtype's largest number is rounded up to a power of two in e4m3, which the dtype does not hold."""
    big = torch.finfo(DTYPES[dtype]).max
    cache = make_cache(2, 16, 2, 64, dtype)
    x = torch.full((18, 2, 64), big, device="cuda", dtype=DTYPES[dtype])
    x[3, 0, 5] = -big
    x[4, 1, 7] = float("nan")
    cache.write_kv_slots(0, torch.arange(18, dtype=torch.int32, device="cuda"), x, -x)
    k, v = cache.read_kv_blocks(0, [0, 1], 18)
    for got, want in ((k, x), (v, -x)):
        nan = torch.isnan(want)
        assert torch.equal(torch.isnan(got), nan) and torch.equal(got[~nan], want[~nan])


@gpu
@pytest.mark.parametrize("bs", [16, 5])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_chunk_rows_do_not_see_huge_elements_that_they_do_not_attend(bs, d):
    """K and V of the largest bf16 magnitude at one position: the rows before it are what they are without it."""
    rng = rng_of(80)
    n, start, hq, hkv = 100, 30, 4, 2
    cache, held, q, table = chunk_case(rng, n, start, hq, hkv, d, bs, "bfloat16")
    at = start + 60
    blk, row = int(table[at // bs]), at % bs
    k8, v8, ks, vs = held
    for c, s, plain, scale in ((cache.k_cache[0], cache.k_scale[0], k8, ks), (cache.v_cache[0], cache.v_scale[0], v8, vs)):
        c[blk, 0] = torch.zeros((bs, d), device="cuda").to(torch.float8_e4m3fn)
        c[blk, 0, row] = torch.full((d,), 256.0, device="cuda").to(torch.float8_e4m3fn)
        s[blk, 0] = 2.0 ** 120
        plain[blk, 0] = 0.0
        scale[blk, 0] = 1.0
    got = run_chunk(cache, q, table, start)
    assert int((~torch.isfinite(got[0, :60])).sum()) == 0
    check_chunk(got, held, q, table, start, "bfloat16", rows=slice(0, 60))
    assert int((~torch.isfinite(got[0, :, 2:])).sum()) == 0              # the other KV head's
