"""The 8-bit cache's kernels at sizes where they take another form: row tiles of 128 with two key groups."""

import math

import numpy as np
import pytest
import torch

from oracle import fp8_cache as ref
from tests.fp8_tolerance import rounded_weights_bound
from tests.test_fp8_cache import gpu, rng_of
from tests.test_fp8_prefill import chunk_case, run_chunk


def cus():
    return torch.cuda.get_device_properties(0).multi_processor_count


def check_rows_of_chunk(got, held, q, table, start, dtype, rows, causal=True, heads=slice(None), out_dtype=None):
    """Some rows of a chunk against float64."""
    k8, v8, ks, vs = held
    n, hq, d = q.shape[1:]
    hkv = k8.shape[1]
    k, v = ref.rows_ref(k8, ks, table, start + n), ref.rows_ref(v8, vs, table, start + n)
    vmax = float(np.nanmax(np.abs(v)))
    for i in rows:
        m = start + i + 1 if causal else start + n
        want, bound, dev = ref.attend_ref(q[0, i:i + 1].double().cpu().numpy(), k[:m], v[:m], m - 1, 1 / math.sqrt(d),
                                          spread=True)
        tol = rounded_weights_bound(want, bound, dev, vmax, m, d, dtype, out_dtype or dtype)
        diff = np.abs(got[0, i:i + 1].double().cpu().numpy() - want)
        assert np.all(diff[:, heads] <= tol[:, heads]), (i, float(np.nanmax(diff)), float(np.nanmax(diff / tol)))


def wide_case(rng, d, bs, dtype, n=901, start=37):
    """A chunk of 128-row work-groups: tiles of 128 rows on seven eighths of the CUs, none of its keys split."""
    from tinyvllm_amd import _lib
    hq, hkv = 32, 8
    assert -(-n * (hq // hkv) // 128) * hkv * 8 >= 7 * cus()
    assert _lib.load().tv_flash_prefill_paged_fp8_workspace_bytes(n, start, hq, hkv, d) == 0
    return chunk_case(rng, n, start, hq, hkv, d, bs, dtype)


@gpu
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("d,bs", [(64, 16), (64, 5), (128, 16), (128, 5), (128, 32)])
def test_chunk_of_128_row_tiles(dtype, d, bs):
    """28 whole tiles and one of 20 rows, after a prefix that ends inside a tile and a block."""
    rng = rng_of(90)
    cache, held, q, table = wide_case(rng, d, bs, dtype)
    rows = [0, 1, 15, 26, 27, 31, 32, 90, 91, 447, 448, 863, 864, 895, 896, 899, 900]
    got = run_chunk(cache, q, table, 37)
    assert int((~torch.isfinite(got)).sum()) == 0
    check_rows_of_chunk(got, held, q, table, 37, dtype, rows)
    assert torch.equal(got, run_chunk(cache, q, table, 37))
    full = run_chunk(cache, q, table, 37, False, out_dtype=torch.float32)
    check_rows_of_chunk(full, held, q, table, 37, dtype, rows[::4], causal=False, out_dtype="float32")


@gpu
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("d,bs", [(64, 16), (128, 16), (64, 10)])
def test_nan_and_bad_blocks_in_128_row_tiles(dtype, d, bs):
    """They stay with the rows and heads that attend them; what lies past the sequence's end is not seen."""
    rng = rng_of(91)
    n, start = 901, 37
    cache, held, q, table = wide_case(rng, d, bs, dtype)
    last = int(table[(start + n - 1) // bs])
    for c in (cache.k_cache[0], cache.v_cache[0]):
        c.view(torch.uint8)[last, :, (start + n - 1) % bs + 1:] = 0x7F
    for c, head, row, dim in ((cache.v_cache[0], 3, 500, 7), (cache.k_cache[0], 5, 700, d - 1)):
        c.view(torch.uint8)[int(table[(start + row) // bs]), head, (start + row) % bs, dim] = 0xFF
    got = run_chunk(cache, q, table, start)[0]
    want = torch.zeros((n, 32), dtype=torch.bool, device="cuda")
    want[500:, 12:16] = True
    want[700:, 20:24] = True
    nan = torch.isnan(got)
    assert torch.equal(nan.all(-1), want) and torch.equal(nan.any(-1), want)
    check_rows_of_chunk(got[None], held, q, table, start, dtype, [0, 480, 499])
    check_rows_of_chunk(got[None], held, q, table, start, dtype, [500, 699, 900], heads=slice(0, 12))
    broken = table.copy()
    col = (start + 800) // bs
    broken[col] = cache.num_blocks
    want[col * bs - start:] = True
    assert torch.equal(torch.isnan(run_chunk(cache, q, broken, start)[0]).all(-1), want)


@gpu
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("d", [64, 128])
def test_peaked_softmax_in_128_row_tiles(dtype, d):
    """Scores of hundreds: the two key groups' maxima lie far apart, and rise tile after tile."""
    rng = rng_of(92)
    cache, held, q, table = wide_case(rng, d, 16, dtype)
    q.mul_(16)
    check_rows_of_chunk(run_chunk(cache, q, table, 37), held, q, table, 37, dtype, [0, 30, 200, 511, 777, 900])
