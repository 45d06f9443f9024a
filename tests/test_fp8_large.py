"""The 8-bit cache's kernels at sizes where they take another form: row tiles of 128 with two key groups,
a longest-first batch, a merge of more than a thousand partitions, several heads for a wave of the write."""

import math

import numpy as np
import pytest
import torch

from oracle import fp8_cache as ref
from tests.fp8_tolerance import rounded_weights_bound
from tests.test_fp8_cache import DTYPES, check_decode, check_write, decode_case, fill, gpu, make_cache, rng_of, run_decode
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


@gpu
@pytest.mark.parametrize("dtype,d", [("float16", 64), ("bfloat16", 128), ("float32", 64)])
def test_decode_of_a_longest_first_batch(dtype, d):
    """More work-groups than two a CU run in the order of their lengths, which changes no result."""
    from tinyvllm_amd import _lib
    lib = _lib.load()
    rng = rng_of(93)
    b, hq, hkv, bs = 130, 16, 8, 16
    ctx = rng.integers(0, 400, b)
    ctx[[0, 7, 129]] = [0, 600, 1]
    assert b * hkv > 2 * cus()
    cache, held, q, tables, ctx = decode_case(rng, ctx, hq, hkv, d, bs, dtype)
    part = -(-tables.shape[1] * bs // 32) * 32
    assert lib.tv_paged_decode_fp8_workspace_bytes(b, hq, d, tables.shape[1], bs, part) > 0     # the order's
    got = run_decode(cache, q, tables, ctx, hq, hkv, d, bs, partition_size=part)
    assert torch.count_nonzero(got[torch.from_numpy(ctx == 0).cuda()]) == 0
    check_decode(got, held, q, tables, ctx, d, dtype)
    out = torch.full_like(q, float("nan"))
    tb, cx = torch.from_numpy(tables).cuda(), torch.from_numpy(ctx).cuda()
    code = _lib.dtype_code(q.dtype)
    _lib.check(lib.tv_paged_decode_fp8(
        out.data_ptr(), q.data_ptr(), cache.k_cache[0].data_ptr(), cache.v_cache[0].data_ptr(),
        cache.k_scale[0].data_ptr(), cache.v_scale[0].data_ptr(), tb.data_ptr(), cx.data_ptr(), b, hq, hkv, d, bs,
        cache.num_blocks, tables.shape[1], tables.shape[1], 1 / math.sqrt(d), code, code, part, None, 0,
        _lib.stream_ptr(q.device)), "batch order")
    assert torch.equal(out, got)


@gpu
@pytest.mark.parametrize("dtype,d", [("bfloat16", 64), ("float16", 128), ("float32", 256)])
def test_decode_over_more_than_1024_partitions(dtype, d):
    """The merge holds 1024 partitions' weights at a time.  Two tokens of each sequence take most of the weight,
    one in a partition before that and one in a partition past it (and in the last, a shorter one)."""
    rng = rng_of(94)
    hq, hkv, bs = 2, 1, 16
    cache, held, q, tables, ctx = decode_case(rng, [33001, 9, 32769, 32768], hq, hkv, d, bs, dtype)
    q[:, :, 1] = q[:, :, 0]
    k8 = held[0]
    for b, tokens in ((0, (300, 32900)), (2, (32767, 32768)), (3, (5, 32767))):
        for t in tokens:
            blk, row = int(tables[b, t // bs]), t % bs
            one = (q[b, 0, 0].float() * 90 * 64 / d).clamp(-448, 448).to(torch.float8_e4m3fn)
            cache.k_cache[0][blk, 0, row] = one
            k8[blk, 0, row] = one.double().cpu().numpy()
            for s, mine in ((cache.k_scale[0], held[2]), (cache.v_scale[0], held[3])):
                s[blk, 0] = 2.0 ** -5
                mine[blk, 0] = 2.0 ** -5
    want, _ = ref.decode_ref(q[:, 0].double().cpu().numpy(), *held, tables, ctx, 1 / math.sqrt(d))
    for b, t in ((0, 32900), (0, 300), (2, 32768), (3, 32767)):     # leaving one out would show
        v = ref.rows_ref(held[1], held[3], tables[b], t + 1)[t, 0]
        assert np.abs(v).max() > 2 and np.corrcoef(want[b, 0], v)[0, 1] > 0.3
    got = run_decode(cache, q, tables, ctx, hq, hkv, d, bs, partition_size=32)
    check_decode(got, held, q, tables, ctx, d, dtype)
    # half a step of bf16 on outputs below 448 * 2^-5 = 14 is 0.055, and the errors above it are far smaller here; a
    # token left out, of a weight above 0.3 and a value above 2, moves an output by more than 0.3
    assert np.abs(got[:, 0].double().cpu().numpy() - want).max() <= 0.1
    whole = run_decode(cache, q, tables, ctx, hq, hkv, d, bs, partition_size=33024)
    check_decode(whole, held, q, tables, ctx, d, dtype)


@gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("count,hkv,d", [(8192, 8, 64), (6600, 5, 128), (9400, 7, 64), (4100, 16, 64)])
def test_write_of_several_heads_a_wave(dtype, count, hkv, d):
    """Long writes give a work-group more (head, cache) pairs than it has waves, and a last group of fewer heads;
    the first block is entered in its middle and holds rows that are rounded again."""
    rng = rng_of(95)
    bs = 16
    assert -(-count // 16) * hkv >= 2048
    nb = count // bs + 20
    cache = make_cache(nb, bs, hkv, d, dtype)
    held = fill(cache, rng)
    blocks = rng.permutation(nb)
    pos = np.arange(9, 9 + count)
    slots = blocks[pos // bs] * bs + pos % bs
    slots[100] = -1
    slots[count // 2] = slots[3]                      # among rows of another block: the last token is the one written
    k, v = (torch.from_numpy(rng.standard_normal((count, hkv, d)) * np.exp2(rng.integers(-4, 8, (count, 1, 1)))
                             ).to("cuda", DTYPES[dtype]) for _ in range(2))
    cache.write_kv_slots(0, torch.from_numpy(slots.astype(np.int32)).cuda(), k, v)
    check_write(cache, held, k, v, slots)


@gpu
def test_calls_repeat_bit_for_bit():
    """Split contexts, split keys and log-probabilities with ties: no order of arrival shows in the results."""
    from tinyvllm_amd.sampling import token_logprobs
    rng = rng_of(96)
    cache, held, q, tables, ctx = decode_case(rng, [4000, 33, 2900], 8, 2, 128, 16, "bfloat16")
    rows = torch.from_numpy(rng.integers(0, 40, (20, 70000)).astype(np.float32)).cuda()
    tokens = torch.arange(20, dtype=torch.int32, device="cuda")
    chunk_cache, _, cq, table = chunk_case(rng, 21, 3000, 8, 2, 128, 16, "float16")

    def once():
        return (run_decode(cache, q, tables, ctx, 8, 2, 128, 16, partition_size=128), run_chunk(chunk_cache, cq, table, 3000),
                *token_logprobs(rows, tokens, 20))
    first = once()
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, once()))
