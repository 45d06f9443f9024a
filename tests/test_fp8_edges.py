"""The 8-bit cache at the edges of its number range and of its callers' contracts."""

import ctypes

import pytest
import torch

from tests.test_fp8_cache import DTYPES, check_decode, decode_case, gpu, make_cache, rng_of, run_decode
from tests.test_fp8_llama import build
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


def test_model_calls_refuse_an_8_bit_caches_misuse_before_any_launch():
    """Shapes and sizes that a layer's kernels would refuse after others have run; no workspace is given, so a
    call that passes these checks stops at that."""
    from tinyvllm_amd import _lib
    from tinyvllm_amd.llama import _Cache, _DecodeArgs, _Model, _PP, _PrefillArgs
    lib = _lib.load()
    keep = [(ctypes.c_void_p * 2)(*x) for x in ((256, 256), (256, 264), (256, None), (256, 258))]
    pp, off8, null, off2 = (ctypes.cast(x, _PP) for x in keep)

    def model(head_dim=64, dtype=_lib.TV_F16, heads=4):
        return _Model(2, 64, heads, 1, head_dim, 64, 64, dtype, 1e-5, 256, pp, pp, pp, pp, pp, pp, 256, 256, 256, 16)

    def decode(m, cache, batch=1, blocks=4, part=64):
        args = _DecodeArgs(batch, 256, 256, 256, 256, blocks, blocks, part, 1, None, None, 0, None, 0)
        rc = lib.tv_llama_decode_step(ctypes.byref(m), ctypes.byref(cache), ctypes.byref(args), None)
        return rc, lib.tv_last_error()

    def prefill(m, cache, n, start, attend=1, width=1 << 24):
        args = _PrefillArgs(n, 256, start, 256, width, None, 0, None, None, 0, attend)
        rc = lib.tv_llama_prefill(ctypes.byref(m), ctypes.byref(cache), ctypes.byref(args), None)
        return rc, lib.tv_last_error()

    good = _Cache(pp, pp, 8, 16, pp, pp)
    for m, cache, code, what in ((model(32), good, _lib.TV_EUNSUPPORTED, b"head_dim 32"),
                                 (model(), _Cache(pp, pp, 8, 1040, pp, pp), _lib.TV_EUNSUPPORTED, b"block_size 1040"),
                                 (model(), _Cache(off8, pp, 8, 16, pp, pp), _lib.TV_EINVAL, b"aligned"),
                                 (model(), _Cache(pp, null, 8, 16, pp, pp), _lib.TV_EINVAL, b"layer 1"),
                                 (model(), _Cache(pp, pp, 8, 16, pp, null), _lib.TV_EINVAL, b"layer 1"),
                                 (model(), _Cache(pp, pp, 8, 16, off2, pp), _lib.TV_EINVAL, b"scales 4-byte")):
        for rc, error in (decode(m, cache), prefill(m, cache, 4, 0)):
            assert rc == code and what in error
    for got in (decode(model(), good, part=48), decode(model(), good, batch=65536), decode(model(), good, blocks=1 << 27),
                decode(model(), good, blocks=1 << 18, part=32)):
        assert got[0] == _lib.TV_EINVAL and b"over an 8-bit cache" in got[1]
    for got in (prefill(model(dtype=_lib.TV_F32), good, 65536, 8), prefill(model(), good, 65535 * 16 + 1, 8),
                prefill(model(), good, 9, (1 << 30) - 8, width=1 << 27)):
        assert got[0] == _lib.TV_EINVAL and b"too long over an 8-bit cache" in got[1]
    # the same without a prefix, over a 16-bit cache, and at the limits: only the workspace is missing
    plain = _Cache(pp, pp, 8, 16)
    for got in (decode(model(), good), decode(model(), plain, part=48), prefill(model(dtype=_lib.TV_F32), good, 65536, 8, 0),
                prefill(model(dtype=_lib.TV_F32), good, 65535, 8), prefill(model(), plain, 9, 8)):
        assert got[0] == _lib.TV_EINVAL and b"workspace" in got[1], got[1]


@gpu
@pytest.mark.parametrize("columns", [4, 1 << 21])
def test_fp32_chunk_over_a_table_wider_than_it_needs(columns):
    """2^21 columns of 1024 tokens: the table's tokens pass 32 bits, the chunk's do not."""
    from tinyvllm_amd.kv_cache import FP8KVCache
    config, model, _ = build("float32")
    tokens = torch.arange(60, dtype=torch.int32)
    out = []
    for width in (1, columns):
        cache = FP8KVCache(config.n_layers, 2, 1024, config.n_kv_heads, config.head_dim, "float32")
        table = torch.zeros(width, dtype=torch.int32, device="cuda")
        table[0] = 1
        model.prefill_table(tokens[:20], cache, table, logits=None)
        out.append(model.prefill_table(tokens[20:], cache, table, 20, attend_prefix=True))
    assert torch.equal(*out)


@gpu
def test_a_captured_step_keeps_its_scales():
    """A step points at the scales as at the numbers: both outlive their place in the cache's lists."""
    import gc
    import weakref
    from tinyvllm_amd.kv_cache import FP8KVCache
    from tinyvllm_amd.llama import DecodeGraph
    config, model, _ = build("bfloat16")
    cache = FP8KVCache(config.n_layers, 4, 16, config.n_kv_heads, config.head_dim, "bfloat16")
    graph = DecodeGraph(model, cache, 1, 4)
    lists = (cache.k_cache, cache.v_cache, cache.k_scale, cache.v_scale)
    seen = [weakref.ref(x[1]) for x in lists]
    for x in lists:
        x[1] = torch.zeros_like(x[1].view(torch.uint8)).view(x[1].dtype)
    gc.collect()
    assert all(r() is not None for r in seen)
    del graph
    gc.collect()
    assert all(r() is None for r in seen)


@gpu
@pytest.mark.parametrize("kind", ["FP8KVCache", "KVCache"])
def test_a_replaced_cache_can_be_released(kind):
    """Steps of an old cache are dropped, their memory with them; those of other caches stay."""
    import gc
    import weakref
    from tinyvllm_amd import kv_cache
    config, model, _ = build("float16")

    def make():
        return getattr(kv_cache, kind)(config.n_layers, 4, 16, config.n_kv_heads, config.head_dim, "float16")
    jit = model.create_jit_decode(16)
    old, new = make(), make()
    for batch in (1, 2):
        jit.graph_for(old, batch, 2).run(2)
    kept = jit.graph_for(new, 2, 2)
    jit.release(make())                              # nothing was captured for it
    seen = [weakref.ref(old), weakref.ref(old.k_cache[0])]
    jit.release(old)
    del old
    gc.collect()
    assert all(r() is None for r in seen)
    assert jit.graph_for(new, 2, 2) is kept
    kept.run(1)
    torch.cuda.synchronize()


def test_rows_are_checked_without_making_tensors():
    """``write_kv``'s checks run on every call: they look at sizes and strides and create nothing."""
    import types
    from torch.utils._python_dispatch import TorchDispatchMode
    from tinyvllm_amd.kv_cache import KVCache
    made = []

    class Record(TorchDispatchMode):
        def __torch_dispatch__(self, func, kinds, args=(), kwargs=None):
            made.append(func)
            return func(*args, **(kwargs or {}))

    def cache(hkv, d):
        return types.SimpleNamespace(n_kv_heads=hkv, head_dim=d, dtype=torch.float32, k_cache=[wide])
    wide = torch.zeros(6, 4, 32)
    for x, stride in ((wide[:, 1:2], 128), (wide[:1, 1:2], 32), (wide[:0, :2], 64), (wide, 128), (wide[::2], 256),
                      (wide[2:3], 128), (wide[:, :1, :1], 128), (wide.transpose(0, 1)[:, :1], 32)):
        hkv, d = x.shape[1:]
        with Record():
            assert KVCache._rows(cache(hkv, d), x, "k") == (x, stride)
    for x in (wide[:1, ::2], wide[:, ::2], wide[:1, :, :16], wide[:, :, ::2], wide[:1, :1, ::2]):
        hkv, d = x.shape[1:]
        with pytest.raises(ValueError, match="contiguous"):
            KVCache._rows(cache(hkv, d), x, "k")
    assert made == []


@gpu
@pytest.mark.parametrize("spread", [2.0 ** -80, 2.0 ** 75])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_attention_over_values_of_any_defined_size(dtype, spread):
    """V of 2^-80 to 2^84 (the sums are defined below 2^89): results scale with it."""
    rng = rng_of(81)
    hq, hkv, d, bs = 8, 2, 64, 16
    cache, held, q, tables, ctx = decode_case(rng, [700, 33, 64], hq, hkv, d, bs, dtype)
    cache.v_scale[0].mul_(spread)
    for part in (None, 64):
        got = run_decode(cache, q, tables, ctx, hq, hkv, d, bs, partition_size=part, out_dtype=torch.float32)
        check_decode(got.double() / spread, held, q, tables, ctx, d, dtype, "float32")
    if dtype == "float32":
        return                                        # chunks are of 16-bit queries
    for n, start in ((40, 90), (9, 2100)):            # unsplit and split keys
        cache, held, q, table = chunk_case(rng, n, start, hq, hkv, d, bs, dtype)
        cache.v_scale[0].mul_(spread)
        got = run_chunk(cache, q, table, start, out_dtype=torch.float32)
        check_chunk(got.double() / spread, held, q, table, start, dtype, out_dtype="float32")
