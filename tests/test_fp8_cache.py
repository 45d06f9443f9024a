"""The 8-bit K/V cache: its writes, its reads and the single-token attention over it."""

import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import fp8_cache as ref
from tests.fp8_tolerance import attention_bound
from tests.random_cases import case_count, case_seed

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
gpu = pytest.mark.gpu


def rng_of(seed):
    return np.random.Generator(np.random.PCG64(seed))


# ---- the oracle, on the CPU --------------------------------------------------------

def test_oracle_rounds_as_torch_does():
    x = np.concatenate([np.linspace(-448, 448, 20011), np.exp2(np.linspace(-12, 8.8, 3001)), [0.0, 2.0 ** -10]])
    x = x.astype(np.float32)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).float().numpy()
    assert np.array_equal(ref.round_e4m3(x), want)


def test_oracle_scale():
    for amax, s in ((448.0, 1.0), (448.1, 2.0), (224.0, 0.5), (1.75, 2.0 ** -8), (0.0, 2.0 ** -100), (1.0, 2.0 ** -8)):
        assert ref.scale_for(amax) == s


def test_oracle_grows_and_restarts_a_block():
    c, s = np.zeros((1, 1, 4, 2)), np.full((1, 1), ref.SCALE_MIN)
    ref.write_ref(c, s, np.array([[[1.0, 0.5]]]), [0])
    assert s[0, 0] == 2.0 ** -8 and np.array_equal(c[0, 0, 0] * s[0, 0], [1.0, 0.5])
    ref.write_ref(c, s, np.array([[[1000.0, 0.0]]]), [1])
    assert s[0, 0] == 4.0 and np.array_equal(c[0, 0, 0] * s[0, 0], [1.0, 0.5])     # 2^-2, 2^-3: held exactly
    ref.write_ref(c, s, np.array([[[0.5, 0.0]]]), [0])
    assert s[0, 0] == 2.0 ** -9 and np.array_equal(c[0, 0, 1:], np.zeros((3, 2)))


# ---- refusals: nothing is launched ----------------------------------------------------

def test_entry_points_validate_on_the_host():
    from tinyvllm_amd import _lib
    lib, p = _lib.load(), ctypes.c_void_p(256)
    w = [p, p, p, p, p, p, p, 4, 2, 64, 16, 8, 128, 128, 1, None, None]

    def write(**kw):
        a = list(w)
        for i, v in kw.items():
            a[int(i[1:])] = v
        return lib.tv_reshape_and_cache_fp8(*a)

    assert write(_0=None) == _lib.TV_EINVAL and b"null pointer" in lib.tv_last_error()
    assert write(_6=None) == _lib.TV_EINVAL and b"slot_mapping" in lib.tv_last_error()
    assert write(_9=96) == _lib.TV_EUNSUPPORTED and b"head_dim 96" in lib.tv_last_error()
    assert write(_10=1025) == _lib.TV_EUNSUPPORTED and b"block_size" in lib.tv_last_error()
    assert write(_10=0) == _lib.TV_EINVAL
    assert write(_12=127) == _lib.TV_EINVAL and b"stride" in lib.tv_last_error()
    assert write(_14=3) == _lib.TV_EINVAL and b"dtype" in lib.tv_last_error()
    assert write(_0=ctypes.c_void_p(264)) == _lib.TV_EINVAL and b"aligned" in lib.tv_last_error()
    assert write(_4=ctypes.c_void_p(257)) == _lib.TV_EINVAL and b"misaligned" in lib.tv_last_error()
    assert write(_7=-1) == _lib.TV_EINVAL
    assert write(_7=1 << 28) == _lib.TV_EINVAL and b"grid too large" in lib.tv_last_error()
    assert write(_7=0) == _lib.TV_OK
    b = [p, p, p, p, p, p, 3, 0, 4, 2, 64, 16, 8, 128, 128, 1, None]
    assert lib.tv_write_kv_fp8(*b[:6], 8, *b[7:]) == _lib.TV_EINVAL and b"block_id" in lib.tv_last_error()
    assert lib.tv_write_kv_fp8(*b[:7], 13, *b[8:]) == _lib.TV_EINVAL and b"do not fit" in lib.tv_last_error()
    assert lib.tv_read_kv_blocks_fp8(p, p, p, p, p, p, p, 1, 17, 2, 64, 16, 8, 1, None) == _lib.TV_EINVAL
    assert b"exceeds" in lib.tv_last_error()
    d = [p] * 8 + [2, 8, 2, 64, 16, 8, 4, 4, 0.1, 1, 1, 64, None, 0, None]

    def decode(**kw):
        a = list(d)
        for i, v in kw.items():
            a[int(i[1:])] = v
        return lib.tv_paged_decode_fp8(*a)

    assert decode(_1=None) == _lib.TV_EINVAL and b"null pointer" in lib.tv_last_error()
    assert decode(_9=7) == _lib.TV_EINVAL and b"head counts" in lib.tv_last_error()
    assert decode(_11=32) == _lib.TV_EUNSUPPORTED
    assert decode(_15=5) == _lib.TV_EINVAL and b"block table" in lib.tv_last_error()
    assert decode(_18=2) == _lib.TV_EINVAL and b"out_dtype" in lib.tv_last_error()
    assert decode(_19=48) == _lib.TV_EINVAL and b"multiple of 32" in lib.tv_last_error()
    assert decode(_19=32) == _lib.TV_EINVAL and b"workspace" in lib.tv_last_error()
    assert decode(_1=ctypes.c_void_p(264)) == _lib.TV_EINVAL and b"aligned" in lib.tv_last_error()


def test_workspace_of_a_split_context():
    from tinyvllm_amd import _lib
    lib = _lib.load()
    assert lib.tv_paged_decode_fp8_workspace_bytes(3, 8, 64, 4, 16, 64) == 0
    assert lib.tv_paged_decode_fp8_workspace_bytes(3, 8, 64, 4, 16, 32) == 3 * 8 * 2 * 66 * 4
    assert lib.tv_paged_decode_fp8_workspace_bytes(40, 8, 64, 4, 16, 64) == 256


# ---- on the GPU -------------------------------------------------------------------------

def numbers(c):
    return c.float().cpu().numpy().astype(np.float64)


def make_cache(num_blocks, bs, hkv, d, dtype, layers=1):
    from tinyvllm_amd.kv_cache import FP8KVCache
    return FP8KVCache(layers, num_blocks, bs, hkv, d, dtype)


def fill(cache, rng, spread=1.0, layer=0):
    """Random numbers of every magnitude with scales of their own; returns the oracle's four arrays."""
    out = []
    for c, s in ((cache.k_cache[layer], cache.k_scale[layer]), (cache.v_cache[layer], cache.v_scale[layer])):
        x = rng.standard_normal(c.shape).astype(np.float32) * 60
        c.copy_(torch.from_numpy(np.clip(x, -448, 448)).to(c.device).to(torch.float8_e4m3fn))
        e = rng.integers(-8, -4, s.shape) + (0 if spread == 1.0 else np.log2(spread).astype(int))
        s.copy_(torch.from_numpy(np.exp2(e).astype(np.float32)))
        out.append((numbers(c), s.cpu().numpy().astype(np.float64)))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def check_write(cache, held, k, v, slots):
    """Numbers and scales of a write, bit for bit (they are exact by definition)."""
    k8, v8, ks, vs = held
    for c, s, x, got_c, got_s in ((k8, ks, k, cache.k_cache[0], cache.k_scale[0]),
                                  (v8, vs, v, cache.v_cache[0], cache.v_scale[0])):
        ref.write_ref(c, s, x.float().cpu().numpy().astype(np.float64), slots)
        assert np.array_equal(got_s.cpu().numpy().astype(np.float64), s)
        assert np.array_equal(numbers(got_c), c, equal_nan=True)


@gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("hkv,d,bs", [(8, 128, 16), (4, 64, 16), (1, 256, 16), (3, 64, 7), (5, 128, 33), (2, 64, 1),
                                      (2, 256, 200)])
def test_write_from_a_slot_mapping(dtype, hkv, d, bs):
    """Runs of rows, single rows, rows out of order, a slot named twice, padding and a slot past the cache."""
    rng = rng_of(11)
    nb = max(6, 96 // bs)
    cache = make_cache(nb, bs, hkv, d, dtype)
    held = fill(cache, rng)
    for call in range(3):
        t = 50
        slots = rng.permutation(nb * bs)[:t] if call == 0 else np.arange(t) + call * 3
        slots = np.asarray(slots[:min(t, nb * bs)] % (nb * bs), np.int64)
        slots[5 % len(slots)] = slots[0]
        slots[3 % len(slots)] = -1
        slots[-1] = nb * bs + 2
        k = torch.from_numpy(rng.standard_normal((len(slots), hkv, d)) * np.exp2(rng.integers(-6, 6, (len(slots), 1, 1)))
                             ).to("cuda", DTYPES[dtype])
        v = torch.from_numpy(rng.standard_normal((len(slots), hkv, d))).to("cuda", DTYPES[dtype])
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        print("write", dtype, hkv, d, bs, call, flush=True)
        cache.write_kv_slots(0, torch.from_numpy(slots.astype(np.int32)).cuda(), k, v, err_count=err)
        assert int(err) == 1
        check_write(cache, held, k, v, slots)


@gpu
@pytest.mark.parametrize("count", [1, 2, 257, 4000])
def test_write_of_many_tokens(count):
    rng = rng_of(12)
    hkv, d, bs = 2, 64, 16
    nb = count // bs + 40
    cache = make_cache(nb, bs, hkv, d, "bfloat16")
    held = fill(cache, rng)
    blocks = rng.permutation(nb)
    pos = np.arange(5, 5 + count)
    slots = blocks[pos // bs] * bs + pos % bs
    k, v = (torch.from_numpy(rng.standard_normal((count, hkv, d))).to("cuda", torch.bfloat16) for _ in range(2))
    cache.write_kv_slots(0, torch.from_numpy(slots.astype(np.int32)).cuda(), k, v)
    check_write(cache, held, k, v, slots)


@gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_write_of_strided_and_unaligned_rows(dtype):
    """Rows inside a wider projection, at an address that is no multiple of 16 bytes."""
    rng = rng_of(13)
    hkv, d, bs, t = 2, 64, 16, 21
    for offset, pad in ((0, 64), (1, 3)):
        cache = make_cache(4, bs, hkv, d, dtype)
        held = fill(cache, rng)
        wide = torch.from_numpy(rng.standard_normal((t, 2 * hkv * d + pad))).to("cuda", DTYPES[dtype])
        k = torch.as_strided(wide, (t, hkv, d), (wide.stride(0), d, 1), offset)
        v = torch.as_strided(wide, (t, hkv, d), (wide.stride(0), d, 1), offset + hkv * d)
        slots = np.arange(t) + 2
        cache.write_kv_slots(0, torch.from_numpy(slots.astype(np.int32)).cuda(), k, v)
        check_write(cache, held, k, v, slots)


@gpu
def test_write_of_zeros_extremes_and_non_finite_rows():
    rng = rng_of(14)
    hkv, d, bs = 2, 64, 16
    cache = make_cache(3, bs, hkv, d, "float32")
    held = fill(cache, rng)
    k = torch.zeros((6, hkv, d), device="cuda")
    v = torch.zeros_like(k)
    k[1] = 3.4e38
    k[2, 0, :4] = torch.tensor([float("nan"), float("inf"), -float("inf"), 2.0])
    k[3] = 1e-38
    k[4] = torch.tensor(448 * 2.0 ** -100)
    v[2, 1, 7] = float("inf")
    v[5] = 2.0 ** -109
    for slots in ([0, 1, 2, 3, 4, 5], [20, 21, 22, 23, 24, 25], [32, 33, -1, -1, -1, 47]):
        cache.write_kv_slots(0, torch.tensor(slots, dtype=torch.int32, device="cuda"), k, v)
        check_write(cache, held, k, v, slots)


@gpu
def test_write_one_block_and_read_back():
    rng = rng_of(15)
    hkv, d, bs = 4, 128, 16
    for dtype in sorted(DTYPES):
        cache = make_cache(5, bs, hkv, d, dtype)
        held = fill(cache, rng)
        k, v = (torch.from_numpy(rng.standard_normal((5, hkv, d))).to("cuda", DTYPES[dtype]) for _ in range(2))
        cache.write_kv(0, 3, 9, k, v)
        check_write(cache, held, k, v, 3 * bs + 9 + np.arange(5))
        cache.write_kv(0, 1, 0, k[0], v[0])
        check_write(cache, held, k[:1], v[:1], [bs])
        k8, v8, ks, vs = held
        for ids, n in (([3, 1], 29), ([4], 16), ([0, 2, 4], 1), ([], 5), ([2, 9], 32), ([1], 0)):
            got = cache.read_kv_blocks(0, ids, n)
            as_tensor = cache.read_kv_blocks(0, torch.tensor(ids, dtype=torch.int32, device="cuda"), n)
            for c, s, x, y in zip((k8, v8), (ks, vs), got, as_tensor):
                n_rows = min(n, len(ids) * bs)
                want = ref.rows_ref(c, s, [i if i < 5 else 0 for i in ids] or [0], n_rows)
                if 9 in ids:
                    want[bs:] = 0                               # a block outside the cache
                assert x.dtype == DTYPES[dtype] and torch.equal(x, y)
                assert np.array_equal(x.double().cpu().numpy(), want)      # 4 significant bits fit every type
        assert cache.get_memory_bytes() == 2 * 5 * hkv * (bs * d + 4)


@gpu
def test_read_in_fp16_is_limited_to_its_largest_number():
    cache = make_cache(1, 16, 1, 64, "float16")
    x = torch.full((1, 1, 64), 65504.0, device="cuda", dtype=torch.float16)
    cache.write_kv(0, 0, 0, x, -x)
    k, v = cache.read_kv_blocks(0, [0], 1)
    assert torch.equal(k, x) and torch.equal(v, -x)             # 65536 in e4m3


@gpu
@pytest.mark.parametrize("kind", ["FP8KVCache", "KVCache"])
def test_a_single_token_with_spread_heads_is_refused(kind):
    """One token whose heads are not next to each other: its row is not the memory behind its first element."""
    from tinyvllm_amd import kv_cache
    cache = getattr(kv_cache, kind)(1, 2, 16, 2, 64, "float16")
    x = torch.randn((2, 2, 128), device="cuda").half()[:1, :, :64]
    with pytest.raises(ValueError, match="contiguous"):
        cache.write_kv(0, 0, 0, x, x)
    with pytest.raises(ValueError, match="contiguous"):
        cache.write_kv(0, 0, 0, x.contiguous()[0], x[0])
    cache.write_kv(0, 0, 0, x.contiguous(), x[0].contiguous())
    one = getattr(kv_cache, kind)(1, 2, 16, 1, 64, "float16")
    y = torch.randn((3, 5, 64), device="cuda").half()[:, 2:3]      # one head: any stride of it will do
    one.write_kv(0, 0, 0, y, y)
    k, v = one.read_kv_blocks(0, [0], 3)
    assert torch.equal(k, v) and (k - y).abs().max() <= 2.0 ** -4 * y.abs().max()


def test_python_refusals_need_no_gpu():
    from tinyvllm_amd.kv_cache import FP8KVCache, reshape_and_cache_fp8
    with pytest.raises(ValueError, match="HIP device"):
        FP8KVCache(1, 4, 16, 2, 64, "float16", device="cpu")
    for hd, bs in ((96, 16), (64, 2000), (64, 0)):
        with pytest.raises(ValueError, match="head_dim|block_size"):
            FP8KVCache(1, 4, bs, 2, hd, "float16")
    c = torch.zeros((4, 2, 16, 64), dtype=torch.uint8).view(torch.float8_e4m3fn)
    s = torch.ones((4, 2))
    x = torch.zeros((3, 2, 64))
    slots = torch.zeros(3, dtype=torch.int32)
    for args, what in (((c, c[:3], s, s, x, x, slots), "one shape"), ((c.float(), c.float(), s, s, x, x, slots), "e4m3"),
                       ((c, c, s[:3], s, x, x, slots), "k_scale"), ((c, c, s, s.double(), x, x, slots), "k_scale"),
                       ((c, c, s, s, x[:, :1], x[:, :1], slots), "k/v must be"),
                       ((c, c, s, s, x, x.half(), slots), "share a dtype"),
                       ((c, c, s, s, x, x, slots[:2]), "slot_mapping"), ((c, c, s, s, x, x, slots.long()), "slot_mapping")):
        with pytest.raises(ValueError, match=what):
            reshape_and_cache_fp8(*args)


@gpu
def test_values_near_fp16s_largest_give_finite_outputs():
    """65504 is held as 65536; an average of such values is limited to 65504, split or not."""
    hq, hkv, d, bs = 4, 2, 64, 16
    cache = make_cache(6, bs, hkv, d, "float16")
    tables = np.arange(6, dtype=np.int32)[None]
    k = torch.zeros((90, hkv, d), device="cuda", dtype=torch.float16)
    v = torch.full_like(k, 65504.0)
    v[:, 1] = -65504.0
    cache.write_kv_slots(0, torch.arange(90, dtype=torch.int32, device="cuda"), k, v)
    q = torch.zeros((1, 1, hq, d), device="cuda", dtype=torch.float16)
    for part in (None, 32):
        got = run_decode(cache, q, tables, np.array([90], np.int32), hq, hkv, d, bs, partition_size=part)
        assert torch.equal(got[0, 0, :2], torch.full_like(got[0, 0, :2], 65504.0))
        assert torch.equal(got[0, 0, 2:], torch.full_like(got[0, 0, 2:], -65504.0))
        wide = run_decode(cache, q, tables, np.array([90], np.int32), hq, hkv, d, bs, partition_size=part,
                          out_dtype=torch.float32)
        assert torch.equal(wide[0, 0, 0], torch.full_like(wide[0, 0, 0], 65536.0))


@gpu
def test_padded_rows_of_a_batch_write_and_read_nothing():
    """Slots of -1 and contexts of 0, as a fixed-size batch with absent sequences has them."""
    rng = rng_of(30)
    hq, hkv, d, bs = 8, 2, 64, 16
    cache, held, q, tables, ctx = decode_case(rng, [33, 20], hq, hkv, d, bs, "bfloat16")
    k, v = (torch.from_numpy(rng.standard_normal((4, hkv, d))).to("cuda", torch.bfloat16) for _ in range(2))
    slots = [-1, int(tables[0, 32 // bs]) * bs + 32 % bs, -1, -1]
    cache.write_kv_slots(0, torch.tensor(slots, dtype=torch.int32, device="cuda"), k, v)
    check_write(cache, held, k, v, slots)
    padded = np.zeros((4, tables.shape[1]), np.int32)
    padded[1:3] = tables
    got = run_decode(cache, torch.cat([q[:1], q, q[:1]]), padded, np.array([0, 33, 20, 0], np.int32), hq, hkv, d, bs)
    assert torch.count_nonzero(got[0]) == 0 and torch.count_nonzero(got[3]) == 0
    check_decode(got[1:3], held, q, tables, ctx, d, "bfloat16")


@gpu
def test_writes_of_two_streams_to_different_blocks():
    rng = rng_of(33)
    hkv, d, bs = 4, 128, 16
    cache = make_cache(80, bs, hkv, d, "float16")
    held = fill(cache, rng)
    parts = []
    for i in range(2):
        t = 600
        slots = (np.arange(t) + i * 640).astype(np.int32)
        k, v = (torch.from_numpy(rng.standard_normal((t, hkv, d))).to("cuda", torch.float16) for _ in range(2))
        parts.append((torch.from_numpy(slots).cuda(), k, v, slots))
    streams = [torch.cuda.Stream() for _ in parts]
    torch.cuda.synchronize()
    for _ in range(3):
        for s, (slots, k, v, _) in zip(streams, parts):
            with torch.cuda.stream(s):
                cache.write_kv_slots(0, slots, k, v)
    torch.cuda.synchronize()
    check_write(cache, held, torch.cat([p[1] for p in parts]), torch.cat([p[2] for p in parts]),
                np.concatenate([p[3] for p in parts]))


@gpu
def test_decode_over_a_cache_past_32_bit_offsets():
    """Blocks that lie more than 4 GiB into the cache's storage."""
    hq, hkv, d, bs = 4, 2, 128, 16
    nb = (9 << 29) // (hkv * bs * d)                      # 4.5 GiB each of K and V
    cache = make_cache(nb, bs, hkv, d, "bfloat16")
    rng = rng_of(34)
    blocks = np.array([nb - 1, 3, nb - 20000, nb // 2], np.int32)
    pos = np.arange(50)
    slots = torch.from_numpy((blocks[pos // bs].astype(np.int64) * bs + pos % bs).astype(np.int32)).cuda()
    k, v = (torch.from_numpy(rng.standard_normal((50, hkv, d))).to("cuda", torch.bfloat16) for _ in range(2))
    cache.write_kv_slots(0, slots, k, v)
    ids = torch.from_numpy(blocks.astype(np.int64)).cuda()
    held = []
    for c, s in ((cache.k_cache[0], cache.k_scale[0]), (cache.v_cache[0], cache.v_scale[0])):
        held.append((numbers(c[ids]), s[ids].double().cpu().numpy()))
    small = (held[0][0], held[1][0], held[0][1], held[1][1])
    written = [np.zeros_like(small[0]), np.full((4, hkv), ref.SCALE_MIN)]
    ref.write_ref(*written, k.double().cpu().numpy(), pos)
    assert np.array_equal(written[0], small[0]) and np.array_equal(written[1], small[2])
    q = torch.from_numpy(rng.standard_normal((1, 1, hq, d))).to("cuda", torch.bfloat16)
    ctx = np.array([50], np.int32)
    got = run_decode(cache, q, blocks[None], ctx, hq, hkv, d, bs)
    check_decode(got, small, q, np.arange(4, dtype=np.int32)[None], ctx, d, "bfloat16")
    got = cache.read_kv_blocks(0, blocks.tolist(), 50)
    assert np.array_equal(got[1].double().cpu().numpy(), ref.rows_ref(small[1], small[3], np.arange(4), 50))
    from tinyvllm_amd.attention import flash_prefill_paged_fp8
    chunk = flash_prefill_paged_fp8(q, cache.k_cache[0], cache.v_cache[0], cache.k_scale[0], cache.v_scale[0],
                                    torch.from_numpy(blocks).cuda(), 49)
    want = ref.attend_ref(q[0].double().cpu().numpy(), ref.rows_ref(small[0], small[2], np.arange(4), 50),
                          ref.rows_ref(small[1], small[3], np.arange(4), 50), 49, 1 / math.sqrt(d))[0]
    assert np.abs(chunk[0].double().cpu().numpy() - want).max() <= 2.0 ** -6 * np.abs(small[1] * small[3][..., None, None]).max()


# ---- attention of single tokens ------------------------------------------------------------

def decode_case(rng, ctx, hq, hkv, d, bs, dtype, spread=1.0, extra_cols=0):
    ctx = np.asarray(ctx, np.int32)
    need = np.maximum(-(-ctx // bs), 0)
    nb = int(need.sum()) + 3
    perm = rng.permutation(nb).astype(np.int32)
    tables = np.zeros((len(ctx), int(need.max()) + extra_cols or 1), np.int32)
    at = 0
    for i, n in enumerate(need):
        tables[i, :n] = perm[at:at + n]
        at += n
    cache = make_cache(nb, bs, hkv, d, dtype)
    held = fill(cache, rng, spread)
    q = torch.from_numpy(rng.standard_normal((len(ctx), 1, hq, d))).to("cuda", DTYPES[dtype])
    return cache, held, q, tables, ctx


def run_decode(cache, q, tables, ctx, hq, hkv, d, bs, **kw):
    from tinyvllm_amd.attention import paged_decode_attention_fp8
    return paged_decode_attention_fp8(q, cache.k_cache[0], cache.v_cache[0], cache.k_scale[0], cache.v_scale[0],
                                      torch.from_numpy(tables).cuda(), torch.from_numpy(ctx).cuda(), hq, hkv, d, bs, **kw)


def check_decode(got, held, q, tables, ctx, d, dtype, out_dtype=None):
    want, bound = ref.decode_ref(q[:, 0].double().cpu().numpy(), *held, tables, ctx, 1 / math.sqrt(d))
    vmax = float(np.max(np.abs(held[1]) * held[3][:, :, None, None]))
    tol = attention_bound(want, bound, vmax, int(ctx.max()), d, dtype, out_dtype or dtype)
    diff = np.abs(got[:, 0].double().cpu().numpy() - want)
    assert np.all(diff <= tol), (float(diff.max()), float((diff / tol).max()))


@gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (32, 4, 64), (8, 1, 256), (12, 12, 64), (10, 2, 128), (34, 1, 64)])
@pytest.mark.parametrize("bs", [16, 32, 5])
def test_decode_lengths(dtype, hq, hkv, d, bs):
    """One token to several hundred; lengths that end inside a tile, at its end, inside a block; none."""
    rng = rng_of(21)
    ctx = [1, 0, 15, 16, 17, 31, 33, 64, 65, 127, 300]
    cache, held, q, tables, ctx = decode_case(rng, ctx, hq, hkv, d, bs, dtype, extra_cols=2)
    got = run_decode(cache, q, tables, ctx, hq, hkv, d, bs)
    assert got.dtype == DTYPES[dtype] and got.shape == q.shape
    assert torch.count_nonzero(got[1]) == 0
    check_decode(got, held, q, tables, ctx, d, dtype)
    for part in (32, 96):
        split = run_decode(cache, q, tables, ctx, hq, hkv, d, bs, partition_size=part)
        check_decode(split, held, q, tables, ctx, d, dtype)
    if dtype != "float32":
        full = run_decode(cache, q, tables, ctx, hq, hkv, d, bs, out_dtype=torch.float32)
        check_decode(full, held, q, tables, ctx, d, dtype, "float32")


@gpu
def test_decode_longest_first_batch():
    rng = rng_of(22)
    ctx = rng.integers(0, 500, 70)
    cache, held, q, tables, ctx = decode_case(rng, ctx, 8, 2, 64, 16, "float16")
    got = run_decode(cache, q, tables, ctx, 8, 2, 64, 16, partition_size=512)
    check_decode(got, held, q, tables, ctx, 64, "float16")


@gpu
def test_decode_long_context_split_over_many_partitions():
    rng = rng_of(23)
    cache, held, q, tables, ctx = decode_case(rng, [20001, 9], 4, 1, 64, 16, "bfloat16")
    for part in (None, 64):                         # 313 partitions: past one chunk of the merge
        got = run_decode(cache, q, tables, ctx, 4, 1, 64, 16, partition_size=part)
        check_decode(got, held, q, tables, ctx, 64, "bfloat16")


@gpu
@pytest.mark.parametrize("spread", [2.0 ** -60, 2.0 ** 30])
def test_decode_scales_of_any_range(spread):
    """Very small and very large values: the weights' parts hold the scale whatever its exponent."""
    rng = rng_of(24)
    cache, held, q, tables, ctx = decode_case(rng, [40, 7], 4, 2, 128, 16, "float32")
    k8, v8, ks, vs = held
    cache.v_scale[0].mul_(spread)
    vs *= spread
    got = run_decode(cache, q, tables, ctx, 4, 2, 128, 16)
    want, bound = ref.decode_ref(q[:, 0].double().cpu().numpy(), *held, tables, ctx, 1 / math.sqrt(128))
    vmax = float(np.max(np.abs(v8) * vs[:, :, None, None]))
    tol = attention_bound(want / spread, bound, vmax / spread, 40, 128, "float32", "float32") * spread
    assert np.all(np.abs(got[:, 0].double().cpu().numpy() - want) <= tol)


@gpu
def test_decode_peaked_softmax():
    """Scores of hundreds: one token takes all of the weight, and the maximum rises tile after tile."""
    rng = rng_of(25)
    cache, held, q, tables, ctx = decode_case(rng, [290, 64], 8, 2, 64, 16, "float16")
    q.mul_(20)
    check_decode(run_decode(cache, q, tables, ctx, 8, 2, 64, 16), held, q, tables, ctx, 64, "float16")


@gpu
@pytest.mark.parametrize("bs", [16, 6])
def test_decode_stale_rows_bad_blocks_and_non_finite_rows(bs):
    """What lies past a context is not seen, whatever it holds; a bad block id and a NaN row stay in
    their own sequence."""
    rng = rng_of(26)
    hq, hkv, d = 8, 2, 64
    cache, held, q, tables, ctx = decode_case(rng, [20, 37, 50, 41], hq, hkv, d, bs, "float16", extra_cols=3)
    nan = torch.full((1,), float("nan"), device="cuda").to(torch.float8_e4m3fn)[0]
    for b, n in enumerate(ctx):                                   # rows past the end of each last block
        last = tables[b, (n - 1) // bs]
        for c in (cache.k_cache[0], cache.v_cache[0]):
            c.view(torch.uint8)[int(last), :, (n - 1) % bs + 1:] = 0x7F
    assert torch.isnan(nan.float())
    tables[:, -3:] = 10 ** 6                                      # never attended
    tables[2, 1] = cache.num_blocks
    cache.v_cache[0].view(torch.uint8)[int(tables[3, 0]), 0, 2, 5] = 0x7F
    cache.k_cache[0].view(torch.uint8)[int(tables[3, 1]), 1, 1, 9] = 0xFF
    for part in (None, 32):
        got = run_decode(cache, q, tables, ctx, hq, hkv, d, bs, partition_size=part)
        good = np.array([0, 1])
        check_decode(got[:2], held, q[:2], tables[good], ctx[good], d, "float16")
        assert torch.isnan(got[2]).all()
        assert torch.isnan(got[3, 0, :4, 5]).all() and torch.isfinite(got[3, 0, :4, :5]).all()
        assert torch.isnan(got[3, 0, 4:]).all()


@gpu
def test_decode_trims_to_max_context_len_and_table_width():
    rng = rng_of(27)
    cache, held, q, tables, ctx = decode_case(rng, [100, 60], 4, 4, 64, 16, "bfloat16")
    got = run_decode(cache, q, tables, ctx, 4, 4, 64, 16, max_context_len=40)
    cut = np.minimum(ctx, 48)
    check_decode(got, held, q, tables, cut.astype(np.int32), 64, "bfloat16")


@gpu
def test_decode_plan_in_a_graph_beside_eager_calls():
    """A captured plan follows its inputs on every replay; a second plan has a workspace of its own."""
    from tinyvllm_amd.attention import PagedDecodeFP8Plan
    rng = rng_of(28)
    hq, hkv, d, bs = 8, 2, 64, 16
    cache, held, q, tables, ctx = decode_case(rng, [300, 40, 129], hq, hkv, d, bs, "float16")
    tb, cx = torch.from_numpy(tables).cuda(), torch.from_numpy(ctx).cuda()
    args = (cache.k_cache[0], cache.v_cache[0], cache.k_scale[0], cache.v_scale[0], tb, cx, hq, hkv, d, bs)
    plan = PagedDecodeFP8Plan(q, *args, partition_size=64)
    other = PagedDecodeFP8Plan(q * 2, *args, partition_size=64)
    graphs = []
    for p in (plan, other):
        p.run()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            p.run()
        graphs.append(g)
    for step in range(3):
        q.copy_(torch.from_numpy(rng.standard_normal(tuple(q.shape))).to("cuda", torch.float16))
        cx.copy_(torch.from_numpy(ctx - 7 * step))
        for g in graphs:
            g.replay()
        eager = run_decode(cache, q, tables, ctx - 7 * step, hq, hkv, d, bs, partition_size=64)
        torch.cuda.synchronize()
        assert torch.equal(plan.out, eager)
        check_decode(plan.out, held, q, tables, ctx - 7 * step, d, "float16")


@gpu
def test_write_then_decode_on_another_stream():
    rng = rng_of(29)
    hq, hkv, d, bs = 8, 2, 128, 16
    cache, held, q, tables, ctx = decode_case(rng, [33, 50], hq, hkv, d, bs, "bfloat16")
    k, v = (torch.from_numpy(rng.standard_normal((2, hkv, d))).to("cuda", torch.bfloat16) for _ in range(2))
    slots = [int(tables[b, (n - 1) // bs]) * bs + (n - 1) % bs for b, n in enumerate(ctx.tolist())]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.write_kv_slots(0, torch.tensor(slots, dtype=torch.int32, device="cuda"), k, v)
        got = run_decode(cache, q, tables, ctx, hq, hkv, d, bs)
    side.synchronize()
    check_write(cache, held, k, v, slots)
    check_decode(got, held, q, tables, ctx, d, "bfloat16")


@gpu
def test_decode_random_shapes():
    rng = rng_of(case_seed(40))
    for i in range(case_count(12)):
        dtype = ["float32", "float16", "bfloat16"][rng.integers(3)]
        d = int(rng.choice([64, 128, 256]))
        hkv = int(rng.integers(1, 5))
        hq = hkv * int(rng.integers(1, 20))
        bs = int(rng.choice([16, 16, 32, 48, 1, 7, 24]))
        ctx = rng.integers(0, 400, int(rng.integers(1, 7)))
        if not ctx.max():
            ctx[0] = 3
        print("decode", i, dtype, d, hkv, hq, bs, ctx, flush=True)
        cache, held, q, tables, ctx = decode_case(rng, ctx, hq, hkv, d, bs, dtype)
        part = [None, 32, 128][rng.integers(3)]
        got = run_decode(cache, q, tables, ctx, hq, hkv, d, bs, partition_size=part)
        check_decode(got, held, q, tables, ctx, d, dtype)
