"""A model over the 8-bit cache: prompt, chunk over the cached prefix, decode steps, and the
log-probabilities of what they return.

The float64 model attends over the values that the GPU's cache holds (the cache's own rounding is
checked where it is written), so its logits differ by the model dtype's roundings alone.
"""

import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import fp8_cache as ref
from tests.test_fp8_cache import numbers
from tests.test_logprobs import check as check_logprobs

gpu = pytest.mark.gpu
# A logit is the end of about 30 roundings of activations to the dtype (15 a layer: two norms, q, k, v, two rotations,
# attention, four products, gate, two sums), each up to 2^-8 of its value in bf16, 2^-8 / sqrt(3) / 1.4 rms over a binade.
# Unrelated, on logits of rms 1: sqrt(30) * 1.6e-3 = 9e-3, and 4.5 times that is the largest of 20000; twice it is
# allowed.  fp16 has an eighth.  fp32 sums up to 512 products, of which each addition rounds: 2^-24 * sqrt(512) *
# sqrt(30) * 4.5, twice, is 7e-5 at most.
TOL = {"float32": 7e-5, "float16": 1e-2, "bfloat16": 8e-2}


class Model64:
    """The layers in float64; attention gets its keys and values from a callback."""

    def __init__(self, config, weights):
        self.c = config
        self.w = {k: v.double().cpu().numpy() for k, v in weights.items()}

    def _norm(self, x, w):
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + self.c.norm_eps) * w

    def _rope(self, x, positions):
        d = x.shape[-1]
        angle = np.asarray(positions, np.float64)[:, None, None] * self.c.rope_theta ** (-np.arange(0, d, 2) / d)
        a, b = x[..., 0::2], x[..., 1::2]
        return np.stack([a * np.cos(angle) - b * np.sin(angle), a * np.sin(angle) + b * np.cos(angle)], -1).reshape(x.shape)

    def run(self, tokens, positions, attend):
        """attend(layer, q [n, Hq, D], k, v [n, Hkv, D]) -> [n, Hq, D]; returns logits [n, vocab] and each layer's k, v."""
        c, w = self.c, self.w
        x = w["tok_embeddings.weight"][np.asarray(tokens)]
        n, made = len(x), []
        for i in range(c.n_layers):
            def mul(a, name):
                return a @ w[f"layers.{i}.{name}.weight"].T
            a = self._norm(x, w[f"layers.{i}.attention_norm.weight"])
            q = self._rope(mul(a, "attention.wq").reshape(n, c.n_heads, c.head_dim), positions)
            k = self._rope(mul(a, "attention.wk").reshape(n, c.n_kv_heads, c.head_dim), positions)
            v = mul(a, "attention.wv").reshape(n, c.n_kv_heads, c.head_dim)
            made.append((k, v))
            x = x + mul(attend(i, q, k, v).reshape(n, -1), "attention.wo")
            a = self._norm(x, w[f"layers.{i}.ffn_norm.weight"])
            h = mul(a, "feed_forward.w1")
            x = x + mul(h / (1 + np.exp(-h)) * mul(a, "feed_forward.w3"), "feed_forward.w2")
        return self._norm(x, w["norm.weight"]) @ w["output.weight"].T, made


def held(cache, layer, table, count):
    k = ref.rows_ref(numbers(cache.k_cache[layer]), cache.k_scale[layer].double().cpu().numpy(), table, count)
    v = ref.rows_ref(numbers(cache.v_cache[layer]), cache.v_scale[layer].double().cpu().numpy(), table, count)
    return k, v


def check_rows(cache, layer, table, first, made, tol):
    """Rows of positions first .. hold the model's k, v to half a step of e4m3, 2^-4 of a value or
    2^-10 of its block's scale (twice each: a later row of the block may round it again)."""
    n = len(made[0])
    k, v = held(cache, layer, table, first + n)
    for got, want, scale in ((k, made[0], cache.k_scale[layer]), (v, made[1], cache.v_scale[layer])):
        s = scale.cpu().numpy()[np.asarray(table)].max(0)[None, :, None]
        assert np.all(np.abs(got[first:] - want) <= 2 * (2.0 ** -4 * np.abs(want) + 2.0 ** -10 * s) + tol)


def build(dtype, write_before_attend=True):
    from tinyvllm_amd.llama import Llama, LlamaConfig, random_weights
    config = LlamaConfig(dim=256, n_layers=2, n_heads=4, n_kv_heads=2, vocab_size=512, hidden_dim=512, max_seq_len=256,
                         dtype=dtype)
    weights = random_weights(config, seed=3, std=0.06)
    return config, Llama(config, weights, write_before_attend=write_before_attend), Model64(config, weights)


@gpu
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("bs,before", [(16, True), (16, False), (5, True)])
def test_prompt_chunk_and_steps(dtype, bs, before):
    from tinyvllm_amd.block_manager import BlockManager
    from tinyvllm_amd.kv_cache import FP8KVCache
    from tinyvllm_amd.sampling import token_logprobs
    config, model, exact = build(dtype, before)
    tol = TOL[dtype]
    scale = 1 / math.sqrt(config.head_dim)
    cache = FP8KVCache(config.n_layers, 64, bs, config.n_kv_heads, config.head_dim, dtype)
    manager = BlockManager(1, 64, bs)
    rng = np.random.Generator(np.random.PCG64(71))
    prompts = {0: rng.integers(0, 512, 45), 7: rng.integers(0, 512, 18)}
    for sid, tokens in prompts.items():
        manager.register_sequence(sid)
        first = 29 if sid == 0 else len(tokens)
        got = model.prefill(tokens[:first], cache, manager, sid)
        want, made = exact.run(tokens[:first], range(first), lambda i, q, k, v: ref.attend_ref(q, k, v, 0, scale)[0])
        assert np.abs(got[0].double().cpu().numpy() - want).max() <= tol
        table = manager.get_block_table(sid)
        for i in range(config.n_layers):
            check_rows(cache, i, table, 0, made[i], tol)
        check_logprobs(token_logprobs(got[0, :-1], torch.from_numpy(tokens[1:first].astype(np.int32)).cuda(), 5),
                       got[0, :-1].double().cpu().numpy(), tokens[1:first], 5)
        if first < len(tokens):
            got = model.prefill(tokens[first:], cache, manager, sid, first, attend_prefix=True)
            table = manager.get_block_table(sid)
            want, made = exact.run(tokens[first:], range(first, len(tokens)), lambda i, q, k, v: ref.attend_ref(
                q, *held(cache, i, table, len(tokens)), first, scale)[0])
            assert np.abs(got[0].double().cpu().numpy() - want).max() <= tol
            for i in range(config.n_layers):
                check_rows(cache, i, table, first, made[i], tol)

    jit = model.create_jit_decode(bs)
    ids = list(prompts)
    tokens = np.array([5, 9])
    for step in range(4):
        pos = [manager.get_context_length(s) for s in ids]
        ctx = [p + (1 if before else 0) for p in pos]
        for s, p in zip(ids, pos):
            manager.ensure_block_for_position(s, p)
        tables = np.zeros((2, 16), np.int32)
        for row, s in zip(tables, ids):
            t = manager.get_block_table(s)
            row[:len(t)] = t
        was = [[held(cache, i, manager.get_block_table(s), n) for s, n in zip(ids, ctx)] for i in range(config.n_layers)]
        logits = model.decode(torch.tensor(tokens[:, None]), cache, manager, ids, pos, torch.from_numpy(tables),
                              torch.tensor(ctx, dtype=torch.int32), jit, 16)[:, 0]
        if before:
            was = [[held(cache, i, manager.get_block_table(s), n) for s, n in zip(ids, ctx)]
                   for i in range(config.n_layers)]
        want, made = exact.run(tokens, pos, lambda i, q, k, v: np.stack(
            [ref.attend_ref(q[b:b + 1], *was[i][b], ctx[b] - 1, scale)[0][0] for b in range(2)]))
        assert np.abs(logits.double().cpu().numpy() - want).max() <= tol
        for i in range(config.n_layers):
            for b, s in enumerate(ids):
                check_rows(cache, i, manager.get_block_table(s), pos[b], [x[b:b + 1] for x in made[i]], tol)
        tokens = logits.argmax(-1).cpu().numpy()
        scored = token_logprobs(logits, torch.from_numpy(tokens.astype(np.int32)).cuda(), 3)
        check_logprobs(scored, logits.double().cpu().numpy(), tokens, 3)
        assert np.array_equal(scored.top_ids[:, 0].cpu().numpy(), tokens)


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_device_loop_equals_single_steps(dtype):
    """``DecodeGraph.run(n)`` over an 8-bit cache: the same tokens, numbers and scales as n calls."""
    from tinyvllm_amd.kv_cache import FP8KVCache
    from tinyvllm_amd.llama import DecodeGraph
    config, model, _ = build(dtype)
    results = []
    for eager in (True, False):
        cache = FP8KVCache(config.n_layers, 40, 16, config.n_kv_heads, config.head_dim, dtype)
        tables = torch.arange(24, dtype=torch.int32).view(3, 8).cuda()
        for b in range(3):
            model.prefill_table(torch.arange(20 + b), cache, tables[b], logits=None)
        g = DecodeGraph(model, cache, 3, 8, history_len=64)
        g.set_inputs([1, 2, 3], [20, 21, 22], [21, 22, 23], tables)
        if eager:
            for _ in range(20):
                g.step_eager()
        else:
            g.run(20)
        torch.cuda.synchronize()
        results.append([g.history.clone(), g.logits.clone(), g.positions.clone()] +
                       [t.view(torch.uint8).clone() for t in cache.k_cache + cache.v_cache] +
                       [t.clone() for t in cache.k_scale + cache.v_scale])
        g.close()
    assert all(torch.equal(a, b) for a, b in zip(*results))


@gpu
@pytest.mark.parametrize("kind", ["FP8KVCache", "KVCache"])
def test_a_captured_step_keeps_its_cache(kind):
    """The steps of a decode are kept by the cache they were captured for: neither its memory nor its
    identity may pass to another cache before they are gone."""
    import gc
    import weakref
    from tinyvllm_amd import kv_cache
    config, model, _ = build("float16")

    def make():
        return getattr(kv_cache, kind)(config.n_layers, 4, 16, config.n_kv_heads, config.head_dim, "float16")
    jit = model.create_jit_decode(16)
    first = make()
    storage = first.k_cache[0].data_ptr()
    graph = jit.graph_for(first, 2, 2)
    seen = weakref.ref(first)
    del first
    gc.collect()
    assert seen() is not None
    second = make()
    assert second.k_cache[0].data_ptr() != storage and jit.graph_for(second, 2, 2) is not graph
    del graph, jit, second
    gc.collect()
    assert seen() is None


def test_cache_struct_is_validated_on_the_host():
    """One scale array of two, and slots past 32 bits, are refused before any launch."""
    from tinyvllm_amd import _lib
    from tinyvllm_amd.llama import _Cache, _DecodeArgs, _Model, _PP
    lib = _lib.load()
    p = (ctypes.c_void_p * 1)(256)
    pp = ctypes.cast(p, _PP)
    m = _Model(1, 64, 1, 1, 64, 64, 64, _lib.TV_F16, 1e-5, 256, pp, pp, pp, pp, pp, pp, 256, 256, 256, 16)
    args = _DecodeArgs(1, 256, 256, 256, 256, 4, 4, 64, 1, None, None, 0, None, 0)
    for cache, what in ((_Cache(pp, pp, 8, 16, pp, None), b"both scale arrays"),
                        (_Cache(pp, pp, 1 << 28, 16, pp, pp), b"32 bits"), (_Cache(None, pp, 8, 16), b"bad cache")):
        rc = lib.tv_llama_decode_step(ctypes.byref(m), ctypes.byref(cache), ctypes.byref(args), None)
        assert rc != _lib.TV_OK and what in lib.tv_last_error()
