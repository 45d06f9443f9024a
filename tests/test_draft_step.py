"""A whole verified step: layout, rotated cache write, tree attention, verdict and kept rows in the place of single-token
steps of the model, whose tokens and cache it has to reproduce."""

import numpy as np
import pytest
import torch

from tests.test_draft_tree import cuda, gpu, rng_of


def build(dtype, **kw):
    from tinyvllm_amd.llama import Llama, LlamaConfig
    config = LlamaConfig(dim=256, n_layers=2, n_heads=4, n_kv_heads=2, vocab_size=512, hidden_dim=512, max_seq_len=256,
                         dtype=dtype, **kw)
    model = Llama(config, seed=3)
    rng = rng_of(17)                                  # projections that matter: 0.02 would leave all logits alike
    from tinyvllm_amd.llama import weight_shapes
    model.load_weights({n: torch.from_numpy(rng.standard_normal(s).astype(np.float32) * (s[-1] ** -0.5))
                        for n, s in weight_shapes(config).items() if len(s) == 2})
    return model


class Sequences:
    """Sequences in a cache with a block manager, decoded token by token by the model."""

    def __init__(self, model, prompts, blocks=64, bs=16):
        from tinyvllm_amd.block_manager import BlockManager
        from tinyvllm_amd.kv_cache import KVCache
        c = model.config
        self.model, self.bs = model, bs
        self.cache = KVCache(c.n_layers, blocks, bs, c.n_kv_heads, c.head_dim, c.dtype)
        self.manager = BlockManager(1, blocks, bs)
        self.jit = model.create_jit_decode(bs)
        self.next = []
        for i, p in enumerate(prompts):
            self.manager.register_sequence(i)
            logits = model.prefill(np.asarray(p), self.cache, self.manager, i)
            self.next.append(int(logits[0, -1].argmax()))
        self.ids = list(range(len(prompts)))

    def tables(self, spare=0, width=12):
        for i in self.ids:
            self.manager.ensure_block_for_position(i, self.manager.get_context_length(i) + spare)
        return self.manager.prepare_batch_tensors(self.ids, [self.manager.get_context_length(i) for i in self.ids], width)

    def step(self):
        """One token of every sequence; logits [B, V]."""
        table, lens = self.tables()
        start = [self.manager.get_context_length(i) for i in self.ids]
        logits = self.model.decode(np.asarray(self.next), self.cache, self.manager, self.ids, start, table, lens, self.jit, 12)
        self.next = logits[:, 0].argmax(1).tolist()
        return logits[:, 0]


def norm(x, w, eps):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * w


def verified_step(seqs, tokens, parents, lens, **kw):
    """tokens / parents [B, T], lens [B] -> (logits [B, T, V], verdict); the kept path's K/V are in place after it."""
    from tinyvllm_amd.attention import paged_tree_attention
    from tinyvllm_amd.draft_tree import draft_tree_layout
    from tinyvllm_amd.sampling import verify_draft_tree
    m, c, cache = seqs.model, seqs.model.config, seqs.cache
    b, t = tokens.shape
    hq, hkv, d, h = c.n_heads, c.n_kv_heads, c.head_dim, c.hidden_dim
    table, _ = seqs.tables(spare=t)
    ctx = cuda(np.asarray([seqs.manager.get_context_length(i) for i in seqs.ids], np.int32))
    table, parents, lens = cuda(table), cuda(parents), cuda(lens)
    layout = draft_tree_layout(parents, lens, ctx, table, seqs.bs, cache.num_blocks)
    x = m.tok_embeddings[cuda(tokens).long()].float().view(b * t, -1)
    for i in range(c.n_layers):
        qkv = (norm(x, m.attention_norm[i], c.norm_eps) @ m.wqkv[i].float().T).to(c.dtype)
        q, k, v = (y.unflatten(1, (-1, d)) for y in qkv.split([hq * d, hkv * d, hkv * d], 1))
        q = cache.write_rope_slots(i, layout.slots, layout.positions, m.rope, q, k, v)
        o = paged_tree_attention(q.view(b, t, hq, d), cache.k_cache[i], cache.v_cache[i], table, ctx, lens, layout.mask, hq,
                                 hkv, d, seqs.bs)
        x = x + o.float().view(b * t, -1) @ m.wo[i].float().T
        w13 = m.w13[i].float().view(h // 2, 2, 2, c.dim)
        w1, w3 = w13[:, 0].reshape(h, c.dim), w13[:, 1].reshape(h, c.dim)
        y = norm(x, m.ffn_norm[i], c.norm_eps)
        x = x + (torch.nn.functional.silu(y @ w1.T) * (y @ w3.T)) @ m.w2[i].float().T
    logits = (norm(x, m.norm, c.norm_eps) @ m.output.float().T).view(b, t, -1)
    verdict = verify_draft_tree(logits, cuda(tokens), parents, lens, **kw)
    cache.keep_draft_path(verdict.path, verdict.counts, ctx, table)
    for i, n in zip(seqs.ids, verdict.counts.tolist()):
        for _ in range(n):
            seqs.manager.advance_position(i)
    return logits, verdict


def drafted(rng, first, greedy, t, right):
    """A tree over the tokens `greedy` that follow `first`: the first `right` of them along a path, with wrong siblings."""
    tokens, parents = np.zeros(t, np.int32), np.full(t, -1, np.int32)
    tokens[0], at, path = first, 0, [0]
    for j in range(1, t):
        on = rng.random() < 0.6 and len(path) <= right
        parents[j] = path[-1] if on else rng.integers(0, j)
        tokens[j] = greedy[len(path) - 1] if on else rng.integers(0, 512)
        if on:
            path.append(j)
    return tokens, parents, path


@gpu
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_verified_steps_are_the_model_s_own(dtype):
    """Greedy: the accepted tokens and the next one are those of single-token steps, and so is what the cache holds then."""
    model = build(dtype)
    rng = rng_of(5)
    prompts = [rng.integers(0, 512, n) for n in (5, 16, 37)]
    single, tree = Sequences(model, prompts), Sequences(model, prompts)
    assert single.next == tree.next
    greedy = [list(single.next)]
    steps = []
    for _ in range(24):
        steps.append(single.step())
        greedy.append(list(single.next))
    scale = float(max(s.abs().max() for s in steps))
    done = np.zeros(3, int)                                       # tokens that the tree side has cached beyond the prompt
    for right in (3, 0, 5):
        trees = [drafted(rng, greedy[done[b]][b], [g[b] for g in greedy[done[b] + 1:]], 14, right) for b in range(3)]
        tokens, parents = np.stack([x[0] for x in trees]), np.stack([x[1] for x in trees])
        logits, verdict = verified_step(tree, tokens, parents, np.full(3, 14, np.int32))
        counts = verdict.counts.tolist()
        for b in range(3):
            path = verdict.path[b, :counts[b]].tolist()
            for j, node in enumerate(path):
                # the model's logits at this position; 2e-2 of their scale is what its step is held to
                assert float((logits[b, node] - steps[done[b] + j][b]).abs().max()) < (1e-4 if dtype == "float32" else 2e-2) * scale
            if dtype == "float32":                                # margins of greedy tokens are far above fp32's errors
                assert counts[b] >= len(trees[b][2]) and path[:len(trees[b][2])] == trees[b][2]
                assert [int(tokens[b, n]) for n in path] == [greedy[done[b] + j][b] for j in range(counts[b])]
                assert int(verdict.next_tokens[b]) == greedy[done[b] + counts[b]][b]
        if dtype != "float32":
            return
        done += counts
        tree.next = verdict.next_tokens.tolist()
    # the cache is as if it had been written token by token: the next single step's logits are the same
    more = tree.step()
    for b in range(3):
        assert float((more[b] - steps[done[b]][b]).abs().max()) < 1e-4 * scale


@gpu
def test_sampled_steps_accept_what_is_likely():
    """A sampled verdict over the model's own logits agrees with the definition in float64."""
    from oracle.draft_tree import verify_ref
    model = build("float32")
    rng = rng_of(6)
    seqs = Sequences(model, [rng.integers(0, 512, n) for n in (9, 20)])
    tokens = rng.integers(0, 512, (2, 40)).astype(np.int32)
    tokens[:, 0] = seqs.next
    parents = np.stack([np.concatenate([[-1], rng.integers(0, np.arange(1, 40))]) for _ in range(2)]).astype(np.int32)
    lens = np.array([40, 31], np.int32)
    temps, u = np.array([1.5, 0.8], np.float32), rng.random((2, 40)).astype(np.float32)
    logits, verdict = verified_step(seqs, tokens, parents, lens, temperatures=cuda(temps), uniforms=cuda(u))
    path, counts, follow, near = verify_ref(logits.double().cpu().numpy(), tokens, parents, lens, temps, u)
    assert (near > 2.0 ** -32).all()
    for got, want in zip(verdict, (path, counts, follow)):
        assert np.array_equal(got.cpu().numpy(), want)


@gpu
def test_rows_of_a_cache_of_more_than_4_gib():
    """Writes and moves beyond 2^32 bytes and 2^31 elements are those in a small cache."""
    from tinyvllm_amd.kv_cache import keep_draft_rows, rope_and_cache
    from tests.test_rope_cache import table_of
    rng = rng_of(8)
    n, hq, hkv, d, bs, nb = 20, 4, 2, 128, 16, 6
    first = (1 << 31) // (bs * hkv * d)
    small = [torch.from_numpy(rng.standard_normal((nb, bs, hkv, d))).to("cuda", torch.bfloat16) for _ in range(2)]
    large = [torch.empty((first + nb, bs, hkv, d), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    for x, y in zip(large, small):
        x[first:] = y
    q, k, v = (torch.from_numpy(rng.standard_normal((n, h, d))).to("cuda", torch.bfloat16) for h in (hq, hkv, hkv))
    slots, positions = rng.permutation(nb * bs)[:n].astype(np.int32), np.arange(n, dtype=np.int32)
    path, counts = np.array([[0, 3, 4, 11] + [-1] * 8], np.int32), np.array([4], np.int32)
    ctx, table = np.array([21], np.int32), rng.permutation(nb).astype(np.int32)[None]
    for caches, base in ((small, 0), (large, first)):
        rope_and_cache(*caches, q, k, v, cuda(slots + np.int32(base * bs)), cuda(positions), cuda(table_of(64, d)))
        keep_draft_rows(caches[:1], caches[1:], cuda(path), cuda(counts), cuda(ctx), cuda(table + np.int32(base)))
    for x, y in zip(large, small):
        assert torch.equal(x[first:], y)


@gpu
def test_a_step_in_one_graph():
    """Layout, write, attention, verdict and kept rows captured together: replays follow their inputs and agree with eager calls."""
    from tinyvllm_amd.attention import PagedTreePlan
    from tinyvllm_amd.draft_tree import draft_tree_layout
    from tinyvllm_amd.kv_cache import keep_draft_rows, rope_and_cache
    from tinyvllm_amd.sampling import verify_draft_tree
    from tests.test_draft_tree import random_tree
    from tests.test_rope_cache import table_of
    rng = rng_of(7)
    b, t, hq, hkv, d, bs, nb, v = 4, 12, 4, 2, 64, 16, 64, 300
    bufs = {"parents": torch.zeros((b, t), dtype=torch.int32), "tokens": torch.zeros((b, t), dtype=torch.int32),
            "lens": torch.zeros(b, dtype=torch.int32), "ctx": torch.zeros(b, dtype=torch.int32),
            "table": torch.zeros((b, nb // b), dtype=torch.int32), "qkv": torch.zeros((b * t, (hq + 2 * hkv) * d)),
            "logits": torch.zeros((b, t, v)), "k": torch.zeros((nb, bs, hkv, d)), "v": torch.zeros((nb, bs, hkv, d))}
    bufs = {n: x.cuda() for n, x in bufs.items()}
    rope = cuda(table_of(512, d))
    turned = torch.zeros((b * t, hq, d), device="cuda")
    mask = torch.zeros((b, t, 1), dtype=torch.int64, device="cuda")
    plan = PagedTreePlan(turned.view(b, t, hq, d), bufs["k"], bufs["v"], bufs["table"], bufs["ctx"], bufs["lens"], mask, hq, hkv,
                         d, bs, work_groups=16)

    def step():
        q, k, x = (y.unflatten(1, (-1, d)) for y in bufs["qkv"].split([hq * d, hkv * d, hkv * d], 1))
        layout = draft_tree_layout(bufs["parents"], bufs["lens"], bufs["ctx"], bufs["table"], bs, nb)
        mask.copy_(layout.mask)
        rope_and_cache(bufs["k"], bufs["v"], q, k, x, layout.slots, layout.positions, rope, out=turned)
        out = plan.run()
        verdict = verify_draft_tree(bufs["logits"], bufs["tokens"], bufs["parents"], bufs["lens"])
        keep_draft_rows([bufs["k"]], [bufs["v"]], verdict.path, verdict.counts, bufs["ctx"], bufs["table"])
        return out, *verdict, bufs["k"], bufs["v"]

    def fill(seed):
        r = rng_of(seed)
        new = {"parents": random_tree(r, b, t), "tokens": r.integers(0, 5, (b, t)), "lens": r.integers(0, t + 1, b),
               "ctx": r.integers(0, 200, b), "table": r.permutation(nb).reshape(b, -1),
               "qkv": r.standard_normal((b * t, (hq + 2 * hkv) * d)), "k": r.standard_normal((nb, bs, hkv, d)),
               "logits": r.standard_normal((b, t, v)) + (np.arange(v) < 5) * 3.0, "v": r.standard_normal((nb, bs, hkv, d))}
        for n, x in new.items():
            bufs[n].copy_(torch.from_numpy(np.ascontiguousarray(x)))

    fill(0)
    step()
    torch.cuda.synchronize()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        held = step()
    for seed in range(1, 5):
        fill(seed)
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in held]
        fill(seed)
        want = step()
        torch.cuda.synchronize()
        for a, x in zip(got, want):
            assert torch.equal(a, x)
