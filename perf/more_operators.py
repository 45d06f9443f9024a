"""Drafted tokens verified several at a time, as cases that can be timed and checked.

A draft gives every sequence a tree of tokens: node 0 is the token that the sequence has last got, every
other node continues its parent.  Five operators, in the order in which a step meets them:

* ``layout`` -- what each node sees, its position and its place in the cache, from the parents
  (``draft_tree_layout``);
* ``append`` -- queries and keys are rotated to their positions, keys and values written into the paged
  cache (``rope_and_cache``);
* ``tree``   -- attention of all nodes over the cached context and the nodes before them
  (``paged_tree_attention``, or the ``PagedTreePlan`` that a loop keeps);
* ``verify`` -- the path that the model's logits accept, and the token after it (``verify_draft_tree``);
* ``keep``   -- the accepted path's keys and values move to where the sequence goes on
  (``keep_draft_rows``).

Definitions.  A parent is a lower index of the same tree or -1; nodes at ``tree_lens`` and beyond are
padding.  ``mask[b, i]`` holds bit t of word t // 64 for t = i and all its ancestors; node i stands at position
``context + depth`` and its K/V at cache row ``context + i`` of the sequence.  A node attends all context
rows and the rows of its mask.  From node 0 on, a greedy verdict goes to the first child whose token is the first
maximum of the node's logits; a sampled one draws u per node and goes to the first child at which the children's
probabilities (softmax of logits / temperature, in the children's order) sum to more than u.  Where there is no such
child the path ends, and the next token is the maximum, or the one at which the probabilities of the
tokens that no child has sum, in the vocabulary's order, to more than (u - c) / (1 - c) of theirs, c being the
children's.

With ``own`` false everything is computed by elementary torch operations in 32 bits; the
probabilities that a draw is compared with in 64.
"""

import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}

# (query heads, KV heads, head size): TinyLlama, Llama-3-8B, its 4-way shard, and the generic
# layouts without shared KV heads, with five heads to a group and with heads of 256
HEADS = {"tinyllama": (32, 4, 64), "llama3_8b": (32, 8, 128), "llama3_8b_shard": (8, 2, 128),
         "single": (12, 12, 64), "five": (40, 8, 128), "wide": (8, 1, 256)}

POSITIONS = 16384           # rows of the rotation table (32-bit cos and sin)


def listed():
    return [
        # Four conversations with short drafts.
        {"name": "layout_few", "kind": "layout", "batch": 4, "nodes": 8, "ctx_max": 250, "block": 16},
        # A full serving batch with wide drafts.
        {"name": "layout_batch", "kind": "layout", "batch": 256, "nodes": 64, "ctx_max": 4000, "block": 16},
        # The same four conversations in the reference's default type.
        {"name": "append_f32_few", "kind": "append", "dtype": "float32", "heads": "tinyllama", "block": 16, "batch": 4,
         "nodes": 8, "ctx_max": 250, "pairs": "adjacent", "share": 1.0},
        # Sixty-four sequences, each with a draft of up to 32 nodes; weights that pair halves.
        {"name": "append_bf16_batch", "kind": "append", "dtype": "bfloat16", "heads": "llama3_8b", "block": 16,
         "batch": 64, "nodes": 32, "ctx_max": 300, "pairs": "halves", "share": 1.0},
        # Four short conversations in the reference's default type.
        {"name": "tree_f32_few", "kind": "tree", "dtype": "float32", "heads": "tinyllama", "block": 16, "batch": 4,
         "nodes": 8, "ctx_min": 17, "ctx_max": 250, "plan": False},
        # A serving batch of mixed context lengths, as a captured loop launches it.
        {"name": "tree_f16_batch", "kind": "tree", "dtype": "float16", "heads": "llama3_8b", "block": 16, "batch": 64,
         "nodes": 16, "ctx_min": 512, "ctx_max": 4096, "plan": True},
        # Wide drafts: many rows to every key.
        {"name": "tree_bf16_wide", "kind": "tree", "dtype": "bfloat16", "heads": "tinyllama", "block": 16, "batch": 32,
         "nodes": 61, "ctx_min": 1000, "ctx_max": 6000, "plan": True},
        # Two sequences of very long context.
        {"name": "tree_bf16_long", "kind": "tree", "dtype": "bfloat16", "heads": "llama3_8b", "block": 16, "batch": 2,
         "nodes": 32, "ctx_min": 31000, "ctx_max": 32700, "plan": False},
        # A serving batch that decodes greedily.
        {"name": "verify_f32_greedy", "kind": "verify", "dtype": "float32", "batch": 64, "nodes": 16, "vocab": 32000,
         "longest": 6, "temperature": 0.0},
        # Two sequences that sample from a large vocabulary.
        {"name": "verify_bf16_sampled", "kind": "verify", "dtype": "bfloat16", "batch": 2, "nodes": 32, "vocab": 128256,
         "longest": 5, "temperature": 0.8},
        # Four conversations of a small model.
        {"name": "keep_f32_few", "kind": "keep", "dtype": "float32", "heads": "tinyllama", "block": 16, "layers": 22,
         "batch": 4, "nodes": 8, "ctx_max": 60, "longest": 4},
        # A serving batch of a larger one.
        {"name": "keep_bf16_batch", "kind": "keep", "dtype": "bfloat16", "heads": "llama3_8b", "block": 16, "layers": 32,
         "batch": 64, "nodes": 48, "ctx_max": 40, "longest": 16},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["layout", "append", "append", "tree", "tree", "tree", "verify", "verify", "keep"])
    dtype = rng.choice(["float32", "float16", "bfloat16"])
    block = rng.choice([16, 16, 16, 32, 8])
    heads = rng.choice(sorted(HEADS))
    hq, hkv, d = HEADS[heads]
    if kind == "layout":
        nodes = _log_int(rng, 1, 256)
        return {"kind": kind, "batch": _log_int(rng, 1, min(256, 16384 // nodes)), "nodes": nodes,
                "ctx_max": _log_int(rng, 1, 4000), "block": block}
    if kind == "append":
        nodes = _log_int(rng, 1, 64)
        return {"kind": kind, "dtype": dtype, "heads": heads, "block": block, "nodes": nodes,
                "batch": _log_int(rng, 1, max(1, min(64, (24 << 20) // (DTYPES[dtype].itemsize * nodes * (hq + 2 * hkv) * d)))),
                "ctx_max": _log_int(rng, 1, 300),
                "pairs": rng.choice(["adjacent", "halves"]), "share": rng.choice([1.0, 1.0, 0.5])}
    if kind == "tree":
        nodes = _log_int(rng, 1, 128)
        batch = _log_int(rng, 1, 64)
        es = DTYPES[dtype].itemsize
        most = min(32000, (1 << 29) // (2 * es * hkv * d * batch), (1 << 28) // (hq * nodes * batch),
                   (1 << (31 if dtype == "float32" else 33)) // (hq * d * nodes * batch))
        ctx = _log_int(rng, 16, max(17, most))
        return {"kind": kind, "dtype": dtype, "heads": heads, "block": block, "batch": batch, "nodes": nodes,
                "ctx_min": max(0, int(ctx * rng.uniform(0.1, 1.0))), "ctx_max": ctx, "plan": rng.random() < 0.5}
    if kind == "verify":
        vocab, nodes = _log_int(rng, 1000, 128256), _log_int(rng, 1, 64)
        return {"kind": kind, "dtype": dtype, "batch": _log_int(rng, 1, max(1, min(128, (1 << 25) // (vocab * nodes)))),
                "nodes": nodes, "vocab": vocab, "longest": rng.choice([0, 2, 4, 8]),
                "temperature": rng.choice([0.0, 0.6, 1.0])}
    nodes, layers = _log_int(rng, 2, 64), rng.choice([2, 22, 32])
    batch = _log_int(rng, 1, max(1, min(64, (1 << 27) // (layers * hkv * d * (nodes + 60)))))
    return {"kind": kind, "dtype": dtype, "heads": heads, "block": block, "layers": layers, "batch": batch,
            "nodes": nodes, "ctx_max": 40, "longest": rng.choice([1, 4, 8, 16])}


# ---- inputs -------------------------------------------------------------------------

def _ints(seed, stream):
    return np.random.Generator(np.random.PCG64([seed, stream]))


def _floats(seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    return gen


def _normal(gen, shape, dtype):
    return torch.randn(shape, generator=gen, dtype=dtype, device=DEVICE)


def _device(x):
    return torch.from_numpy(np.ascontiguousarray(x)).to(DEVICE)


def _dealt(x, seed, stream):
    """Numbers (or rows) that belong to the case, in the seed's order."""
    return x[_ints(seed, stream).permutation(len(x))]


def _trees(case):
    """Trees as a draft grows them, level by level: (parents [B, T], lens [B]), depths of up to eight; the case's own."""
    rng = _ints(0, 11)
    b, t = case["batch"], case["nodes"]
    lens = rng.integers(max(1, (3 * t) // 4), t + 1, b).astype(np.int32)
    level = np.maximum(1, -(-t // 8))
    parents = np.full((b, t), -1, np.int32)
    for i in range(1, t):
        d = (i - 1) // level + 1                         # depth of node i
        lo = 0 if d == 1 else (d - 2) * level + 1
        hi = 1 if d == 1 else (d - 1) * level + 1
        parents[:, i] = rng.integers(lo, hi, b)
    return parents, lens


def _contexts(case):
    return _ints(0, 1).integers(case.get("ctx_min", 0), case["ctx_max"] + 1, case["batch"]).astype(np.int32)


def _tables(rows, block, seed):
    """Block tables of sequences of `rows` positions over a shuffled pool with a tenth to spare."""
    need = -(-np.asarray(rows, dtype=np.int64) // block)
    pool = int(need.sum() * 1.1) + 1
    perm = _ints(seed, 2).permutation(pool).astype(np.int32)
    table = np.zeros((len(need), int(need.max())), np.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = perm[at:at + n]
        at += n
    return table, pool


def _batch(case, seed):
    """(parents, lens, ctx, table, pool) on the host: the case's sequences in the seed's order."""
    parents, lens = _trees(case)
    order = _ints(seed, 3).permutation(case["batch"])
    parents, lens, ctx = parents[order], lens[order], _dealt(_contexts(case), seed, 4)
    table, pool = _tables(ctx + case["nodes"], case["block"], seed)
    return parents, lens, ctx, table, pool


def _words(parents, lens):
    """Mask words [B, T, W] int64 and depths [B, T] of trees, on the host."""
    b, t = parents.shape
    seen = np.zeros((b, t, -(-t // 64) * 64), bool)
    depth = np.zeros((b, t), np.int32)
    rows = np.arange(b)
    for i in range(t):
        p = parents[:, i]
        has = (p >= 0)[:, None]
        seen[:, i] = seen[rows, np.maximum(p, 0)] & has
        depth[:, i] = np.where(p >= 0, depth[rows, np.maximum(p, 0)] + 1, 0)
        seen[:, i, i] = True
    dead = np.arange(t) >= lens[:, None]
    seen[dead] = False
    depth[dead] = 0
    return np.packbits(seen, axis=2, bitorder="little").view(np.int64), depth


def _layout_inputs(case, seed):
    parents, lens, ctx, table, pool = _batch(case, seed)
    return {"parents": _device(parents), "lens": _device(lens), "ctx": _device(ctx), "table": _device(table),
            "block": case["block"], "pool": pool}


def _append_inputs(case, seed):
    """q, k, v of all nodes of a batch, as the rows of one projection."""
    hq, hkv, d = HEADS[case["heads"]]
    dtype, block = DTYPES[case["dtype"]], case["block"]
    parents, lens, ctx, table, pool = _batch(case, seed)
    _, depth = _words(parents, lens)
    live = np.arange(case["nodes"]) < lens[:, None]
    at = ctx[:, None] + np.arange(case["nodes"])
    slots = np.take_along_axis(table, at // block, 1).astype(np.int64) * block + at % block
    gen = _floats(seed)
    n = int(live.sum())
    qkv = _normal(gen, (n, (hq + 2 * hkv) * d), dtype)
    q, k, v = (x.unflatten(1, (-1, d)) for x in qkv.split([hq * d, hkv * d, hkv * d], 1))
    turned = int(d * case["share"])
    freq = 10000.0 ** (-torch.arange(0, turned, 2, dtype=torch.float64, device=DEVICE) / turned)
    angle = torch.arange(POSITIONS, dtype=torch.float64, device=DEVICE)[:, None] * freq
    return {"q": q, "k": k, "v": v, "rope": torch.stack([angle.cos(), angle.sin()], 2).float(),
            "slots": _device(slots[live].astype(np.int32)), "positions": _device((ctx[:, None] + depth)[live]),
            "k_cache": _normal(gen, (pool, block, hkv, d), dtype), "v_cache": _normal(gen, (pool, block, hkv, d), dtype),
            "pairs": case["pairs"]}


def _tree_inputs(case, seed):
    hq, hkv, d = HEADS[case["heads"]]
    dtype = DTYPES[case["dtype"]]
    parents, lens, ctx, table, pool = _batch(case, seed)
    gen = _floats(seed)
    q = _normal(gen, (case["batch"], case["nodes"], hq, d), dtype)
    k = _normal(gen, (pool, case["block"], hkv, d), dtype)
    k[..., ::8] *= 2                                     # some channels of keys stand out
    return {"q": q, "k_cache": k, "v_cache": _normal(gen, k.shape, dtype), "table": _device(table), "ctx": _device(ctx),
            "lens": _device(lens), "mask": _device(_words(parents, lens)[0]), "heads": (hq, hkv, d),
            "block": case["block"], "longest": int((ctx + case["nodes"]).max())}


def _paths(case, parents, lens, seed, stream):
    """Accepted paths of the case: (path [B, T], -1 beyond, counts [B]), each of up to `longest` drafted nodes."""
    rng = _ints(seed, stream)
    b, t = parents.shape
    path = np.full((b, t), -1, np.int32)
    counts = np.ones(b, np.int32)
    path[:, 0] = 0
    for i in range(b):
        for j in range(1, case["longest"] + 1):
            nodes = np.flatnonzero(parents[i, :lens[i]] == path[i, j - 1])
            if not len(nodes) or path[i, j - 1] < 0:
                break
            path[i, j] = rng.choice(nodes)
            counts[i] += 1
    return path, counts


def _verify_inputs(case, seed):
    """Logits as a trained model's head leaves them, a bulk of N(0, 2.5), whose likeliest token is a child's along a
    path of the tree and none of the children's at its end."""
    m, t, n = case["batch"], case["nodes"], case["vocab"]
    parents, lens = _trees(case)
    order = _ints(seed, 3).permutation(m)
    parents, lens = parents[order], lens[order]
    rng = _ints(seed, 5)
    tokens = np.stack([rng.choice(n, t + 1, replace=False) for _ in range(m)]).astype(np.int32)
    path, counts = _paths(case, parents, lens, seed, 6)
    rows = np.arange(m)
    likely = rng.integers(0, n, (m, t))
    for j in range(int(counts.max())):
        on = counts > j
        more = counts > j + 1
        follow = tokens[rows, np.where(more, path[:, min(j + 1, t - 1)], t)]
        likely[rows[on], path[on, j]] = follow[on]
    gen = _floats(seed)
    x = torch.randn((m, t, n), generator=gen, device=DEVICE) * 2.5
    temp = case["temperature"]
    height = 16.0 if temp == 0 else temp * (math.log(n) + (2.5 / temp) ** 2 / 2 + 2.5)      # e^2.5 times all the others
    x.scatter_(2, _device(likely)[:, :, None], height)
    state = {"logits": x.to(DTYPES[case["dtype"]]), "tokens": _device(tokens[:, :t]), "parents": _device(parents),
             "lens": _device(lens), "uniforms": None, "temperatures": None}
    if temp > 0:
        # requests set their own; every fourth decodes greedily
        temps = np.where(np.arange(m) % 4 == 3, 0.0, temp).astype(np.float32)
        state["uniforms"] = torch.rand((m, t), generator=gen, device=DEVICE)
        state["temperatures"] = _device(temps)
    return state


def _keep_paths(case):
    """Paths that go down the tree's first nodes, then over to nodes behind the kept rows (so that a second pass over
    the same rows changes nothing): (path [B, T], counts [B]); the case's own."""
    rng = _ints(0, 7)
    b, t = case["batch"], case["nodes"]
    path = np.full((b, t), -1, np.int32)
    counts = np.minimum(rng.integers(1, case["longest"] + 2, b), max(1, t // 2)).astype(np.int32)
    for i, n in enumerate(counts):
        same = int(rng.integers(1, n + 1))
        path[i, :same] = np.arange(same)
        path[i, same:n] = np.sort(rng.choice(np.arange(n, t), n - same, replace=False))
    return path, counts


def _keep_inputs(case, seed):
    _, hkv, d = HEADS[case["heads"]]
    path, counts = _keep_paths(case)
    order = _ints(seed, 3).permutation(case["batch"])
    ctx = _dealt(_contexts(case), seed, 4)
    table, pool = _tables(ctx + case["nodes"], case["block"], seed)
    rows = _normal(_floats(seed), (2, case["layers"], pool, case["block"], hkv, d), DTYPES[case["dtype"]])
    return {"rows": rows, "k": list(rows[0]), "v": list(rows[1]), "path": _device(path[order]),
            "counts": _device(counts[order]), "ctx": _device(ctx), "table": _device(table)}


_INPUTS = {"layout": _layout_inputs, "append": _append_inputs, "tree": _tree_inputs, "verify": _verify_inputs,
           "keep": _keep_inputs}


def prepare(case, seed):
    state = _INPUTS[case["kind"]](case, seed)
    state["kind"] = case["kind"]
    if case["kind"] == "tree":
        state["args"] = (state["q"], state["k_cache"], state["v_cache"], state["table"], state["ctx"], state["lens"],
                         state["mask"], *state["heads"], state["block"])
        if own and case["plan"]:
            from tinyvllm_amd.attention import PagedTreePlan
            state["plan"] = PagedTreePlan(*state["args"])
    return state


# ---- the framework's operators -------------------------------------------------------

def _run_own(state):
    kind = state["kind"]
    if kind == "layout":
        from tinyvllm_amd.draft_tree import draft_tree_layout
        return tuple(draft_tree_layout(state["parents"], state["lens"], state["ctx"], state["table"], state["block"],
                                       state["pool"]))
    if kind == "append":
        from tinyvllm_amd.kv_cache import rope_and_cache
        q = rope_and_cache(state["k_cache"], state["v_cache"], state["q"], state["k"], state["v"], state["slots"],
                           state["positions"], state["rope"], pairs=state["pairs"])
        return q, state["k_cache"], state["v_cache"]
    if kind == "tree":
        if "plan" in state:
            return state["plan"].run()
        from tinyvllm_amd.attention import paged_tree_attention
        return paged_tree_attention(*state["args"])
    if kind == "verify":
        from tinyvllm_amd.sampling import verify_draft_tree
        return tuple(verify_draft_tree(state["logits"], state["tokens"], state["parents"], state["lens"],
                                       temperatures=state["temperatures"], uniforms=state["uniforms"]))
    from tinyvllm_amd.kv_cache import keep_draft_rows
    keep_draft_rows(state["k"], state["v"], state["path"], state["counts"], state["ctx"], state["table"])
    return state["rows"]


# ---- the plain forms -------------------------------------------------------------------

def _ancestors(parents, lens):
    """[B, T, T] float: 1 where t is i or an ancestor of i; rows of padding are 0."""
    t = parents.shape[1]
    node = torch.arange(t, device=parents.device)
    live = (node < lens[:, None]).float()
    step = (parents[:, :, None] == node).float() * live[:, :, None]
    whole = torch.eye(t, device=parents.device)
    reach = whole + step                                 # up to one step, then two, four, ...
    for _ in range(max(1, (t - 1).bit_length()) - 1):
        step = torch.matmul(step, step)
        reach = torch.matmul(whole + step, reach)
    return reach * live[:, :, None]


def _plain_layout(state):
    lens, ctx, table, block = state["lens"], state["ctx"], state["table"], state["block"]
    seen = _ancestors(state["parents"], lens)
    b, t = seen.shape[:2]
    live = torch.arange(t, device=DEVICE) < lens[:, None]
    depth = (seen.sum(2) - 1).clamp_min(0).to(torch.int32)
    positions = torch.where(live, ctx[:, None] + depth, 0)
    bits = torch.nn.functional.pad(seen, (0, -t % 64)).to(torch.int64).view(b, t, -1, 64)
    mask = (bits << torch.arange(64, device=DEVICE)).sum(3)
    at = ctx[:, None] + torch.arange(t, device=DEVICE, dtype=torch.int32)
    slots = table.gather(1, (at // block).long()) * block + at % block
    return mask, positions, torch.where(live, slots, -1)


def _rotated(x, cs, pairs):
    """x [N, H, D] with its first elements rotated by the rows' (cos, sin) [N, R/2, 2], in 32 bits."""
    x = x.float()
    half = cs.shape[1]
    cos, sin = cs[:, None, :, 0], cs[:, None, :, 1]
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    if pairs == "adjacent":
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], 3).flatten(2)
    else:
        a, b = turned[..., :half], turned[..., half:]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], 2)
    return torch.cat([turned, rest], 2)


def _plain_append(state):
    cs = state["rope"][state["positions"].long()]
    slots = state["slots"].long()
    k_cache, v_cache = state["k_cache"], state["v_cache"]
    k_cache.flatten(0, 1)[slots] = _rotated(state["k"], cs, state["pairs"]).to(k_cache.dtype)
    v_cache.flatten(0, 1)[slots] = state["v"]
    return _rotated(state["q"], cs, state["pairs"]).to(k_cache.dtype), k_cache, v_cache


def _plain_tree(state):
    hq, hkv, d = state["heads"]
    q, ctx, lens, mask, longest = state["q"], state["ctx"], state["lens"], state["mask"], state["longest"]
    b, t = q.shape[:2]
    ids = state["table"].long()
    k, v = (c[ids].flatten(1, 2)[:, :longest].float().transpose(1, 2) for c in (state["k_cache"], state["v_cache"]))
    x = q.float().view(b, t, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, -1, d)     # rows (node, head)
    s = torch.matmul(x, k.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(d))
    key = torch.arange(longest, device=DEVICE)
    node = (key - ctx[:, None]).clamp(0, t - 1)                                                   # [B, keys]
    word = mask.gather(2, (node // 64)[:, None].expand(b, t, longest))
    drafted = (key >= ctx[:, None]) & (key < (ctx + lens)[:, None])
    seen = (key < ctx[:, None])[:, None] | (drafted[:, None] & ((word >> (node % 64)[:, None] & 1) == 1))
    seen &= (torch.arange(t, device=DEVICE) < lens[:, None])[:, :, None]
    s = s.view(b, hkv, t, -1, longest).masked_fill(~seen[:, None, :, None], -math.inf).view(s.shape)
    top = s.amax(3, keepdim=True)
    p = torch.exp(s - torch.where(top > -math.inf, top, 0.0))
    o = torch.matmul(p, v.contiguous()) / p.sum(3, keepdim=True).clamp_min(1e-30)
    return o.view(b, hkv, t, -1, d).permute(0, 2, 1, 3, 4).reshape(b, t, hq, d).to(q.dtype)


def _plain_verify(state):
    x, tokens, parents, lens = state["logits"], state["tokens"].long(), state["parents"].long(), state["lens"]
    m, t, n = x.shape
    node = torch.arange(t, device=DEVICE)
    up = parents.clamp_min(0)
    best = x.float().argmax(2)
    # elder siblings [B, T, T], and those that have the node's own token
    elder = (parents[:, :, None] == parents[:, None]) & (node < node[:, None])
    first = ~(elder & (tokens[:, :, None] == tokens[:, None])).any(2)
    child = (parents >= 0) & (node < lens[:, None]) & first
    fits = child & (best.gather(1, up) == tokens)
    if state["temperatures"] is not None:
        temp = state["temperatures"][:, None]
        y = x.double() / torch.where(temp > 0, temp, 1.0)[:, :, None].double()
        y = torch.exp(y - y.amax(2, keepdim=True))
        p = y / y.sum(2, keepdim=True)
        mine = torch.where(child, p.gather(1, up[:, :, None].expand(m, t, n)).gather(2, tokens[:, :, None])[:, :, 0], 0.0)
        before = (elder * mine[:, None]).sum(2)
        u = state["uniforms"].double()
        at = u.gather(1, up)
        fits = torch.where(temp > 0, child & (at >= before) & (at < before + mine), fits)
    fits[:, 0] = True
    seen = _ancestors(parents, lens) > 0
    on = (seen <= fits[:, None]).all(2) & seen[:, :, 0] & (node < lens[:, None])       # every ancestor fits
    counts = on.sum(1)
    depth = torch.where(on, seen.sum(2) - 1, t)
    path = torch.full((m, t + 1), -1, device=DEVICE).scatter(1, depth, node.expand(m, t))[:, :t]
    last = path.gather(1, (counts - 1).clamp_min(0)[:, None]).clamp_min(0)             # [B, 1]
    follow = best.gather(1, last)[:, 0]
    if state["temperatures"] is not None:
        here = child & (parents == last)
        rest = p.gather(1, last[:, :, None].expand(m, 1, n))[:, 0]
        rest = rest.scatter_reduce(1, tokens, torch.where(here, 0.0, math.inf).double(), "amin")
        total = rest.cumsum(1)
        c = (mine * here).sum(1, keepdim=True)
        target = (u.gather(1, last) - c) / (1 - c) * total[:, -1:]
        drawn = (total <= target).sum(1).clamp_max(n - 1)
        follow = torch.where(temp[:, 0] > 0, drawn, follow)
    follow = torch.where(counts > 0, follow, -1)
    return path.to(torch.int32), counts.to(torch.int32), follow.to(torch.int32)


def _plain_keep(state):
    rows, path, ctx, table = state["rows"], state["path"], state["ctx"], state["table"]
    block = rows.shape[3]
    j = torch.arange(path.shape[1], device=DEVICE)
    kept = j < state["counts"][:, None]
    at = [ctx[:, None] + torch.where(kept, x, 0) for x in (path, j)]        # node 0 stays where it is
    source, place = ((table.gather(1, (x // block).long()) * block + x % block).long().flatten() for x in at)
    flat = rows.view(2 * rows.shape[1], -1, rows.shape[4] * rows.shape[5])
    flat[:, place] = flat[:, source]
    return rows


_PLAIN = {"layout": _plain_layout, "append": _plain_append, "tree": _plain_tree, "verify": _plain_verify,
          "keep": _plain_keep}


def run(state):
    return _run_own(state) if own else _PLAIN[state["kind"]](state)


# ---- what a pass cannot do without --------------------------------------------------

def work(case):
    kind, b, t = case["kind"], case["batch"], case["nodes"]
    if kind == "layout":
        words = -(-t // 64)
        return {"bytes": b * (t * (4 + 8 * words + 8) + 8 + 4 * (t // case["block"] + 1)), "flops": b * t * 8}
    es = DTYPES[case["dtype"]].itemsize
    parents, lens = _trees(case)
    if kind == "verify":
        rows = int(_paths(case, parents, lens, 0, 6)[1].sum())              # near what another seed's are
        return {"bytes": rows * case["vocab"] * es + b * (t * 12 + 12), "flops": 4 * rows * case["vocab"]}
    hq, hkv, d = HEADS[case["heads"]]
    if kind == "append":
        n = int(lens.sum())
        return {"bytes": n * (2 * es * (hq + 2 * hkv) * d + 8 + 4 * int(d * case["share"])),
                "flops": 3 * n * (hq + hkv) * int(d * case["share"])}
    if kind == "keep":
        path, counts = _keep_paths(case)
        moved = int(((path != np.arange(t)) & (path >= 0)).sum())
        return {"bytes": moved * 4 * case["layers"] * hkv * d * es + 4 * int(counts.sum()) + 8 * b, "flops": 0}
    ctx = _contexts(case).astype(np.int64)
    # a node sees its context and, of the tree, its ancestors and itself; sequences meet their trees in any order
    pairs = int(lens.mean() * ctx.sum()) + int(_words(parents, lens)[1].sum() + lens.sum())
    keys = int((ctx.sum() + lens.sum()))
    return {"bytes": 2 * es * hkv * d * keys + int(lens.sum()) * (2 * es * hq * d + 8 * -(-t // 64)) +
            4 * keys // case["block"], "flops": 4 * hq * d * pairs}


# ---- the same in 64 bits, from the definitions ---------------------------------------

def _exact_layout(case, seed):
    parents, lens, ctx, table, _ = _batch(case, seed)
    block, (b, t) = case["block"], parents.shape
    mask = np.zeros((b, t, -(-t // 64)), np.uint64)
    positions, slots = np.zeros((b, t), np.int32), np.full((b, t), -1, np.int32)
    for i in range(b):
        for j in range(lens[i]):
            at, steps = j, -1
            while at >= 0:
                mask[i, j, at // 64] |= np.uint64(1 << (at % 64))
                at, steps = int(parents[i, at]), steps + 1
            positions[i, j] = ctx[i] + steps
            row = ctx[i] + j
            slots[i, j] = table[i, row // block] * block + row % block
    return _device(mask.view(np.int64)), _device(positions), _device(slots)


def _exact_append(case, seed):
    inp = _append_inputs(case, seed)
    cs = torch.view_as_complex(inp["rope"].double())[inp["positions"].long()][:, None]           # [N, 1, R/2]
    half = cs.shape[2]

    def turn(x):
        x = x.double().contiguous()
        z = x[..., :2 * half]
        if case["pairs"] == "adjacent":
            z = torch.view_as_real(torch.view_as_complex(z.unflatten(2, (half, 2)).contiguous()) * cs).flatten(2)
        else:
            z = torch.complex(z[..., :half], z[..., half:]) * cs
            z = torch.cat([z.real, z.imag], 2)
        return torch.cat([z, x[..., 2 * half:]], 2)

    k_cache, v_cache = inp["k_cache"].double(), inp["v_cache"].double()
    slots = inp["slots"].long()
    k_cache.view(-1, *k_cache.shape[2:])[slots] = turn(inp["k"])
    v_cache.view(-1, *v_cache.shape[2:])[slots] = inp["v"].double()
    return turn(inp["q"]), k_cache, v_cache


def _exact_tree(case, seed):
    inp = _tree_inputs(case, seed)
    parents, lens, ctx, table, _ = _batch(case, seed)
    hq, hkv, d = inp["heads"]
    out = torch.zeros(inp["q"].shape, dtype=torch.float64, device=DEVICE)
    for i in range(case["batch"]):
        n, c = int(lens[i]), int(ctx[i])
        seen = np.zeros((n, c + n), bool)
        seen[:, :c] = True
        for j in range(n):
            at = j
            while at >= 0:
                seen[j, c + at] = True
                at = parents[i, at]
        seen = _device(seen)
        ids = _device(table[i, :-(-(c + n) // case["block"])]).long()
        for h in range(hkv):
            k, v = (x[ids][:, :, h].reshape(-1, d)[:c + n].double() for x in (inp["k_cache"], inp["v_cache"]))
            for g in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                s = inp["q"][i, :n, g].double() @ k.T.contiguous() / math.sqrt(d)
                out[i, :n, g] = torch.softmax(s.masked_fill(~seen, -math.inf), 1) @ v
    return out


def _exact_verify(case, seed):
    inp = _verify_inputs(case, seed)
    m, t, n = inp["logits"].shape
    tokens, parents, lens = (inp[x].cpu().numpy() for x in ("tokens", "parents", "lens"))
    temps = np.zeros(m) if inp["temperatures"] is None else inp["temperatures"].double().cpu().numpy()
    u = np.zeros((m, t)) if inp["uniforms"] is None else inp["uniforms"].double().cpu().numpy()
    path, counts, follow = np.full((m, t), -1, np.int32), np.zeros(m, np.int32), np.full(m, -1, np.int32)
    for i in range(m):
        at = 0
        while True:
            path[i, counts[i]] = at
            counts[i] += 1
            x = inp["logits"][i, at].double().cpu().numpy()
            children = [j for j in range(lens[i]) if j > at and parents[i, j] == at]
            if temps[i] <= 0:
                follow[i] = int(np.argmax(x))
                nxt = [j for j in children if tokens[i, j] == follow[i]][:1]
            else:
                p = np.exp((x - x.max()) / temps[i])
                p /= p.sum()
                c, nxt, met = 0.0, [], set()
                for j in children:
                    if tokens[i, j] in met:
                        continue
                    met.add(tokens[i, j])
                    c += p[tokens[i, j]]
                    if u[i, at] < c:
                        nxt = [j]
                        break
                if not nxt:
                    p[list(met)] = 0.0
                    total = np.cumsum(p)
                    follow[i] = min(n - 1, int(np.sum(total <= (u[i, at] - c) / (1 - c) * total[-1])))
            if not nxt:
                break
            at = nxt[0]
    return _device(path), _device(counts), _device(follow)


def _exact_keep(case, seed):
    inp = _keep_inputs(case, seed)
    block = case["block"]
    path, counts, ctx, table = (inp[x].cpu().numpy() for x in ("path", "counts", "ctx", "table"))
    old = inp["rows"].flatten(2, 3)
    new = old.clone()
    for i in range(case["batch"]):
        for j in range(counts[i]):
            a, b = (int(table[i, r // block]) * block + r % block for r in (int(ctx[i] + path[i, j]), int(ctx[i] + j)))
            new[:, :, b] = old[:, :, a]
    return new.view(inp["rows"].shape)


def exact(case, seed):
    return {"layout": _exact_layout, "append": _exact_append, "tree": _exact_tree, "verify": _exact_verify,
            "keep": _exact_keep}[case["kind"]](case, seed)
