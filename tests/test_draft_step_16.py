"""Verified steps in 16 bits: the verdict is the definition's over the step's own logits, and the cache that it leaves is that of a
prompt with the accepted tokens."""

import numpy as np
import pytest
import torch

from oracle.draft_tree import verify_ref
from tests.test_draft_step import Sequences, build, drafted, verified_step
from tests.test_draft_tree import gpu, rng_of


def rows(seqs, b, n):
    """K and V of the sequence's first n positions, in all layers: [2, layers, n, heads, dim] float32."""
    table = torch.as_tensor(np.asarray(seqs.tables()[0]))[b].long().cuda()
    at = torch.arange(n, device="cuda")
    blocks, offsets = table[at // seqs.bs], at % seqs.bs
    return torch.stack([torch.stack([c[blocks, offsets].float() for c in side])
                        for side in (seqs.cache.k_cache, seqs.cache.v_cache)])


@gpu
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_verified_steps_of_16_bits(dtype):
    model = build(dtype)
    rng = rng_of(5)
    prompts = [rng.integers(0, 512, n) for n in (5, 16, 37)]
    guess, tree = Sequences(model, prompts), Sequences(model, prompts)
    greedy = [list(guess.next)]
    for _ in range(24):
        guess.step()
        greedy.append(list(guess.next))
    text = [list(p) for p in prompts]                            # what each sequence has cached
    longest = 0
    for right in (3, 0, 5):
        done = [len(t) - len(p) for t, p in zip(text, prompts)]
        trees = [drafted(rng, tree.next[b], [g[b] for g in greedy[done[b] + 1:]], 14, right) for b in range(3)]
        tokens, parents = np.stack([x[0] for x in trees]), np.stack([x[1] for x in trees])
        logits, verdict = verified_step(tree, tokens, parents, np.full(3, 14, np.int32))
        path, counts, follow, _ = verify_ref(logits.double().cpu().numpy(), tokens, parents, [14] * 3)
        for got, want in zip(verdict, (path, counts, follow)):
            assert np.array_equal(got.cpu().numpy(), want)
        longest = max(longest, int(counts.max()))
        for b in range(3):
            text[b] += [int(tokens[b, n]) for n in path[b, :counts[b]]]
            assert tree.manager.get_context_length(b) == len(text[b])
        tree.next = follow.tolist()
        # the same tokens as one prompt: its cache and its next step.  2e-2 of their scale is what a 16-bit step is held to
        fresh = Sequences(model, text)
        for b in range(3):
            a, x = rows(tree, b, len(text[b])), rows(fresh, b, len(text[b]))
            for i in range(2):                                   # K, V
                scale = float(x[i].abs().max())
                assert float((a[i] - x[i]).abs().max()) < 2e-2 * scale
                # rows of other positions are further away than that: one in a wrong place would be seen
                other = x[i].roll(1, 1)
                assert float((other - x[i]).abs().amax((0, 2, 3)).min()) > 1e-1 * scale
        fresh.next = list(tree.next)
        want = fresh.step()
        text = [t + [n] for t, n in zip(text, tree.next)]        # a single-token step in between, which caches them
        got = tree.step()
        assert float((got - want).abs().max()) < 2e-2 * float(want.abs().max())
    assert longest > 3
