"""Log-probabilities of rows at every alignment, and on a stream of the caller's."""

import numpy as np
import pytest
import torch

from tests.test_logprobs import DTYPES, check, gpu


@gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("vocab,stride", [(517, 1031), (1003, 1003), (4099, 4104), (33001, 33007)])
def test_rows_at_every_offset(dtype, vocab, stride):
    """Views whose rows start anywhere in a 16-byte word, each row elsewhere than the last where the stride is odd."""
    from tinyvllm_amd.sampling import token_logprobs
    rng = np.random.Generator(np.random.PCG64(66))
    rows = 3
    wide = torch.from_numpy((rng.standard_normal(rows * stride + 8) * 2).astype(np.float32)).to("cuda", DTYPES[dtype])
    tokens = rng.integers(0, vocab, rows)
    for offset in range(8):
        view = torch.as_strided(wide, (rows, vocab), (stride, 1), offset)
        out = token_logprobs(view, torch.from_numpy(tokens.astype(np.int32)).cuda(), 6)
        check(out, view.double().cpu().numpy(), tokens, 6)


@gpu
def test_neighbours_of_a_view_are_not_read_into_it():
    """What lies around the rows, NaN and larger logits, shows nowhere."""
    from tinyvllm_amd.sampling import token_logprobs
    rng = np.random.Generator(np.random.PCG64(67))
    for dtype in DTYPES.values():
        for vocab, offset in ((1003, 5), (1000, 8), (70001, 3)):
            wide = torch.full((3, vocab + 16), float("nan"), device="cuda", dtype=dtype)
            wide[:, ::2] = 100.0
            x = torch.from_numpy((rng.standard_normal((3, vocab)) * 2).astype(np.float32)).to("cuda", dtype)
            wide[:, offset:offset + vocab] = x
            tokens = rng.integers(0, vocab, 3)
            out = token_logprobs(wide[:, offset:offset + vocab], torch.from_numpy(tokens.astype(np.int32)).cuda(), 9)
            check(out, x.double().cpu().numpy(), tokens, 9)


@gpu
def test_on_another_stream():
    from tinyvllm_amd.sampling import token_logprobs
    rng = np.random.Generator(np.random.PCG64(68))
    x = torch.from_numpy((rng.standard_normal((5, 70000)) * 2).astype(np.float32)).cuda()
    tokens = torch.arange(5, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x += 1.0
        out = token_logprobs(x, tokens, 4)
    side.synchronize()
    check(out, x.double().cpu().numpy(), tokens.cpu().numpy(), 4)
