"""examples/hybrid_decode.py: the mixers together, between the lookup and the
head. A prompt gives its last tokens the same hidden rows whether it comes in one
call (chunks, many query rows) or its tail token by token (steps, one row), and the
example's draws repeat."""
import os
import sys

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "examples"))


@pytest.mark.parametrize("cache", ["bf16", "f16", "f8"])
def test_prompts_at_once_and_token_by_token(device, cache):
    import hybrid_decode as H
    g = np.random.default_rng(3)
    counts = [70, 1, 33]
    tokens = [g.integers(0, 4096, n + 5).astype(np.int32) for n in counts]

    def rows(parts):
        m = H.HybridModel(3, 128, 256, cache=cache)
        at, last = [0, 0, 0], None
        for part in parts:
            chunk = np.concatenate([t[a:a + c] for t, a, c in zip(tokens, at, part)])
            y = m.hidden_rows(torch.from_numpy(chunk).to(device), part)
            at = [a + c for a, c in zip(at, part)]
            last = y[torch.tensor(np.cumsum(part) - 1, device=device)]
        torch.cuda.synchronize()
        return last.cpu().double().numpy()

    whole = rows([[n + 5 for n in counts]])
    tail = rows([counts] + [[1, 1, 1]] * 5)
    uneven = rows([[60, 1, 20], [15, 5, 18]])
    # Every mixer is good to f32 in either form, but a key or value near the middle of two codes may be stored one
    # code apart: 2^-8, 2^-11 or 2^-4 of itself, in one of the 64 values of some heads of some tokens.
    size = np.sqrt((whole ** 2).mean())
    near = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f8": 2.0 ** -4}[cache] / 8 + 2.0 ** -13
    assert np.sqrt(((tail - whole) ** 2).mean()) <= near * size
    assert np.sqrt(((uneven - whole) ** 2).mean()) <= near * size


def test_the_example_repeats(device):
    import hybrid_decode as H
    a, b = (H.decode(seqs=3, prompt=25, steps=6, seed=5) for _ in range(2))
    assert a.shape == (3, 6) and np.array_equal(a, b) and (a >= 0).all() and (a < 4096).all()
    assert not np.array_equal(a, H.decode(seqs=3, prompt=25, steps=6, seed=6))
