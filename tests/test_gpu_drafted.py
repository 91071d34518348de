"""examples/drafted_batch.py: the convolution, the scan, attention behind a shared
prompt, the sampler and the verification together. A sequence behind a shared prompt has
the same hidden rows as one that holds the prompt itself, whether its own tokens come in
one call or one by one, and the example repeats."""
import os
import sys

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "examples"))


@pytest.mark.parametrize("cache", ["bf16", "f8"])
@pytest.mark.parametrize("prompt", [96, 333])
def test_behind_a_shared_prompt_and_with_it(device, cache, prompt):
    import drafted_batch as X
    g = np.random.default_rng(prompt)
    counts = [9, 1, 30]
    said = g.integers(0, 4096, prompt).astype(np.int32)
    own = [g.integers(0, 4096, n).astype(np.int32) for n in counts]
    dev = lambda t: torch.from_numpy(t).to(device)  # noqa: E731

    def model(seqs, length):
        return X.DraftedModel(seqs, length, 32, 12, cache=cache, seed=5)

    whole = []
    for tokens in own:
        hidden = model(1, prompt + len(tokens)).read_prompt(dev(np.concatenate([said, tokens])))
        whole.append(hidden[prompt:].cpu().double().numpy())

    def behind(parts):
        m = model(3, prompt)
        m.read_prompt(dev(said))
        at, rows = [0, 0, 0], [[], [], []]
        for part in parts:
            chunk = np.concatenate([t[a:a + c] for t, a, c in zip(own, at, part)])
            hidden, _ = m.run(dev(chunk), part, m.own, m.own)
            for s, y in enumerate(hidden.split(part)):
                rows[s].append(y.cpu().double().numpy())
            at = [a + c for a, c in zip(at, part)]
            m.lens = at
        return [np.concatenate(r) for r in rows]

    # Every mixer is good to f32 in either form, but a key or value near the middle of two codes may be stored one code
    # apart: 2^-8 or 2^-4 of itself, in one of the 64 values of some heads of some tokens.
    near = {"bf16": 2.0 ** -8, "f8": 2.0 ** -4}[cache] / 8 + 2.0 ** -13
    for got in (behind([counts]), behind([[4, 1, 10], [5, 0, 20]]), behind([[1, 1, 1]] + [[1, 0, 1]] * 8 + [[0, 0, 21]])):
        for a, b in zip(got, whole):
            assert a.shape == b.shape and np.sqrt(((a - b) ** 2).mean()) <= near * np.sqrt((b ** 2).mean())


def test_the_example_repeats(device):
    import drafted_batch as X
    (a, n), (b, m) = (X.decode(seqs=3, prompt=70, steps=5, drafts=4, seed=2) for _ in range(2))
    assert a == b and n == m and 0 <= n <= 60
    assert sum(len(row) for row in a) == 3 + 15 + n and all(0 <= t < 4096 for row in a for t in row)
    assert a != X.decode(seqs=3, prompt=70, steps=5, drafts=4, seed=3)[0]
