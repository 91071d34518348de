"""Batches of thousands of sequences, most of them of one token or none: their grids
have to fit a launch."""
import numpy as np
import pytest
import torch

import mixer_fixtures as F
import rl_mixers as M
from test_gpu_mixers import delta_check, delta_inputs, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("at", [0, 5000, 8191])
def test_a_prompt_among_thousands_of_single_tokens(device, at):
    # 4096 rows of 8 heads are 2048 blocks of 16: for each of 8192 sequences they would pass what one launch takes.
    g = np.random.default_rng(70)
    seqs, prompt, heads, dim, window, page = 8192, 4096, 8, 256, 5, 16
    counts = np.ones(seqs, int)
    counts[at] = prompt
    counts[[3, 4, 6000]] = 0
    lens = g.integers(1, 4 * page + 1, seqs)
    lens[at] = prompt
    cache = M.DeviceCache(prompt // page, page, 1, dim, "bf16")
    k, v = (randn(g, (prompt, 1, dim), "bf16", device) for _ in range(2))
    cache.write(k, v, torch.arange(prompt, device=device))
    table = g.integers(0, prompt // page, (seqs, prompt // page))  # sequences share pages
    rows = int(counts.sum())
    q = randn(g, (rows, heads, dim), "bf16", device)
    out, lse = torch.full_like(q, 7.0), torch.full((rows, heads), 7.0, device=device)
    i32 = lambda x: torch.from_numpy(np.ascontiguousarray(x, np.int32)).to(device)  # noqa: E731
    att = M.DeviceAttention(rows, heads, 1, dim, prompt)
    att.rows(cache, q, out, i32(lens), i32(table), starts=i32(np.cumsum(np.r_[0, counts])), lse=lse, window=window,
             most_rows=prompt)
    torch.cuda.synchronize()
    # Every row's last `window` tokens, all at once.
    of = np.repeat(np.arange(seqs), counts)
    place = lens[of] - counts[of] + np.arange(rows) - np.r_[0, np.cumsum(counts)][of]
    tokens = place[:, None] - np.arange(window)  # [rows][window], the row's own first
    seen = tokens >= 0
    slots = table[of[:, None], np.maximum(tokens, 0) // page] * page + np.maximum(tokens, 0) % page
    keys, values, x = F.as64(k)[:, 0], F.as64(v)[:, 0], F.as64(q)
    scores = np.einsum("rhd,rwd->rhw", x, keys[slots]) * dim ** -0.5
    size = np.einsum("rhd,rwd->rhw", np.abs(x), np.abs(keys[slots])) * dim ** -0.5
    scores[~np.broadcast_to(seen[:, None], scores.shape)] = -np.inf
    top = scores.max(-1)
    p = np.exp(scores - top[..., None])
    want_lse = top + np.log(p.sum(-1))
    p /= p.sum(-1, keepdims=True)
    want, mass = np.einsum("rhw,rwd->rhd", p, values[slots]), np.einsum("rhw,rwd->rhd", p, np.abs(values[slots]))
    d = size.max(-1) * (dim + 8) * 2.0 ** -24
    slack = mass * (2 * d + 2.0 ** -15)[..., None]  # the weights' 16 bits, their scores' errors and a few sums
    assert (np.abs(F.as64(out) - want) / (slack + F.rounding(np.abs(want) + slack, "bf16"))).max() <= 1
    assert (np.abs(F.as64(lse) - want_lse) / (d + 2.0 ** -20 + np.abs(want_lse) * 2.0 ** -23)).max() <= 1


def test_more_states_than_a_launch_of_chunks_takes(device):
    # 8192 sequences of 64 heads of 256 columns are 2^23 workgroups of 512 threads; one sequence has rows.
    g = np.random.default_rng(71)
    seqs, n, kh, vh, dk, dv, at = 8192, 24, 1, 64, 16, 256, 5003
    h = M.DeviceDelta(2 ** 17, seqs, kh, vh, dk, dv)
    inputs = delta_inputs(g, device, [n], kh, vh, dk, dv, "bf16", True, 0.2)
    q, k, v, gates, beta, states = inputs
    before, out = F.as64(states), torch.empty_like(v)
    slots = np.full((2, seqs), -1)
    slots[:, at] = 0, 1
    starts = np.where(np.arange(seqs + 1) > at, n, 0)
    i32 = lambda x: torch.from_numpy(np.ascontiguousarray(x, np.int32)).to(device)  # noqa: E731
    h.rows(q, k, v, gates, beta, out, states, i32(slots[0]), i32(slots[1]), i32(starts), normalise=True, most_rows=n)
    torch.cuda.synchronize()
    delta_check([n], inputs, F.as64(out), before[:1], F.as64(states)[1:2], dk, "bf16", True, dk ** -0.5, n)
    h.close()
