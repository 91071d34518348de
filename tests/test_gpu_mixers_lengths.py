"""Lengths of attention at the ends of their 32 bits: a length that no sequence can
have, and as many tokens as a page table can name."""
import numpy as np
import pytest
import torch

import mixer_fixtures as F
import rl_mixers as M
from test_gpu_mixers import attend_check, randn

pytestmark = pytest.mark.gpu

MOST = 2 ** 31 - 1


@pytest.mark.parametrize("page", [2 ** 16, 2 ** 16 - 3])
def test_the_last_tokens_of_the_longest_sequences(device, page):
    # One page that every entry of the tables names: token t is in slot t % page. Lengths below zero are none.
    g = np.random.default_rng(40)
    lens, counts, window, dim = [MOST, MOST, -2 ** 31, 70, MOST - 31, -5], [3, 1, 3, 2, 40, 1], 50, 16
    cache = M.DeviceCache(1, page, 1, dim, "bf16")
    k, v = (randn(g, (page, 1, dim), "bf16", device) for _ in range(2))
    cache.write(k, v, torch.arange(page, device=device))
    q = randn(g, (sum(counts), 2, dim), "bf16", device)
    out, lse = torch.full_like(q, 7.0), torch.full((len(q), 2), 7.0, device=device)
    table = torch.zeros(len(lens), -(-MOST // page), dtype=torch.int32, device=device)
    starts = torch.from_numpy(np.cumsum([0] + counts).astype(np.int32)).to(device)
    att = M.DeviceAttention(len(q), 2, 1, dim, MOST)
    att.rows(cache, q, out, torch.tensor(lens, dtype=torch.int32, device=device), table, starts=starts, lse=lse,
             window=window, most_rows=max(counts))
    torch.cuda.synchronize()
    seen = [max(min(n, window + c - 1), 0) for n, c in zip(lens, counts)]
    slots = [np.arange(n - m, n) % page if m else np.arange(0) for n, m in zip(lens, seen)]
    stored = [(F.as64(k)[s], F.as64(v)[s]) for s in slots]
    attend_check(q, out, lse, seen, counts, stored, "bf16", "bf16", window, dim)


def test_every_token_of_the_longest_sequence(device):
    # Equal scores and values of 1: the result is 1, the lse the logarithm of the length, and sums of ones are exact in f32.
    page, dim = 2 ** 16, 16
    cache = M.DeviceCache(1, page, 1, dim, "bf16")
    ones = torch.ones(page, 1, dim, device=device)
    cache.write(torch.zeros_like(ones), ones, torch.arange(page, device=device))
    q = torch.ones(2, 1, dim, device=device)
    out, lse = torch.empty_like(q), torch.empty(2, 1, device=device)
    att = M.DeviceAttention(2, 1, 1, dim, MOST)
    att.rows(cache, q, out, torch.tensor([MOST], dtype=torch.int32, device=device),
             torch.zeros(1, 2 ** 15, dtype=torch.int32, device=device),
             starts=torch.tensor([0, 2], dtype=torch.int32, device=device), lse=lse)
    torch.cuda.synchronize()
    assert np.abs(F.as64(out) - 1).max() <= 2.0 ** -22
    assert np.abs(F.as64(lse) - np.log(float(MOST))).max() <= 2.0 ** -18
