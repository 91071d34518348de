"""Attention behind shared prefixes with scales that leave nothing of the scores: 0,
which weighs all tokens alike whatever the scores are, and NaN."""
import numpy as np
import pytest
import torch

import mixer_fixtures as F
import rl_mixers as M
from test_gpu_mixers import randn
from test_gpu_shared import Case, i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seqs", [3, 120])  # few and many rows of a prefix
@pytest.mark.parametrize("fmt,dtype,size", [("bf16", "bf16", 1e18), ("bf16", "f32", 1e18), ("i8", "bf16", 1e33), ("i8", "f32", 1e33)])
def test_a_scale_of_zero_weighs_all_tokens_alike(device, seqs, fmt, dtype, size):
    g = np.random.default_rng(31)
    prefix, own, dim, page = 90, 3, 32, 16
    pages = -(-prefix // page)
    cache = M.DeviceCache(pages + seqs, page, 1, dim, fmt)
    tokens = (pages + seqs) * page
    # Scores of up to 1e38 before the scale: q k is finite in f32.
    k = torch.from_numpy((g.uniform(-1, 1, (tokens, 1, dim)) * size).astype(np.float32)).to(device).to(torch.bfloat16)
    v = randn(g, (tokens, 1, dim), "bf16", device)
    cache.write(k, v, torch.arange(tokens, device=device))
    q = torch.from_numpy((g.uniform(-1, 1, (seqs, 1, dim)) * 1e36 / size).astype(np.float32)).to(device).to(F.TYPES[dtype])
    out, lse = torch.empty_like(q), torch.empty(seqs, 1, device=device)
    att = M.DeviceAttention(seqs, 1, 1, dim, prefix)
    own_pages = i32(np.arange(seqs)[:, None] + pages, device)
    args = (cache, q, out, i32([own] * seqs, device), own_pages, i32([0, seqs], device), i32([prefix], device),
            i32(np.arange(pages)[None], device))
    held = F.encode(F.as64(v), fmt)
    n = prefix + own
    want = np.stack([np.concatenate([held[:prefix], held[(pages + s) * page:(pages + s) * page + own]]).mean(0) for s in range(seqs)])
    most = np.abs(held).max()
    for scale in (0.0, -0.0):
        att.shared(*args, lse=lse, scale=scale)
        torch.cuda.synchronize()
        # Every weight is 1 within 2^-20, and rounded to two parts of 16 bits or more; sums of n tokens.
        slack = most * (2.0 ** -19 + 2.0 ** -15 + n * 2.0 ** -24)
        assert np.all(np.abs(F.as64(out) - want) <= slack + F.rounding(np.abs(want) + slack, dtype))
        assert np.all(np.abs(F.as64(lse) - np.log(n)) <= 2.0 ** -18)
    att.shared(*args, lse=lse, scale=float("nan"))
    torch.cuda.synchronize()
    assert torch.isnan(out).all() and torch.isnan(lse).all()


def test_a_scale_of_nan_where_rows_see_the_prefix_alone(device):
    g = np.random.default_rng(32)
    c = Case(g, device, [70], [120], [0] * 120, [1] * 120, 1, 1, 32, 16, "bf16", "bf16")
    c.call()
    assert torch.isfinite(c.out).all()
    c.call(scale=float("nan"))
    assert torch.isnan(c.out).all() and torch.isnan(c.lse).all()
