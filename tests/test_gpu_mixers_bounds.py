"""What include/rl_mixers.h promises of the token mixers' exactness, held to bounds
that a loss of bits would break. Bounds are formed before the comparison."""
import numpy as np
import pytest
import torch

import mixer_fixtures as F
import rl_mixers as M
from test_gpu_mixers import randn

pytestmark = pytest.mark.gpu


def i32(x, device):
    return torch.from_numpy(np.ascontiguousarray(x, np.int32)).to(device)


# ----------------------------------------------------------- attention --
@pytest.mark.parametrize("offset", [0.0, 2.0, 8.0])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 24), (256, 32)])
def test_scores_of_queries_with_a_common_offset(device, dim, page, dtype, offset):
    # One token a sequence: the lse is its score. Keys have a few channels far larger than the rest, so most int8 codes
    # are small beside what a constant added to every code would be.
    g = np.random.default_rng(30)
    seqs, heads, kv = 96, 8, 2
    cache = M.DeviceCache(seqs, page, kv, dim, "i8")
    k = g.standard_normal((seqs, kv, dim)) * (1 + 7 * (g.random((kv, dim)) < 0.03))
    k = torch.from_numpy(k.astype(np.float32)).to(device)
    q = randn(g, (seqs, heads, dim), "f32", device) + offset
    q = q.to(F.TYPES[dtype])
    cache.write(k, k, torch.arange(seqs, device=device) * page)
    out, lse = torch.empty_like(q), torch.empty(seqs, heads, device=device)
    att = M.DeviceAttention(seqs, heads, kv, dim, page)
    att.rows(cache, q, out, i32([1] * seqs, device), i32(np.arange(seqs)[:, None], device), lse=lse)
    torch.cuda.synchronize()
    keys, x = np.repeat(F.encode(F.as64(k), "i8"), heads // kv, 1), F.as64(q)
    want, size = (keys * x).sum(-1) * dim ** -0.5, (np.abs(keys * x)).sum(-1) * dim ** -0.5
    # dim products and sums in f32 with the scale and the step (f32 queries: 22 bits in two parts), then to base 2 and
    # back, and a logarithm of 1.
    slack = size * ((dim + 8) * 2.0 ** -24 + (2.0 ** -22 if dtype == "f32" else 0)) + np.abs(want) * 2.0 ** -22 + 2.0 ** -22
    off = np.abs(F.as64(lse) - want)
    print("scores", dim, dtype, offset, "off at most", off.max(), "of the bound", (off / slack).max(), flush=True)
    assert (off / slack).max() <= 1
