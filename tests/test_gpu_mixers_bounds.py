"""What include/rl_mixers.h promises of the token mixers' exactness, held to bounds
that a loss of bits would break. Bounds are formed before the comparison; where an
output has 16 bits, its error's mean square is compared with that of rounding the
float64 value to the same type, which no other error may add much to."""
import numpy as np
import pytest
import torch

import mixer_fixtures as F
import rl_mixers as M
from test_gpu_mixers import delta_inputs, randn

pytestmark = pytest.mark.gpu


def i32(x, device):
    return torch.from_numpy(np.ascontiguousarray(x, np.int32)).to(device)


def rms(x):
    return np.sqrt((np.asarray(x) ** 2).mean())


def rounded(x, dtype):
    return F.as64(torch.from_numpy(np.ascontiguousarray(x)).to(F.TYPES[dtype]))


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


# --------------------------------------------------------------- delta --
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("form", ["steps", "chunks"])
def test_delta_outputs_are_as_good_as_their_rounding(device, dtype, form):
    # Operands of 16 bits or more are off by 2^-16 of a term, a few times that of the output; the output's rounding by
    # 2^-9 (bf16) or 2^-12 (f16) and more in the mean: a hundredth may be added. An operand of 8 bits adds a quarter.
    g = np.random.default_rng(32)
    n, kh, vh, dk, dv = 700, 2, 4, 128, 64
    inputs = delta_inputs(g, device, [n], kh, vh, dk, dv, dtype, True, 0.2)
    q, k, v, gates, beta, states = inputs
    before, out = F.as64(states), torch.empty_like(v)
    h = M.DeviceDelta(n, 1, kh, vh, dk, dv)
    h.rows(q, k, v, gates, beta, out, states, i32([0], device), i32([1], device), i32([0, n], device), normalise=True,
           most_rows=1 if form == "steps" else n)
    torch.cuda.synchronize()
    want, _ = F.delta(*(F.as64(x) for x in inputs[:5]), before[0], dk ** -0.5, 1e-6)
    ratio = rms(F.as64(out) - want) / rms(rounded(want, dtype) - want)
    print("delta outputs", dtype, form, "error over the rounding's", ratio, flush=True)
    assert ratio <= 1.01
