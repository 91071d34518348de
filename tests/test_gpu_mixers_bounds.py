"""What include/rl_mixers.h promises of the token mixers' exactness, held to bounds
that a loss of bits would break. Bounds are formed before the comparison; where an
output has 16 bits, its error's mean square is compared with that of rounding the
float64 value to the same type, which no other error may add much to."""
import numpy as np
import pytest
import torch

import mixer_fixtures as F
import rl_mixers as M
from test_gpu_mixers import attend_case, attend_check, delta_check, delta_inputs, randn

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


WEIGHTS = [
    # lens, rows of each, q heads, kv heads, dim, page, format, type
    ([1500, 700, 64], [1, 1, 1], 16, 2, 128, 32, "bf16", "bf16"),
    ([1500, 700, 64], [1, 1, 1], 16, 2, 128, 32, "i8", "bf16"),
    ([900], [5], 16, 2, 64, 24, "f8", "bf16"),
    ([1500, 700, 64], [1, 1, 1], 16, 2, 128, 32, "f16", "f16"),
    ([900], [5], 16, 2, 256, 16, "i8", "f16"),
    ([900], [5], 16, 2, 64, 16, "f8", "f16"),
]


@pytest.mark.parametrize("case", range(len(WEIGHTS)))
def test_weights_of_16_bit_queries(device, case):
    # Weights of 16 bits are off by 2^-17 of themselves, the output's rounding by 2^-9 (bf16) or 2^-12 (f16) and more in the
    # mean: the mean square may grow by a thousandth; weights of 8 bits double it.
    lens, counts, qh, kv, dim, page, fmt, dtype = WEIGHTS[case]
    g = np.random.default_rng(900 + case)
    cache, att, q, out, lse, starts, stored, call, _ = attend_case(g, device, *WEIGHTS[case], 0, spread=0.5)
    call(most_rows=max(counts))
    torch.cuda.synchronize()
    at, off, own = 0, [], []
    for n, c, (k, v) in zip(lens, counts, stored):
        want = F.attention(F.as64(q[at:at + c]), k, v, dim ** -0.5, n)[0]
        off.append((F.as64(out[at:at + c]) - want).ravel())
        own.append((rounded(want, dtype) - want).ravel())
        at += c
    ratio = rms(np.concatenate(off)) / rms(np.concatenate(own))
    print("weights", WEIGHTS[case], "error over the rounding's", ratio, flush=True)
    assert ratio <= 1.01


@pytest.mark.parametrize("fmt", ["bf16", "f16", "i8", "f8"])
def test_weights_of_f32_queries(device, fmt):
    # Scores below a tenth are good to 2^-24 and better, weights to 22 bits, the exponential and the sums over 1500 tokens
    # to 2^-21 in the mean: 2^-20 in all. Weights of 16 bits would be 2^-18 off in the mean.
    case = ([1500, 700, 64], [1, 1, 1], 16, 2, 128, 32, fmt, "f32", 0)
    g = np.random.default_rng(31)
    cache, att, q, out, lse, starts, stored, call, _ = attend_case(g, device, *case, spread=0.02)
    call(most_rows=1)
    torch.cuda.synchronize()
    for s, n in enumerate(case[0]):
        want, want_lse, _, _ = F.attention(F.as64(q[s:s + 1]), *stored[s], 128 ** -0.5, n)
        off = rms(F.as64(out[s:s + 1]) - want) / rms(want)
        print("f32 weights", fmt, n, off, flush=True)
        assert off <= 2.0 ** -20
        assert np.abs(F.as64(lse[s:s + 1]) - want_lse).max() <= 2.0 ** -20 + np.abs(want_lse).max() * 2.0 ** -23


MANY = [
    # lens, rows of each, q heads, kv heads, dim, page, format, type, window
    ([400], [400], 4, 2, 128, 32, "bf16", "bf16", 0),
    ([700, 260], [300, 260], 4, 1, 64, 24, "i8", "bf16", 0),
    ([513], [257], 2, 1, 256, 16, "f8", "f16", 100),
    ([300, 130], [300, 111], 2, 2, 80, 40, "f16", "f32", 37),
    # A prompt beside single tokens, sequences without rows among them.
    ([380] + [50 + 7 * i for i in range(63)], [380] + [1] * 63, 4, 2, 128, 16, "i8", "bf16", 0),
    ([90, 200, 0, 31, 600, 5], [1, 200, 0, 1, 300, 5], 8, 1, 256, 20, "bf16", "bf16", 0),
]


@pytest.mark.parametrize("case", range(len(MANY)))
def test_attention_of_prompts_and_mixed_batches(device, case):
    lens, counts, qh, kv, dim, page, fmt, dtype, window = MANY[case]
    g = np.random.default_rng(950 + case)
    cache, att, q, out, lse, starts, stored, call, _ = attend_case(g, device, *MANY[case], fill=float("nan"))
    print("attend", MANY[case][2:], flush=True)
    for kw in (dict(most_rows=max(counts)), {}):
        out.fill_(7.0)
        call(**kw)
        torch.cuda.synchronize()
        attend_check(q, out, lse, lens, counts, stored, fmt, dtype, window, dim)


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


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("form", ["steps", "chunks"])
def test_delta_states_are_as_good_as_f32(device, dtype, form):
    # A chunk's sums of dk + 64 terms in f32 are off by 2^-24 sqrt(dk + 64) of the state in the mean, and the state forgets
    # in a few chunks: 2^-19. Operands of 16 bits would leave 2^-18 and more.
    g = np.random.default_rng(33)
    n, kh, vh, dk, dv = 700, 1, 2, 128, 64
    inputs = delta_inputs(g, device, [n], kh, vh, dk, dv, dtype, True, 0.02)
    q, k, v, gates, beta, states = inputs
    before, out = F.as64(states), torch.empty_like(v)
    h = M.DeviceDelta(n, 1, kh, vh, dk, dv)
    h.rows(q, k, v, gates, beta, out, states, i32([0], device), i32([1], device), i32([0, n], device), normalise=True,
           most_rows=1 if form == "steps" else n)
    torch.cuda.synchronize()
    want_out, want = F.delta(*(F.as64(x) for x in inputs[:5]), before[0], dk ** -0.5, 1e-6)
    off = rms(F.as64(states)[1] - want) / rms(want)
    print("delta state", dtype, form, off, flush=True)
    assert off <= 2.0 ** -19
    if dtype == "f32":
        off = rms(F.as64(out) - want_out) / rms(want_out)
        print("delta f32 outputs", form, off, flush=True)
        assert off <= 2.0 ** -19


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_delta_of_a_prompt_beside_single_tokens(device, dtype):
    g = np.random.default_rng(34)
    lens, kh, vh, dk, dv = [1] * 20 + [300] + [1] * 30 + [0, 0, 9] + [1] * 10, 1, 2, 64, 48
    inputs = delta_inputs(g, device, lens, kh, vh, dk, dv, dtype, True, 0.2)
    q, k, v, gates, beta, states = inputs
    n, rows = len(lens), sum(lens)
    before, out = F.as64(states), torch.empty_like(v)
    h = M.DeviceDelta(rows, n, kh, vh, dk, dv)
    slots = torch.arange(2 * n, dtype=torch.int32, device=device)
    h.rows(q, k, v, gates, beta, out, states, slots[:n], slots[n:], i32([0] + list(np.cumsum(lens)), device), normalise=True,
           most_rows=300)
    torch.cuda.synchronize()
    delta_check(lens, inputs, F.as64(out), before[:n], F.as64(states)[n:2 * n], dk, dtype, True, dk ** -0.5, 300)
