"""The token mixers at their limits: caches past 4 GiB, lengths that split into the
most parts, every head size's widest form, graphs, and batches of many sequences.
Bounds as in test_gpu_mixers.py."""
import numpy as np
import pytest
import torch

import mixer_fixtures as F
import rl_mixers as M
from test_gpu_mixers import attend_case, attend_check, delta_check, delta_inputs, randn

pytestmark = pytest.mark.gpu

ATTEND = [
    # lens, rows of each, q heads, kv heads, dim, page, format, type, window
    ([30000], [1], 1, 1, 16, 48, "bf16", "bf16", 0),          # as many parts as there are
    ([9000, 1], [9, 1], 16, 2, 256, 32, "i8", "bf16", 0),     # two row tiles of 256 columns
    ([2500], [7], 24, 4, 256, 64, "f8", "f32", 0),
    ([1800, 1700], [5, 6], 16, 2, 256, 30, "bf16", "f32", 0),
    ([4000, 70], [33, 2], 8, 1, 128, 128, "bf16", "bf16", 0),  # several row blocks a sequence
    ([1000, 999], [20, 17], 4, 2, 64, 33, "i8", "f32", 64),
    ([257] * 70, [1] * 70, 8, 8, 32, 16, "f8", "bf16", 0),
    ([1] * 40 + [3000], [1] * 41, 4, 1, 96, 16, "f16", "f16", 0),
]


@pytest.mark.parametrize("case", range(len(ATTEND)))
def test_attention_forms(device, case):
    lens, counts, qh, kv, dim, page, fmt, dtype, window = ATTEND[case]
    g = np.random.default_rng(700 + case)
    cache, att, q, out, lse, starts, stored, call, _ = attend_case(g, device, *ATTEND[case], fill=float("inf"))
    print("attend", ATTEND[case][2:], flush=True)
    call(most_rows=max(counts))
    torch.cuda.synchronize()
    attend_check(q, out, lse, lens, counts, stored, fmt, dtype, window, dim)


@pytest.mark.parametrize("fmt", ["bf16", "i8"])
def test_a_cache_past_four_gib(device, fmt):
    # 8 heads of 256: 2^32 bytes of keys are 2^20 (bf16) or 2^21 (int8) tokens; the last pages lie past that.
    page, heads, dim = 64, 8, 256
    pages = (2 ** 32 // (heads * dim * (2 if fmt == "bf16" else 1))) // page + 40
    g = np.random.default_rng(20)
    cache = M.DeviceCache(pages, page, heads, dim, fmt)
    assert cache.bytes() > 2 ** 33
    n = 300
    k, v = (randn(g, (n, heads, dim), "bf16", device) for _ in range(2))
    table = np.array([[pages - 1 - 7 * i for i in range(4)] + [0]], np.int32)
    t = np.arange(n)
    slots = torch.from_numpy(table[0, t // page].astype(np.int64) * page + t % page).to(device)
    cache.write(k, v, slots)
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    cache.read(slots, ko, vo)
    want = [F.encode(F.as64(x), fmt) for x in (k, v)]
    q = randn(g, (1, 16, dim), "bf16", device, 2.0)
    out, lse = torch.empty_like(q), torch.empty(1, 16, device=device)
    att = M.DeviceAttention(1, 16, heads, dim, n)
    att.rows(cache, q, out, torch.tensor([n], dtype=torch.int32, device=device), torch.from_numpy(table).to(device), lse=lse)
    torch.cuda.synchronize()
    for got, x in ((ko, want[0]), (vo, want[1])):
        assert np.all(np.abs(F.as64(got) - x) <= F.rounding(x, "bf16"))
    attend_check(q, out, lse, [n], [1], [tuple(want)], fmt, "bf16", 0, dim)
    cache.close()


DELTA = [
    # rows of each sequence, key heads, value heads, key dim, value dim, type, normalise, strongest decay
    ([100, 64], 1, 2, 256, 64, "f32", True, 0.2),
    ([90], 2, 2, 256, 256, "f16", True, 0.2),
    ([30] * 20 + [0] * 5 + [65], 2, 4, 64, 32, "bf16", True, 0.5),
    ([40, 3, 1, 0, 80], 1, 1, 16, 16, "f32", False, 0.1),
    ([2] * 600, 1, 1, 32, 16, "bf16", True, 0.3),
]


@pytest.mark.parametrize("case", range(len(DELTA)))
def test_delta_forms(device, case):
    lens, kh, vh, dk, dv, dtype, normalise, decay = DELTA[case]
    g = np.random.default_rng(800 + case)
    inputs = delta_inputs(g, device, lens, kh, vh, dk, dv, dtype, normalise, decay)
    q, k, v, gates, beta, states = inputs
    n = len(lens)
    before = F.as64(states)
    starts = torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device=device)
    out = torch.empty_like(v)
    h = M.DeviceDelta(sum(lens), n, kh, vh, dk, dv)
    slots = torch.arange(2 * n, dtype=torch.int32, device=device)
    print("delta", DELTA[case][1:], flush=True)
    h.rows(q, k, v, gates, beta, out, states, slots[:n], slots[n:], starts, normalise=normalise, most_rows=max(lens))
    torch.cuda.synchronize()
    delta_check(lens, inputs, F.as64(out), before[:n], F.as64(states)[n:2 * n], dk, dtype, normalise, dk ** -0.5, max(lens))


def test_delta_strides_and_unaligned_rows(device):
    # q, k and v as views of one projection whose rows are no multiple of 16 bytes; gates as its last columns.
    g = np.random.default_rng(21)
    lens, heads, dim = [70, 5], 2, 32
    rows, width = sum(lens), 3 * heads * dim + 2 * heads + 1
    for dtype in ("bf16", "f32"):
        y = randn(g, (rows, width), dtype, device)
        q, k, v = (y[:, i * heads * dim:(i + 1) * heads * dim].view(rows, heads, dim) for i in range(3))
        both = torch.from_numpy(g.random((rows, 2 * heads + 3)).astype(np.float32)).to(device)
        gates, beta = -both[:, :heads], both[:, heads:2 * heads]
        gates = torch.as_strided(torch.cat([gates, both], 1), (rows, heads), (3 * heads + 3, 1))
        states = randn(g, (4, heads, dim, dim), "f32", device, 0.5)
        before = F.as64(states)
        wide = torch.full((rows, heads, dim + 3), 7.0, dtype=y.dtype, device=device)
        out = wide[..., :dim]
        h = M.DeviceDelta(rows, 2, heads, heads, dim, dim)
        slots = torch.arange(4, dtype=torch.int32, device=device)
        starts = torch.tensor([0, 70, 75], dtype=torch.int32, device=device)
        for most in (1, 70):
            h.rows(q, k, v, gates, beta, out, states, slots[:2], slots[2:], starts, normalise=True, most_rows=most)
            torch.cuda.synchronize()
            assert bool((wide[..., dim:] == 7.0).all())
            delta_check(lens, (q, k, v, gates, beta, states), F.as64(out), before[:2], F.as64(states)[2:], dim, dtype, True,
                        dim ** -0.5, 70)


def test_graph_replays(device):
    # Every call in one graph, replayed with other inputs and eager work between: each replay gives the eager result.
    g = np.random.default_rng(22)
    rows, heads, dim = 70, 2, 64
    rotary = M.DeviceRotary(dim)
    cache, eager_cache = (M.DeviceCache(8, 16, heads, dim, "i8") for _ in range(2))
    att = M.DeviceAttention(rows, 4, heads, dim, 128)
    delta = M.DeviceDelta(rows, 1, heads, heads, dim, dim)
    q, k, v = (randn(g, (rows, n, dim), "bf16", device) for n in (4, heads, heads))
    gates, beta = -torch.rand(rows, heads, device=device), torch.rand(rows, heads, device=device)
    states = torch.zeros(2, heads, dim, dim, device=device)
    slots, positions = torch.arange(rows, device=device) + 16, torch.arange(rows, device=device)
    lens = torch.tensor([rows], dtype=torch.int32, device=device)
    table = torch.arange(1, 8, dtype=torch.int32, device=device)[None]
    starts = torch.tensor([0, rows], dtype=torch.int32, device=device)
    ids = torch.arange(2, dtype=torch.int32, device=device)

    def calls(cache):
        turned, out, mixed = torch.empty_like(q), torch.empty_like(q), torch.empty_like(v)
        back = torch.empty_like(k), torch.empty_like(v)
        rotary.apply(q, positions, turned)
        cache.write(k, v, slots, rotary=rotary, positions=positions)
        cache.read(slots, *back)
        att.rows(cache, turned, out, lens, table, starts=starts)
        delta.rows(k, k, v, gates, beta, mixed, states, ids[:1], ids[1:], starts, normalise=True)
        return turned, out, mixed, *back

    calls(cache)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = calls(cache)
    for i in range(4):
        q.copy_(randn(g, q.shape, "bf16", device))
        k.copy_(randn(g, k.shape, "bf16", device))
        want = [x.clone() for x in calls(eager_cache)]
        after = states[1].clone()
        states[1].zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x, y), i
        assert torch.equal(states[1], after), i


def test_nothing_to_do(device):
    empty = lambda *s, t=torch.float32: torch.zeros(*s, dtype=t, device=device)  # noqa: E731
    cache = M.DeviceCache(2, 4, 1, 16, "f8")
    none = empty(0, t=torch.int64)
    cache.write(empty(0, 1, 16), empty(0, 1, 16), none)
    cache.read(none, empty(0, 1, 16), empty(0, 1, 16))
    att = M.DeviceAttention(4, 1, 1, 16, 8)
    att.rows(cache, empty(0, 1, 16), empty(0, 1, 16), empty(2, t=torch.int32), empty(2, 2, t=torch.int32),
             starts=empty(3, t=torch.int32))
    # Sequences without tokens pass their states on.
    delta = M.DeviceDelta(4, 2, 1, 1, 16, 16)
    states = torch.rand(4, 1, 16, 16, device=device)
    ids = torch.arange(4, dtype=torch.int32, device=device)
    before = states.clone()
    x = empty(0, 1, 16)
    delta.rows(x, x, x, empty(0, 1), empty(0, 1), x, states, ids[:2], ids[2:], empty(3, t=torch.int32))
    torch.cuda.synchronize()
    assert torch.equal(states[:2], before[:2]) and torch.equal(states[2:], before[:2])


@pytest.mark.parametrize("what", ["k", "q", "v", "gate", "beta", "state", "zero key"])
@pytest.mark.parametrize("dtype,dk", [("f32", 64), ("bf16", 128), ("f16", 32)])
def test_delta_what_is_not_finite_goes_forward_only(device, dtype, dk, what):
    # Nothing before the token, no other sequence, head or column changes by a bit, in either form.
    g = np.random.default_rng(21)
    lens, kh, vh, dv = [150, 90], 2, 4, 32
    inputs = delta_inputs(g, device, lens, kh, vh, dk, dv, dtype, True, 0.2)
    starts = torch.tensor([0, 150, 240], dtype=torch.int32, device=device)
    slots = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=device)
    h = M.DeviceDelta(240, 2, kh, vh, dk, dv)
    eps = 0.0 if what == "zero key" else 1e-6

    def run(x, most):
        q, k, v, gates, beta, states = (y.clone() for y in x)
        out = torch.empty_like(v)
        h.rows(q, k, v, gates, beta, out, states, slots[0], slots[1], starts, normalise=True, eps=eps, most_rows=most)
        torch.cuda.synchronize()
        return F.as64(out), F.as64(states)[2:4]

    for t, bad in ((70, float("inf")), (131, float("nan")), (149, float("-inf")), (0, float("nan"))):
        if what == "gate" and bad == float("-inf"):
            continue  # forgets the state, and is finite
        spoilt = [x.clone() for x in inputs]
        q, k, v, gates, beta, states = spoilt
        if what == "k":
            k[t, 1, 5] = bad
        elif what == "q":
            q[t, 1, 5] = bad
        elif what == "v":
            v[t, 2, 3] = bad
        elif what == "gate":
            gates[t, 2] = bad
        elif what == "beta":
            beta[t, 2] = bad
        elif what == "state":
            states[0, 2, 5, 3] = bad
        else:
            k[t, 1] = 0.0
        wants = []
        with np.errstate(all="ignore"):
            for s, rows in enumerate((slice(0, 150), slice(150, 240))):
                x = [F.as64(y)[rows] for y in spoilt[:5]]
                wants.append(F.delta(*x, F.as64(states)[s], dk ** -0.5, eps))
        for most in (1, 150):
            print("delta", what, t, bad, dtype, most, flush=True)
            clean, clean_state = run(inputs, most)
            out, state = run(spoilt, most)
            for s, rows in enumerate((slice(0, 150), slice(150, 240))):
                odd, odd_state = ~np.isfinite(wants[s][0]), ~np.isfinite(wants[s][1])
                assert np.array_equal(~np.isfinite(out[rows]), odd)
                assert np.array_equal(~np.isfinite(state[s]), odd_state)
                assert np.array_equal(out[rows][~odd], clean[rows][~odd])
                assert np.array_equal(state[s][~odd_state], clean_state[s][~odd_state])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [1, 17, 40, 64, 70, 129])
def test_delta_norms_without_epsilon(device, dtype, n):
    # The oracle's 1e-6 moves a norm of about 8 by a part in 10^8, far inside the bounds.
    g = np.random.default_rng(22)
    inputs = delta_inputs(g, device, [n], 1, 2, 64, 32, dtype, True, 0.2)
    q, k, v, gates, beta, states = inputs
    before, out = F.as64(states), torch.empty_like(v)
    h = M.DeviceDelta(n, 1, 1, 2, 64, 32)
    slots = torch.tensor([0, 1], dtype=torch.int32, device=device)
    starts = torch.tensor([0, n], dtype=torch.int32, device=device)
    for most in (1, n):
        h.rows(q, k, v, gates, beta, out, states, slots[:1], slots[1:], starts, normalise=True, eps=0.0, most_rows=most)
        torch.cuda.synchronize()
        delta_check([n], inputs, F.as64(out), before[:1], F.as64(states)[1:2], 64, dtype, True, 64 ** -0.5, n)
