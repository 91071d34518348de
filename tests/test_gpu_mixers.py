"""The token mixers on the GPU against float64 statements of their formulas
(mixer_fixtures.py). Every bound is formed from the operation counts before the
comparison: f32 sums of n terms are off by at most n 2^-24 of the sum of
magnitudes, and each rounding to an element type by half a unit."""
import numpy as np
import pytest
import torch

import mixer_fixtures as F
import rl_mixers as M
import rl_sampler as R

pytestmark = pytest.mark.gpu


def randn(g, shape, dtype, device, sigma=1.0):
    return torch.from_numpy((g.standard_normal(shape) * sigma).astype(np.float32)).to(device).to(F.TYPES[dtype])


def strided(x, pad_row, pad_head, device):
    """A copy of x [rows][heads][dim] whose rows and heads lie further apart."""
    rows, heads, dim = x.shape
    buf = torch.full((rows, heads * (dim + pad_head) + pad_row), float("nan"), dtype=x.dtype, device=device)
    y = buf[:, :heads * (dim + pad_head)].view(rows, heads, dim + pad_head)[..., :dim] if pad_row == 0 else \
        torch.as_strided(buf, (rows, heads, dim), (buf.stride(0), dim + pad_head, 1))
    y.copy_(x)
    return y


# -------------------------------------------------------------- rotary --
ROTARY = [
    # rows, heads, second heads, dim, dims, layout, in, out, scaling, pads
    (1, 16, 4, 256, 64, "half", "bf16", "bf16", "none", (0, 0)),
    (5, 3, 1, 128, 128, "interleaved", "f32", "f32", "yarn", (0, 0)),
    (7, 2, 2, 80, 80, "half", "f16", "f16", "linear", (0, 0)),
    (3, 2, 0, 80, 20, "half", "bf16", "f32", "none", (0, 0)),
    (4, 1, 5, 77, 30, "half", "f32", "f32", "ntk", (3, 1)),
    (4, 5, 1, 33, 2, "interleaved", "f16", "bf16", "none", (1, 0)),
    (9, 2, 1, 512, 512, "interleaved", "f32", "f16", "yarn", (0, 8)),
    (300, 2, 1, 64, 32, "half", "bf16", "bf16", "none", (16, 8)),
]


@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("case", range(len(ROTARY)))
def test_rotary(device, case, inverse):
    rows, heads, more, dim, dims, layout, tin, tout, scaling, pads = ROTARY[case]
    g = np.random.default_rng(100 + case)
    spec = dict(base=1e4, scaling=scaling, factor=4.0, original=4096)
    radians, magnitude = F.frequencies(dims, **spec)
    r = M.DeviceRotary(dims, layout=layout, **spec)
    got_radians, got_magnitude = r.frequencies()
    assert np.allclose(got_radians, radians, rtol=1e-14, atol=0) and abs(got_magnitude - magnitude) < 1e-14
    positions = g.integers(-200000, 2000000, rows)
    positions[0] = 0
    xs = [randn(g, (rows, h, dim), tin, device) for h in (heads, more) if h]
    ins = [strided(x, *pads, device) for x in xs]
    outs = [strided(torch.zeros_like(x).to(F.TYPES[tout]), *pads, device) for x in xs]
    second = dict(second=ins[1], second_out=outs[1]) if more else {}
    print("rotary", ROTARY[case], inverse, flush=True)
    r.apply(ins[0], torch.from_numpy(positions).to(device), outs[0], inverse=inverse, **second)
    torch.cuda.synchronize()
    for x, out in zip(xs, outs):
        x, y = F.as64(x), F.as64(out)
        want = F.turn(x, positions, radians, magnitude, layout, -1.0 if inverse else 1.0)
        # Angle 2.5e-7, sine or cosine 2.4e-7 (4 units of 2^-24), magnitude, two products and their sum: 5 2^-24.
        size = F.turn(np.abs(x), np.zeros(rows), radians, 1.0, layout)
        n = dims // 2
        i = np.arange(n)
        a, b = (i, i + n) if layout == "half" else (2 * i, 2 * i + 1)
        size[..., a] = size[..., b] = np.abs(x[..., a]) + np.abs(x[..., b])
        slack = magnitude * size * (2.5e-7 + 2.4e-7 + 5 * 2.0 ** -24)
        slack[..., dims:] = 0
        assert np.all(np.abs(y - want) <= slack + F.rounding(np.abs(want) + slack, tout)), np.abs(y - want).max()
    r.close()


def test_rotary_in_place_copies_and_padding(device):
    g = np.random.default_rng(1)
    x = randn(g, (6, 3, 96), "bf16", device)
    positions = torch.arange(6, device=device) * 1000
    r = M.DeviceRotary(32)
    out = torch.empty_like(x)
    r.apply(x, positions, out)
    y = strided(x, 16, 16, device)
    r.apply(y, positions)
    assert torch.equal(out, y) and torch.equal(out[..., 32:], x[..., 32:])
    assert torch.equal(out[0], x[0])  # position 0
    r.apply(x[:0], positions[:0])  # nothing to do


def test_rotary_inverse_is_the_adjoint_and_takes_back(device):
    # The map is linear, so differences are the map itself: <T x, y> = <x, T' y>
    # for the gradient T', column by column of a basis, and T' T = m^2.
    r = M.DeviceRotary(16, layout="interleaved", scaling="yarn", factor=8.0, original=2048, base=5e5)
    _, m = r.frequencies()
    positions = torch.full((24,), 12345, dtype=torch.int64, device=device)
    basis = torch.eye(24, device=device).view(24, 1, 24)
    forward, back, both = (torch.empty_like(basis) for _ in range(3))
    r.apply(basis, positions, forward)
    r.apply(basis, positions, back, inverse=True)
    r.apply(forward, positions, both, inverse=True)
    torch.cuda.synchronize()
    assert np.array_equal(F.as64(forward)[:, 0], F.as64(back)[:, 0].T)
    want = np.eye(24)
    want[:16, :16] *= m * m
    # Two turns, each off by at most 8.4e-7 m of a unit vector.
    assert np.abs(F.as64(both)[:, 0] - want).max() <= 2 * 8.4e-7 * m * m
    # A finite difference of the forward map along one direction.
    g = np.random.default_rng(2)
    x, d = randn(g, (24, 1, 24), "f32", device), randn(g, (24, 1, 24), "f32", device)
    y0, y1, grad = (torch.empty_like(x) for _ in range(3))
    r.apply(x - d, positions, y0)
    r.apply(x + d, positions, y1)
    w = randn(g, (24, 1, 24), "f32", device)
    r.apply(w, positions, grad, inverse=True)
    torch.cuda.synchronize()
    slope = (F.as64(w) * (F.as64(y1) - F.as64(y0)) / 2).sum()
    size = (np.abs(F.as64(w)) * (np.abs(F.as64(x)) + np.abs(F.as64(d)))).sum()
    assert abs(slope - (F.as64(grad) * F.as64(d)).sum()) <= 4 * 8.4e-7 * m * 2 * size


# --------------------------------------------------------------- cache --
CACHE = [
    # rows, heads, dim, page, pages, format, type, pads
    (1, 1, 16, 1, 3, "i8", "f32", (0, 0)),
    (37, 2, 80, 24, 5, "f8", "bf16", (0, 0)),
    (64, 8, 128, 32, 64, "i8", "bf16", (0, 0)),
    (100, 3, 256, 7, 20, "f8", "f16", (0, 0)),
    (33, 2, 112, 16, 9, "bf16", "f32", (3, 5)),
    (20, 1, 64, 64, 2, "f16", "f32", (8, 8)),
    (50, 5, 96, 10, 11, "i8", "f16", (1, 0)),
]


@pytest.mark.parametrize("turned", [0, 1, 2])
@pytest.mark.parametrize("case", range(len(CACHE)))
def test_cache_write_and_read(device, case, turned):
    rows, heads, dim, page, pages, fmt, dtype, pads = CACHE[case]
    g = np.random.default_rng(200 + 10 * case + turned)
    k, v = (randn(g, (rows, heads, dim), dtype, device, s) for s in (3.0, 0.2))
    if rows > 3:
        k[1], v[2, 0] = 0, 0
        k[3, 0, 5], v[3, heads - 1, 1] = float("inf"), float("nan")
    slots = g.permutation(pages * page)[:rows]
    cache = M.DeviceCache(pages, page, heads, dim, fmt)
    rotary, positions, radians, layout = None, None, None, ["half", "interleaved"][case % 2]
    if turned:
        dims = dim if turned == 1 else max(2, dim // 4 // 2 * 2 - 2)
        rotary, (radians, _) = M.DeviceRotary(dims, layout=layout), F.frequencies(dims, 1e4)
        positions = torch.from_numpy(g.integers(0, 100000, rows)).to(device)
    print("cache", CACHE[case], turned, flush=True)
    dev_slots = torch.from_numpy(slots).to(device)
    cache.write(strided(k, *pads, device), strided(v, *pads, device), dev_slots, rotary=rotary, positions=positions)
    ko, vo = (strided(torch.zeros(rows, heads, dim, device=device), *pads, device) for _ in range(2))
    cache.read(dev_slots, ko, vo)
    torch.cuda.synchronize()
    want_v = F.encode(F.as64(v), fmt)
    assert np.array_equal(F.as64(vo), want_v, equal_nan=True)
    if not turned:
        assert np.array_equal(F.as64(ko), F.encode(F.as64(k), fmt), equal_nan=True)
    else:
        x = F.as64(k)
        fine = np.isfinite(x).all(-1)
        x[~fine] = 0
        y = F.turn(x, positions.cpu().numpy(), radians, 1.0, layout)
        # The turn is off by 8.4e-7 of the pair; a code then by half a step, of its value where it is a float.
        near = 8.4e-7 * 2 * np.abs(x).max(-1, keepdims=True)
        if fmt == "i8":
            slack = near + np.abs(y).max(-1, keepdims=True) / 127 * 0.5 * (1 + 1e-5)
        elif fmt == "f8":  # half a unit of 4 bits, or half the smallest step 2^-9
            slack = near + np.maximum(np.abs(y) * 2.0 ** -4, np.abs(y).max(-1, keepdims=True) / 448 * 2.0 ** -10) * (1 + 1e-5)
        else:
            slack = near + F.rounding(np.abs(y) + near, fmt)
        got = F.as64(ko)
        assert np.all(np.abs(got - y)[fine] <= slack[fine] if fmt not in ("f16", "bf16") else
                      (np.abs(got - y) <= slack)[fine])
        if fmt in ("i8", "f8"):
            assert np.isnan(got[~fine]).all()
    cache.close()


def test_cache_slots_outside_are_left_out(device):
    g = np.random.default_rng(3)
    cache = M.DeviceCache(2, 4, 1, 32, "i8")
    k, v = (randn(g, (5, 1, 32), "f32", device) for _ in range(2))
    slots = torch.tensor([3, -1, 8, 2 ** 40, 7], device=device)
    cache.write(k, v, slots)
    ko, vo = torch.empty(8, 1, 32, device=device), torch.empty(8, 1, 32, device=device)
    cache.read(torch.arange(8, device=device), ko, vo)
    torch.cuda.synchronize()
    for slot in range(8):
        row = {3: 0, 7: 4}.get(slot)
        want = np.zeros((1, 32)) if row is None else F.encode(F.as64(k[row]), "i8")
        assert np.array_equal(F.as64(ko[slot]), want), slot
    cache.read(slots, ko[:5], vo[:5])
    torch.cuda.synchronize()
    assert np.isnan(F.as64(ko[1:4])).all() and np.isnan(F.as64(vo[1:4])).all() and np.isfinite(F.as64(ko[4])).all()


def test_cache_tiny_and_large_steps(device):
    # Steps that are subnormal, zero (max below 127 halves of the smallest number) and near the largest.
    k = torch.zeros(4, 1, 16, device=device)
    k[0, 0, :3] = torch.tensor([1e-40, -5e-41, 2e-41])
    k[1, 0, :2] = torch.tensor([1.4e-45, -2.8e-45])
    k[2, 0, :3] = torch.tensor([3.4e38, -1e38, 1.0])
    k[3, 0, :4] = torch.tensor([1.0, 0.5, 0.25, -0.5])  # halves of the largest: ties
    for fmt in ("i8", "f8"):
        cache = M.DeviceCache(1, 4, 1, 16, fmt)
        out = torch.empty_like(k), torch.empty_like(k)
        slots = torch.arange(4, device=device)
        cache.write(k, k, slots)
        cache.read(slots, *out)
        torch.cuda.synchronize()
        assert np.array_equal(F.as64(out[0]), F.encode(F.as64(k), fmt)), fmt
        cache.close()


# ----------------------------------------------------------- attention --
ATTEND = [
    # lens, rows of each, q heads, kv heads, dim, page, format, type, window
    ([1], [1], 1, 1, 16, 1, "bf16", "bf16", 0),
    ([611], [1], 16, 4, 256, 32, "bf16", "bf16", 0),
    ([5, 0, 64, 129, 1000], [1, 1, 1, 1, 1], 8, 2, 128, 16, "i8", "bf16", 0),
    ([5, 0, 64, 129, 1000], [1, 1, 1, 1, 1], 8, 2, 128, 16, "f8", "f16", 0),
    ([2100], [9], 8, 2, 256, 24, "f16", "f32", 0),
    ([300, 7, 40], [3, 7, 0], 6, 3, 80, 7, "i8", "f32", 0),
    ([300, 7, 40], [3, 9, 1], 12, 1, 96, 40, "f8", "f32", 5),   # rows before the first token
    ([900, 33], [17, 1], 4, 4, 64, 64, "bf16", "f32", 100),
    ([4097], [2], 64, 1, 112, 128, "f16", "f16", 1),
    ([513, 512, 511], [5, 5, 5], 32, 2, 48, 48, "i8", "f16", 333),
    ([3000, 31, 32], [1, 1, 1], 40, 8, 128, 20, "bf16", "bf16", 0),
    ([20000], [1], 5, 1, 64, 16, "f8", "bf16", 0),
]


def paged(g, lens, page, spare=2):
    """Pages in random order for each sequence: (table, pages in all)."""
    need = [-(-n // page) for n in lens]
    width = max(max(need), 1)
    order = g.permutation(sum(need) + spare)
    table = np.full((len(lens), width), -7, np.int32)  # entries past a sequence's end are no pages
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table, len(order)


def attend_case(g, device, lens, counts, qh, kv, dim, page, fmt, dtype, window, fill=None, scale=None, spread=2.0):
    source = "f16" if fmt == "f16" else "bf16"
    table, pages = paged(g, lens, page)
    cache = M.DeviceCache(pages, page, kv, dim, fmt)
    if fill is not None:  # what stands in slots that no sequence holds
        rest = torch.full((pages * page, kv, dim), fill, device=device)
        cache.write(rest, rest, torch.arange(pages * page, device=device))
    stored = []
    for i, n in enumerate(lens):
        k, v = (randn(g, (n, kv, dim), source, device) for _ in range(2))
        t = np.arange(n)
        slots = torch.from_numpy(table[i, t // page].astype(np.int64) * page + t % page).to(device)
        if n:
            cache.write(k, v, slots)
        stored.append((F.encode(F.as64(k), fmt), F.encode(F.as64(v), fmt)))
    rows = sum(counts)
    q = randn(g, (rows, qh, dim), dtype, device, spread)
    starts = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32, device=device)
    out = torch.full_like(q, 7.0)
    lse = torch.full((rows, qh), 7.0, device=device)
    att = M.DeviceAttention(max(rows, 1), qh, kv, dim, max(max(lens), 1))
    single = all(c == 1 for c in counts)
    call = lambda **kw: att.rows(cache, q, out, torch.tensor(lens, dtype=torch.int32, device=device),  # noqa: E731
                                 torch.from_numpy(table).to(device), starts=None if single else starts, lse=lse,
                                 window=window, scale=scale, **kw)
    return cache, att, q, out, lse, starts, stored, call, table


def attend_check(q, out, lse, lens, counts, stored, fmt, dtype, window, dim, scale=None):
    scale = dim ** -0.5 if scale is None else scale
    at = 0
    for n, c, (k, v) in zip(lens, counts, stored):
        x, y, z = F.as64(q[at:at + c]), F.as64(out[at:at + c]), F.as64(lse[at:at + c])
        want, want_lse, mass, size = F.attention(x, k, v, scale, n, window)
        # Scores: dim products and sums, the scale and steps, in f32, and for f32 queries their split (2^-20 at worst).
        d = size * ((dim + 8) * 2.0 ** -24 + (2.0 ** -20 if dtype == "f32" else 0))
        # Weights: e^d, the exponential (2^-21), and rounding to 16 bits (f16 2^-11, bf16 2^-8; f32 queries: two parts, 2^-16);
        # the sums over tokens, at most a few hundred in a row before tiles are joined.
        u = {"f32": 2.0 ** -16, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[dtype]
        w = 2 * d + 2.0 ** -21 + 600 * 2.0 ** -24 + u
        slack = mass * w[..., None]
        assert np.all(np.abs(y - want) <= slack + F.rounding(np.abs(want) + slack, dtype)), (
            n, c, np.abs(y - want).max())
        none = np.isneginf(want_lse)
        assert np.array_equal(np.isneginf(z), none)
        assert np.all(np.abs(z - want_lse)[~none] <=
                      (d + 2.0 ** -20 + 600 * 2.0 ** -24 + np.abs(want_lse) * 2.0 ** -23)[~none])
        at += c


@pytest.mark.parametrize("case", range(len(ATTEND)))
def test_attention(device, case):
    lens, counts, qh, kv, dim, page, fmt, dtype, window = ATTEND[case]
    g = np.random.default_rng(300 + case)
    cache, att, q, out, lse, starts, stored, call, _ = attend_case(g, device, *ATTEND[case], fill=float("nan"))
    print("attend", ATTEND[case], flush=True)
    call(most_rows=max(counts))
    torch.cuda.synchronize()
    attend_check(q, out, lse, lens, counts, stored, fmt, dtype, window, dim)
    first, first_lse = out.clone(), lse.clone()
    call()  # without the bound on rows: the same bits or another split, the same bounds
    torch.cuda.synchronize()
    attend_check(q, out, lse, lens, counts, stored, fmt, dtype, window, dim)
    call(most_rows=max(counts))
    torch.cuda.synchronize()
    assert torch.equal(out, first) and torch.equal(lse, first_lse)  # no result depends on an order of arrival


def test_attention_strides_and_large_scores(device):
    # Scores in the thousands: the largest dominates; queries and outputs with padded rows and heads.
    case = ([130, 77], [2, 1], 4, 2, 64, 16, "bf16", "f32", 0)
    g = np.random.default_rng(5)
    cache, att, q, out, lse, starts, stored, call, table = attend_case(g, device, *case, spread=60.0)
    lens = torch.tensor(case[0], dtype=torch.int32, device=device)
    for pads in ((0, 0), (1, 3), (8, 4)):
        qs, outs = strided(q, *pads, device), strided(out, *pads, device)
        att.rows(cache, qs, outs, lens, torch.from_numpy(table).to(device), starts=starts, lse=lse, scale=1.0)
        torch.cuda.synchronize()
        attend_check(q, outs, lse, *case[:2], stored, "bf16", "f32", 0, 64, scale=1.0)


def test_attention_past_its_bounds_gives_nan(device):
    case = ([100, 50, 60], [1, 1, 1], 2, 1, 32, 16, "i8", "bf16", 0)
    g = np.random.default_rng(6)
    cache, att, q, out, lse, starts, stored, call, table = attend_case(g, device, *case)
    table = table.copy()
    table[1, 2] = 10 ** 6  # no page of the cache
    dev = lambda t: torch.from_numpy(np.ascontiguousarray(t, np.int32)).to(device)  # noqa: E731
    att.rows(cache, q, out, dev([100, 50, 60]), dev(table), lse=lse, max_len=99)
    torch.cuda.synchronize()
    assert np.isnan(F.as64(out[:2])).all() and np.isnan(F.as64(lse[:2])).all()
    attend_check(q[2:], out[2:], lse[2:], [60], [1], stored[2:], "i8", "bf16", 0, 32)
    att.rows(cache, q, out, dev([100, 32, 60]), dev(table[:, :4]), lse=lse)  # 100 tokens need 7 pages, the table has 4
    torch.cuda.synchronize()
    assert np.isnan(F.as64(out[0])).all()
    attend_check(q[1:], out[1:], lse[1:], [32, 60], [1, 1], [tuple(x[:32] for x in stored[1]), stored[2]], "i8", "bf16",
                 0, 32)
    # Three rows of one sequence where the call says there is one.
    att.rows(cache, q, out, dev([100]), dev(table[:1]), starts=dev([0, 3]), lse=lse, most_rows=1)
    torch.cuda.synchronize()
    assert np.isnan(F.as64(out)).all()


def test_attention_infinities_in_sight_stay_in_their_rows(device):
    # A NaN key reaches the rows that see it and no other.
    g = np.random.default_rng(7)
    cache = M.DeviceCache(4, 16, 1, 32, "bf16")
    k, v = (randn(g, (40, 1, 32), "bf16", device) for _ in range(2))
    k[38, 0, 3], v[39, 0, 1] = float("nan"), float("inf")
    cache.write(k, v, torch.arange(40, device=device))
    q = randn(g, (4, 2, 32), "bf16", device)
    out, lse = torch.empty_like(q), torch.empty(4, 2, device=device)
    att = M.DeviceAttention(4, 2, 1, 32, 64)
    att.rows(cache, q, out, torch.tensor([40], dtype=torch.int32, device=device),
             torch.arange(4, dtype=torch.int32, device=device)[None], starts=torch.tensor([0, 4], dtype=torch.int32, device=device),
             lse=lse)
    torch.cuda.synchronize()
    attend_check(q[:2], out[:2], lse[:2], [38], [2], [(F.as64(k[:38]), F.as64(v[:38]))], "bf16", "bf16", 0, 32)
    assert np.isnan(F.as64(out[2:])).all()


# --------------------------------------------------------------- delta --
DELTA = [
    # rows of each sequence, key heads, value heads, key dim, value dim, type, normalise, strongest decay
    ([1], 1, 1, 16, 16, "f32", True, 1.0),
    ([1] * 13, 2, 4, 128, 128, "bf16", True, 1.0),
    ([9], 4, 8, 128, 128, "bf16", True, 1.0),
    ([5, 0, 17, 3], 2, 2, 64, 96, "f16", True, 3.0),
    ([63, 64, 65, 1], 1, 2, 96, 48, "bf16", True, 0.3),
    ([130, 40], 2, 2, 64, 64, "f32", False, 0.5),
    ([257], 1, 2, 256, 80, "bf16", True, 0.1),
    ([200, 0, 191], 1, 2, 128, 128, "f16", False, 20.0),
    ([128, 129], 2, 2, 112, 256, "f32", True, 0.05),
    ([700], 1, 1, 128, 16, "bf16", True, 0.01),
]


def delta_inputs(g, device, lens, kh, vh, dk, dv, dtype, normalise, decay):
    rows = sum(lens)
    q = randn(g, (rows, kh, dk), dtype, device)
    k = g.standard_normal((rows, kh, dk))
    if not normalise:
        k /= np.sqrt((k * k).sum(-1, keepdims=True))
    k = torch.from_numpy(k.astype(np.float32)).to(device).to(F.TYPES[dtype])
    v = randn(g, (rows, vh, dv), dtype, device)
    gates = torch.from_numpy((-decay * g.random((rows, vh))).astype(np.float32)).to(device)
    beta = torch.from_numpy(g.random((rows, vh)).astype(np.float32)).to(device)
    states = randn(g, (2 * len(lens) + 1, vh, dk, dv), "f32", device, 0.5)
    return q, k, v, gates, beta, states


def delta_check(lens, inputs, out, before, after, dk, dtype, normalise, scale, most, untouched=()):
    q, k, v, gates, beta, _ = (F.as64(x) for x in inputs)
    at = 0
    for s, n in enumerate(lens):
        rows = slice(at, at + n)
        at += n
        want, state = F.delta(q[rows], k[rows], v[rows], gates[rows], beta[rows], before[s], scale, 1e-6 if normalise else -1.0)
        got, got_state = out[rows], after[s]
        # With |k| <= 1 + 2^-7 and 0 <= beta <= 1 a step does not grow an error by more than 2^-6 of itself, so a
        # column's error is at most the sum of the steps'. One token after the other a step adds (2 dk + 16) 2^-24 of
        # (|S| + |v|); in chunks of 64 the products with the state are good to 2^-16 and the 64 corrected values of a
        # chunk carry its errors on, so a chunk adds at most 64 times 2^-16 (|S| + |v|), a sixteenth of it in norm.
        top = np.sqrt((v[rows] ** 2).sum((0, 1)).max() if n else 0) + np.abs(before[s]).max() * np.sqrt(dk)
        grow = 1.0 if normalise else (1 + 2.0 ** -6) ** min(n, 64)
        step = max((2 * dk + 16) * 2.0 ** -24, 2.0 ** -14 / 4)
        slack = grow * top * step * (1 + n / 64 if most > 1 else 1)
        assert np.abs(got_state - state).max() <= slack, (s, n, np.abs(got_state - state).max(), slack)
        size = np.sqrt((q[rows] ** 2).sum(-1).max()) if n and not normalise else 1.0
        # The output's products round the state and the corrected values to the element type of the call.
        unit = {"f32": step, "f16": 2.0 ** -10, "bf16": 2.0 ** -7}[dtype] if most > 1 else step
        near = abs(scale) * size * (slack + top * unit)
        assert np.all(np.abs(got - want) <= near + F.rounding(np.abs(want) + near, dtype)), (
            s, n, np.abs(got - want).max(), near)
        # The error's norm is far below its largest value's bound: held to an eighth.
        if n:
            assert np.sqrt(((got_state - state) ** 2).mean()) <= slack / 8


@pytest.mark.parametrize("hint", [True, False])
@pytest.mark.parametrize("case", range(len(DELTA)))
def test_delta(device, case, hint):
    lens, kh, vh, dk, dv, dtype, normalise, decay = DELTA[case]
    g = np.random.default_rng(400 + case)
    inputs = delta_inputs(g, device, lens, kh, vh, dk, dv, dtype, normalise, decay)
    q, k, v, gates, beta, states = inputs
    n, rows = len(lens), sum(lens)
    before = F.as64(states)
    order = g.permutation(2 * n + 1)
    slots_in, slots_out, rest = order[:n], order[n:2 * n], order[2 * n]
    starts = torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device=device)
    out = torch.full_like(v, 7.0)
    h = M.DeviceDelta(rows, n, kh, vh, dk, dv)
    dev = lambda t: torch.from_numpy(np.ascontiguousarray(t, np.int32)).to(device)  # noqa: E731
    print("delta", DELTA[case], hint, flush=True)
    single = max(lens) == 1
    call = lambda a, b: h.rows(q, k, v, gates, beta, out, states, dev(a), dev(b), None if single else starts,  # noqa: E731
                               normalise=normalise, most_rows=max(lens) if hint else 0)
    call(slots_in, slots_out)
    torch.cuda.synchronize()
    after = F.as64(states)
    assert np.array_equal(after[slots_in], before[slots_in]) and np.array_equal(after[rest], before[rest])
    most = max(lens) if hint else rows
    delta_check(lens, inputs, F.as64(out), before[slots_in], after[slots_out], dk, dtype, normalise, dk ** -0.5, most)
    # In place gives the same bits.
    first = out.clone()
    states.copy_(torch.from_numpy(before).to(device).float())
    call(slots_in, slots_in)
    torch.cuda.synchronize()
    assert torch.equal(out, first) and np.array_equal(F.as64(states)[slots_in], after[slots_out])
    # From nothing, to nowhere.
    zero = torch.zeros_like(states)
    h.rows(q, k, v, gates, beta, first, zero, dev(slots_in), dev([-1] * n), None if single else starts,
           normalise=normalise, most_rows=max(lens) if hint else 0)
    assert not zero.any()
    call([-1] * n, [-1] * n)
    torch.cuda.synchronize()
    assert torch.equal(out, first)


def test_delta_strong_decays_and_resets(device):
    # A gate of -inf forgets the state; -1e4 does the same to f32.
    lens, kh, vh, dk, dv = [150], 1, 2, 64, 32
    g = np.random.default_rng(8)
    inputs = delta_inputs(g, device, lens, kh, vh, dk, dv, "bf16", True, 0.2)
    q, k, v, gates, beta, states = inputs
    gates[70, 0], gates[71, 1], gates[100, 0], gates[3, 1] = -np.inf, -1e4, -300.0, -np.inf
    out = torch.empty_like(v)
    before = F.as64(states)
    h = M.DeviceDelta(150, 1, kh, vh, dk, dv)
    slots = torch.tensor([0, 1], dtype=torch.int32, device=device)
    starts = torch.tensor([0, 150], dtype=torch.int32, device=device)
    for most in (1, 150):  # either form
        h.rows(q, k, v, gates, beta, out, states, slots[:1], slots[1:], starts, normalise=True, most_rows=most)
        torch.cuda.synchronize()
        delta_check(lens, inputs, F.as64(out), before[:1], F.as64(states)[1:2], dk, "bf16", True, dk ** -0.5, 150)


def test_delta_slots_and_neighbours(device):
    # Slots from the pool's end on read as NaN and are not written; a sequence's NaN stays its own.
    g = np.random.default_rng(9)
    lens = [70, 70, 70]
    inputs = delta_inputs(g, device, lens, 1, 1, 32, 32, "f16", True, 0.2)
    q, k, v, gates, beta, states = inputs
    v[75] = float("nan")
    before = F.as64(states)
    out = torch.empty_like(v)
    h = M.DeviceDelta(210, 3, 1, 1, 32, 32)
    dev = lambda t: torch.from_numpy(np.ascontiguousarray(t, np.int32)).to(device)  # noqa: E731
    for most in (1, 70):
        h.rows(q, k, v, gates, beta, out, states, dev([0, 1, 99]), dev([3, 4, 100]), dev([0, 70, 140, 210]),
               normalise=True, most_rows=most)
        torch.cuda.synchronize()
        after = F.as64(states)
        delta_check(lens[:1], [x[:70] if i < 5 else x for i, x in enumerate(inputs)], F.as64(out), before[:1],
                    after[3:4], 32, "f16", True, 32 ** -0.5, 70)
        assert np.isnan(after[4]).all() and np.isnan(F.as64(out[140:])).all()
        assert np.isnan(F.as64(out[75:140])).all()
        assert np.array_equal(after[[0, 1, 2, 5, 6]], before[[0, 1, 2, 5, 6]])


def test_delta_rows_once_or_in_parts(device):
    # A prompt in one call or its last tokens one by one: the same within the bounds.
    g = np.random.default_rng(10)
    lens = [140]
    inputs = delta_inputs(g, device, lens, 2, 2, 64, 64, "bf16", True, 0.3)
    q, k, v, gates, beta, states = inputs
    before = F.as64(states)
    out = torch.empty_like(v)
    h = M.DeviceDelta(140, 1, 2, 2, 64, 64)
    slots = torch.tensor([0, 1], dtype=torch.int32, device=device)
    h.rows(q[:130], k[:130], v[:130], gates[:130], beta[:130], out[:130], states, slots[:1], slots[1:],
           torch.tensor([0, 130], dtype=torch.int32, device=device), normalise=True)
    for t in range(130, 140):
        s = slice(t, t + 1)
        h.rows(q[s], k[s], v[s], gates[s], beta[s], out[s], states, slots[1:], slots[1:], normalise=True)
    torch.cuda.synchronize()
    delta_check(lens, inputs, F.as64(out), before[:1], F.as64(states)[1:2], 64, "bf16", True, 64 ** -0.5, 140)


def test_calls_on_another_stream(device):
    g = np.random.default_rng(11)
    x = randn(g, (64, 4, 64), "f32", device)
    positions = torch.arange(64, device=device)
    r = M.DeviceRotary(64)
    want = torch.empty_like(x)
    r.apply(x, positions, want)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    out = torch.empty_like(x)
    with torch.cuda.stream(side):
        r.apply(x, positions, out)
    side.synchronize()
    assert torch.equal(out, want)
    out.zero_()
    torch.cuda.synchronize()
    r.apply(x, positions, out, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(out, want)


def test_refusals(device):
    dev = lambda *s, t=torch.float32: torch.zeros(*s, dtype=t, device=device)  # noqa: E731
    r = M.DeviceRotary(64)
    cache = M.DeviceCache(2, 16, 2, 64, "f16")
    att = M.DeviceAttention(4, 4, 2, 64, 32)
    delta = M.DeviceDelta(4, 2, 2, 4, 64, 64)
    positions, slots = dev(4, t=torch.int64), dev(4, t=torch.int64)
    lens, table = dev(4, t=torch.int32), dev(4, 2, t=torch.int32)

    def refused(code, f, *a, **kw):
        with pytest.raises(R.SamplerError) as e:
            f(*a, **kw)
        assert e.value.code == code, e.value

    refused(R.RL_ERR_ARGUMENT, r.apply, dev(4, 1, 32), positions)  # fewer values than are turned
    refused(R.RL_ERR_ARGUMENT, r.apply, dev(4, 1, 64), positions, second=dev(4, 1, 64, t=torch.float16))
    refused(R.RL_ERR_ARGUMENT, cache.write, dev(4, 2, 32), dev(4, 2, 32), slots)
    refused(R.RL_ERR_ARGUMENT, cache.write, dev(4, 2, 64), dev(4, 2, 64, t=torch.float16), slots)
    refused(R.RL_ERR_ARGUMENT, cache.write, dev(4, 2, 64), dev(4, 2, 64), slots, rotary=M.DeviceRotary(128), positions=positions)
    refused(R.RL_ERR_ARGUMENT, cache.read, slots, dev(1, 1, 64).expand(4, 2, 64), dev(4, 2, 64))  # rows over each other
    q = dev(4, 4, 64, t=torch.float16)
    refused(R.RL_ERR_ARGUMENT, att.rows, cache, q.bfloat16(), q.bfloat16(), lens, table)  # an f16 cache
    refused(R.RL_ERR_ARGUMENT, att.rows, cache, q, q.float(), lens, table)
    refused(R.RL_ERR_ARGUMENT, att.rows, cache, q, q, lens[:3], table[:3])  # four rows, three sequences, no starts
    refused(R.RL_ERR_CAPACITY, att.rows, cache, dev(5, 4, 64), dev(5, 4, 64), dev(5, t=torch.int32), dev(5, 2, t=torch.int32))
    refused(R.RL_ERR_CAPACITY, att.rows, cache, q, q, lens, table, max_len=33)
    refused(R.RL_ERR_ARGUMENT, att.rows, M.DeviceCache(2, 16, 1, 64, "f16"), q, q, lens, table)
    kq, v, gates, states = dev(2, 2, 64), dev(2, 4, 64), dev(2, 4), dev(2, 4, 64, 64)
    two = dev(2, t=torch.int32)
    refused(R.RL_ERR_ARGUMENT, delta.rows, kq, kq, kq, gates, gates, kq, states, two, two)  # value heads
    refused(R.RL_ERR_ARGUMENT, delta.rows, kq, kq.half(), v, gates, gates, v, states, two, two)
    refused(R.RL_ERR_ARGUMENT, delta.rows, kq, kq, v, gates, gates, v, states, two[:1], two[:1])
    refused(R.RL_ERR_CAPACITY, delta.rows, dev(5, 2, 64), dev(5, 2, 64), dev(5, 4, 64), dev(5, 4), dev(5, 4),
            dev(5, 4, 64), states, two, two, dev(3, t=torch.int32))
    refused(R.RL_ERR_ARGUMENT, delta.rows, kq, kq, v, gates, gates, v, states, two, two, scale=float("nan"))
    for f in (lambda: r.apply(dev(4, 1, 64), positions.int()), lambda: r.apply(dev(64, 1, 4).transpose(0, 2), positions),
              lambda: delta.rows(kq, kq, v, gates.half(), gates, v, states, two, two),
              lambda: delta.rows(kq, kq, v, gates, gates, v, states[:, :2], two, two)):
        with pytest.raises(ValueError):
            f()
