"""The short convolution and the state space scan on the GPU against float64 statements
of their formulas (step_fixtures.py), whose bounds of the f32 errors are formed before
the comparison."""
import numpy as np
import pytest
import torch

import mixer_fixtures as F
import rl_mixers as M
import rl_sampler as R
import step_fixtures as S

pytestmark = pytest.mark.gpu


def randn(g, shape, dtype, device, sigma=1.0):
    return torch.from_numpy((g.standard_normal(shape) * sigma).astype(np.float32)).to(device).to(F.TYPES[dtype])


def padded(x, more):
    """A copy of x [rows][..] whose rows lie `more` values further apart, NaN between."""
    rows, rest = x.shape[0], x.shape[1:]
    size = int(np.prod(rest))
    buf = torch.full((rows + 1, size + more), float("nan"), dtype=x.dtype, device=x.device)
    y = buf[:rows, :size].view(rows, *rest) if more == 0 else torch.as_strided(
        buf, x.shape, (size + more,) + tuple(x[0].stride() if rows else torch.empty(rest).stride()))
    y.copy_(x)
    return y


def i32(x, device):
    return torch.tensor(np.ascontiguousarray(x), dtype=torch.int32, device=device)


def slots_for(g, n, how):
    """(slots in, slots out, slots in all): in place, apart, or with none and some past the pool."""
    order = g.permutation(2 * n + 2)
    if how == "place":
        return order[:n], order[:n], 2 * n + 2
    into, to = order[:n].copy(), order[n:2 * n].copy()
    if how == "odd":
        into[0], to[-1] = -1, -3
        if n > 2:
            into[1], to[1] = 2 * n + 2, 2 ** 31 - 1
    return into, to, 2 * n + 2


CONV = [
    # lens, channels, width, type, activation, slots, padding of x and of out
    ([1], 8, 4, "bf16", "silu", "place", 0, 0),
    ([1] * 70, 1024, 4, "bf16", "silu", "place", 0, 0),
    ([9, 0, 1, 2, 3, 4, 31, 32, 33, 64], 520, 4, "f16", "silu", "odd", 8, 16),
    ([300, 17], 77, 3, "f32", "none", "apart", 0, 3),
    ([8, 7, 9, 16], 12, 8, "f32", "silu", "place", 4, 0),
    ([5, 40, 1], 129, 2, "bf16", "none", "odd", 1, 0),
    ([11, 0, 100], 64, 5, "f16", "none", "apart", 0, 0),
    ([70], 33, 6, "f32", "silu", "place", 0, 1),
    ([2, 6, 7], 16, 7, "bf16", "silu", "place", 0, 0),
    ([2100, 1, 700], 2048, 4, "bf16", "silu", "place", 0, 0),   # runs of 32 rows
    ([4000, 1, 0, 99], 2051, 8, "f16", "silu", "odd", 0, 1),    # the same without vectors
]


@pytest.mark.parametrize("case", range(len(CONV)))
def test_conv(device, case):
    lens, channels, width, dtype, act, how, pad_x, pad_out = CONV[case]
    g = np.random.default_rng(100 + case)
    rows, n = sum(lens), len(lens)
    x = padded(randn(g, (rows, channels), dtype, device), pad_x)
    weight, bias = (torch.from_numpy(g.standard_normal(s).astype(np.float32)) for s in ((channels, width), (channels,)))
    into, to, slots = slots_for(g, n, how)
    states = randn(g, (slots, width - 1, channels), dtype, device)
    before = states.clone()
    out = padded(torch.full((rows, channels), 7.0, dtype=x.dtype, device=device), pad_out)
    conv = M.DeviceConv(weight, None if case % 3 == 0 else bias, act)
    single = all(c == 1 for c in lens)
    starts = i32([0] + list(np.cumsum(lens)), device)
    print("conv", CONV[case], flush=True)
    conv.rows(x, out, states, i32(into, device), i32(to, device), None if single else starts)
    torch.cuda.synchronize()
    untouched, at = np.ones(slots, bool), 0
    for i, c in enumerate(lens):
        first = F.as64(before)[into[i]] if 0 <= into[i] < slots else np.full((width - 1, channels), np.nan if into[i] >= 0 else 0.0)
        want, after, off = S.conv(F.as64(x[at:at + c]), first, F.as64(weight), F.as64(bias) * (case % 3 != 0), act)
        got = F.as64(out[at:at + c])
        fine = ~np.isnan(want)
        assert np.array_equal(np.isnan(got), ~fine)
        assert np.all((np.abs(got - want) <= off + F.rounding(np.abs(want) + off, dtype))[fine]), (i, np.abs(got - want)[fine].max())
        if 0 <= to[i] < slots:
            untouched[to[i]] = False
            assert np.array_equal(F.as64(states[int(to[i])]), after, equal_nan=True), i
        at += c
    assert torch.equal(states[torch.from_numpy(untouched)], before[torch.from_numpy(untouched)])
    if pad_out:
        edge = torch.as_strided(out, (rows, pad_out), (out.stride(0), 1), out.storage_offset() + channels)
        assert torch.isnan(edge).all()
    # Token by token, from the same states: the same bits.
    if rows <= 500:
        states.copy_(before)
        again = torch.empty(rows, channels, dtype=x.dtype, device=device)
        for t in range(max(lens)):
            here = [i for i, c in enumerate(lens) if c > t]
            at = torch.tensor([sum(lens[:i]) + t for i in here], device=device)
            now, y = x[at].contiguous(), torch.empty(len(here), channels, dtype=x.dtype, device=device)
            conv.rows(now, y, states, i32([into[i] if t == 0 else to[i] for i in here], device), i32([to[i] for i in here], device))
            again[at] = y
        kept = [i for i, c in enumerate(lens) if 0 <= to[i] < slots]
        torch.cuda.synchronize()
        for i in kept:
            a, b = sum(lens[:i]), sum(lens[:i + 1])
            assert torch.equal(torch.nan_to_num(again[a:b], 9.0), torch.nan_to_num(out[a:b], 9.0)), i
    conv.close()


def test_conv_values_at_the_ends_of_the_range(device):
    # silu of large and tiny sums, of infinities and NaN: y / (1 + e^-y) itself.
    y = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 100.0, -100.0, -80.0, 3e38, -3e38, float("inf"), float("nan")], device=device)
    for dtype in (torch.float32, torch.bfloat16):
        x = y.to(dtype)[:, None].expand(-1, 8).contiguous()
        conv = M.DeviceConv(torch.tensor([[0.0, 1.0]]).expand(8, 2))
        out, states = torch.empty_like(x), torch.zeros(1, 1, 8, dtype=dtype, device=device)
        none = i32([-1] * len(y), device)
        conv.rows(x, out, states, none, none)
        want = S.silu(F.as64(x))
        got = F.as64(out)
        assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.isinf(got), np.isinf(want))
        fine = np.isfinite(want)
        with np.errstate(invalid="ignore"):
            off = S.silu_error(F.as64(x), 0) + F.rounding(np.abs(want), "f32" if dtype == torch.float32 else "bf16") + 2.0 ** -126
        assert np.all(np.abs(got[fine] - want[fine]) <= off[fine])


SCAN = [
    # lens, channels, groups, state, type, gated, slots, softplus, padding
    ([1], 8, 1, 16, "bf16", True, "place", True, 0),
    ([1] * 40, 200, 1, 16, "bf16", True, "place", True, 0),
    ([9, 0, 3, 16], 48, 4, 8, "f16", True, "odd", True, 8),
    ([5, 1, 2], 6, 3, 4, "f32", False, "apart", True, 0),
    ([17, 2], 20, 2, 12, "f32", True, "place", True, 4),
    ([130, 0, 64, 65], 96, 1, 16, "bf16", True, "odd", True, 0),
    ([300, 63], 40, 2, 64, "f32", False, "place", True, 0),
    ([100, 31], 7, 1, 256, "f16", True, "apart", True, 1),
    ([90], 130, 1, 20, "f32", True, "place", False, 0),
    ([257, 1, 640], 24, 4, 32, "bf16", False, "place", True, 0),
    ([200, 70], 10, 5, 128, "bf16", True, "odd", True, 16),
]


def scan_case(g, device, lens, channels, groups, state, dtype, gated, pad):
    rows = sum(lens)
    t = {"x": randn(g, (rows, channels), dtype, device), "dt": randn(g, (rows, channels), dtype, device, 1.5),
         "b": randn(g, (rows, groups, state), dtype, device), "c": randn(g, (rows, groups, state), dtype, device),
         "z": randn(g, (rows, channels), dtype, device) if gated else None}
    t = {k: None if v is None else padded(v, pad) for k, v in t.items()}
    w = {"a": -torch.from_numpy(np.exp(g.standard_normal((channels, state))).astype(np.float32)),
         "skip": torch.from_numpy(g.standard_normal(channels).astype(np.float32)),
         "dt_bias": torch.from_numpy((g.standard_normal(channels) - 2).astype(np.float32))}
    return t, w


@pytest.mark.parametrize("most", ["exact", "none", "one"])
@pytest.mark.parametrize("case", range(len(SCAN)))
def test_scan(device, case, most):
    lens, channels, groups, state, dtype, gated, how, soft, pad = SCAN[case]
    g = np.random.default_rng(200 + case)
    rows, n = sum(lens), len(lens)
    t, w = scan_case(g, device, lens, channels, groups, state, dtype, gated, pad)
    into, to, slots = slots_for(g, n, how)
    states = randn(g, (slots, channels, state), "f32", device)
    before = states.clone()
    out = padded(torch.full((rows, channels), 7.0, dtype=F.TYPES[dtype], device=device), pad)
    if not soft:
        t["dt"] = padded(t["dt"].abs() * 0.1, pad)
        w["dt_bias"] = w["dt_bias"].abs() * 0.1
    scan = M.DeviceScan(rows, n, w["a"], groups, w["skip"], w["dt_bias"])
    hint = {"exact": max(lens), "none": 0, "one": 1}[most]
    starts = i32([0] + list(np.cumsum(lens)), device)
    print("scan", SCAN[case], most, flush=True)
    call = lambda: scan.rows(t["x"], t["dt"], t["b"], t["c"], out, states, i32(into, device), i32(to, device),  # noqa: E731
                             starts, z=t["z"], softplus=soft, most_rows=hint)
    call()
    torch.cuda.synchronize()
    untouched, at = np.ones(slots, bool), 0
    for i, c in enumerate(lens):
        first = F.as64(before)[into[i]] if 0 <= into[i] < slots else np.full((channels, state), np.nan if into[i] >= 0 else 0.0)
        part = {k: None if v is None else F.as64(v[at:at + c]) for k, v in t.items()}
        want, after, off, err = S.scan(**part, a=F.as64(w["a"]), skip=F.as64(w["skip"]), bias=F.as64(w["dt_bias"]),
                                       state=first, softplus=soft, pieces=True)
        got, fine = F.as64(out[at:at + c]), ~np.isnan(want)
        assert np.array_equal(np.isnan(got), ~fine)
        assert np.all((np.abs(got - want) <= off + F.rounding(np.abs(want) + off, dtype))[fine]), (
            i, np.nanmax(np.abs(got - want) / (off + F.rounding(np.abs(want) + off, dtype))))
        if 0 <= to[i] < slots:
            untouched[to[i]] = False
            h = F.as64(states[int(to[i])])
            assert np.array_equal(np.isnan(h), np.isnan(after))
            assert np.all((np.abs(h - after) <= err + 2.0 ** -126)[~np.isnan(after)]), (i, np.nanmax(np.abs(h - after) / (err + 1e-30)))
        at += c
    assert torch.equal(states[torch.from_numpy(untouched)], before[torch.from_numpy(untouched)])
    if pad:
        edge = torch.as_strided(out, (rows, pad), (out.stride(0), 1), out.storage_offset() + channels)
        assert torch.isnan(edge).all()
    # The same bits again, also with outputs in place of x.
    first, after = out.clone(), states.clone()
    states.copy_(before)
    out = t["x"] = padded(t["x"], pad)
    call()
    torch.cuda.synchronize()
    assert torch.equal(torch.nan_to_num(out, 9.0), torch.nan_to_num(first, 9.0))
    assert torch.equal(torch.nan_to_num(states, 9.0), torch.nan_to_num(after, 9.0))
    scan.close()


def test_scan_steps_of_any_size(device):
    # dt from where e^dt is lost beside 1 to where it is the step itself, and past f32's exponential.
    v = torch.tensor([-120.0, -87.0, -40.0, -17.0, -5.0, -1e-3, 0.0, 1e-3, 5.0, 17.0, 90.0, 1000.0], device=device)
    channels = v.shape[0]
    scan = M.DeviceScan(1, 1, torch.zeros(channels, 4))
    one = torch.ones(1, channels, device=device)
    states, out = torch.zeros(1, channels, 4, device=device), torch.empty(1, channels, device=device)
    b = torch.ones(1, 1, 4, device=device)
    scan.rows(one, v[None].contiguous(), b, b, out, states, i32([-1], device), i32([0], device))
    want = np.logaddexp(0, F.as64(v))
    got = F.as64(states[0])[:, 0]
    assert np.all(np.abs(got - want) <= want * 10 * S.E + 2.0 ** -126), (got, want)


@pytest.mark.parametrize("rows,channels", [(1100, 4100), (1999, 2000), (640, 300)])
def test_scan_of_one_long_sequence_and_short_ones(device, rows, channels):
    # As many pieces as the workspace holds: the handle is made for these rows and no more.
    g = np.random.default_rng(rows + channels)
    lens = [rows, 0, 3, 1, 17]
    t, w = scan_case(g, device, lens, channels, 1, 4, "bf16", False, 0)
    n = len(lens)
    states = randn(g, (n, channels, 4), "f32", device)
    before = states.clone()
    scan = M.DeviceScan(sum(lens), n, w["a"], 1, w["skip"], w["dt_bias"])
    out = torch.empty_like(t["x"])
    slots, starts = i32(range(n), device), i32([0] + list(np.cumsum(lens)), device)
    scan.rows(t["x"], t["dt"], t["b"], t["c"], out, states, slots, slots, starts)
    torch.cuda.synchronize()
    at = 0
    for i, c in enumerate(lens):
        part = {k: None if v is None else F.as64(v[at:at + c]) for k, v in t.items()}
        want, after, off, err = S.scan(**part, a=F.as64(w["a"]), skip=F.as64(w["skip"]), bias=F.as64(w["dt_bias"]),
                                       state=F.as64(before[i]), pieces=True)
        assert np.all(np.abs(F.as64(out[at:at + c]) - want) <= off + F.rounding(np.abs(want) + off, "bf16")), i
        assert np.all(np.abs(F.as64(states[i]) - after) <= err + 2.0 ** -126), i
        at += c


@pytest.mark.parametrize("what", ["conv", "scan", "steps"])
def test_captured_calls_and_another_stream(device, what):
    g = np.random.default_rng(7)
    lens = [200, 3, 90] if what != "steps" else [1, 9, 2]
    rows, n = sum(lens), len(lens)
    starts, slots = i32([0] + list(np.cumsum(lens)), device), i32(range(n), device)
    t, w = scan_case(g, device, lens, 64, 2, 16, "bf16", True, 0)
    if what == "conv":
        h = M.DeviceConv(torch.from_numpy(g.standard_normal((64, 4)).astype(np.float32)))
        states = randn(g, (n, 3, 64), "bf16", device)
        out = torch.empty_like(t["x"])
        call = lambda **kw: h.rows(t["x"], out, states, slots, slots, starts, **kw)  # noqa: E731
    else:
        h = M.DeviceScan(rows, n, w["a"], 2, w["skip"], w["dt_bias"])
        states = randn(g, (n, 64, 16), "f32", device)
        out = torch.empty_like(t["x"])
        call = lambda **kw: h.rows(t["x"], t["dt"], t["b"], t["c"], out, states, slots, slots, starts, z=t["z"], **kw)  # noqa: E731
    first, results = states.clone(), []
    for _ in range(4):  # four in a row, each from the states that the one before left
        call()
        results.append((out.clone(), states.clone()))
    torch.cuda.synchronize()
    states.copy_(first)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    call(stream=other.cuda_stream)
    other.synchronize()
    assert torch.equal(out, results[0][0]) and torch.equal(states, results[0][1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    torch.cuda.synchronize()
    states.copy_(first)
    for want_out, want_states in results:
        out.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want_out) and torch.equal(states, want_states)
        assert float((out.float() * 0).sum()) == 0.0  # the program's own work between the replays


@pytest.mark.parametrize("most", [1, 40, 700])  # token by token, whole sequences, pieces
def test_rows_behind_the_last_sequence_stay(device, most):
    g = np.random.default_rng(most)
    lens, rows, channels = [most, 1, most], 2 * most + 20, 96
    at = 2 * most + 1
    starts, slots = i32([0, most, most + 1, at], device), i32([0, 1, 2], device)
    x, dt = (randn(g, (rows, channels), "f32", device) for _ in range(2))
    b, c = (randn(g, (rows, 2, 16), "f32", device) for _ in range(2))
    conv = M.DeviceConv(torch.ones(channels, 4))
    scan = M.DeviceScan(rows, 3, -torch.ones(channels, 16), groups=2)
    for call, shape in ((lambda y, p: conv.rows(x, y, p, slots, slots, starts), (4, 3, channels)),
                        (lambda y, p: scan.rows(x, dt, b, c, y, p, slots, slots, starts, most_rows=most), (4, channels, 16))):
        y, states = torch.full_like(x, 7.0), torch.full(shape, 2.0, device=device)
        call(y, states)
        torch.cuda.synchronize()
        assert (y[at:] == 7.0).all() and (y[:at] != 7.0).any(1).all()
        assert (states[3] == 2.0).all() and all((states[i] != 2.0).any() for i in range(3))


def test_refusals(device):
    conv = M.DeviceConv(torch.zeros(8, 4))
    scan = M.DeviceScan(4, 2, torch.zeros(8, 16), groups=2)
    x = torch.zeros(4, 8, device=device)
    s2, starts = i32([0, 1], device), i32([0, 2, 4], device)
    states, pool = torch.zeros(2, 3, 8, device=device), torch.zeros(2, 8, 16, device=device)
    b = torch.zeros(4, 2, 16, device=device)

    def refused(code, f, *a, **kw):
        with pytest.raises(R.SamplerError) as e:
            f(*a, **kw)
        assert e.value.code == code

    refused(R.RL_ERR_ARGUMENT, conv.rows, x, x, states, s2, s2, starts)          # in place
    refused(R.RL_ERR_ARGUMENT, conv.rows, x, torch.zeros_like(x), states, s2, s2)  # two sequences of four rows
    refused(R.RL_ERR_ARGUMENT, conv.rows, x[:, :4], torch.zeros(4, 4, device=device), states, s2, s2, starts)
    refused(R.RL_ERR_ARGUMENT, conv.rows, x, torch.zeros(4, 8, device=device, dtype=torch.bfloat16), states, s2, s2, starts)
    refused(R.RL_ERR_ARGUMENT, conv.rows, x, torch.zeros(8, device=device).expand(4, 8), states, s2, s2, starts)
    y = torch.zeros_like(x)
    refused(R.RL_ERR_ARGUMENT, scan.rows, x, x.bfloat16(), b, b, y, pool, s2, s2, starts)
    refused(R.RL_ERR_ARGUMENT, scan.rows, x, x, b[:, :1], b, y, pool, s2, s2, starts)
    refused(R.RL_ERR_ARGUMENT, scan.rows, x, x, b, b[..., :8], y, pool, s2, s2, starts)
    refused(R.RL_ERR_ARGUMENT, scan.rows, x, x, b, b, y, pool, s2, s2)
    over = torch.zeros(8, 8, device=device)
    refused(R.RL_ERR_ARGUMENT, scan.rows, over[::2], x, b, b, over[:4], pool, s2, s2, starts)  # in place, but not row by row
    refused(R.RL_ERR_ARGUMENT, scan.rows, x, over[::2], b, b, over[:4], pool, s2, s2, starts)
    refused(R.RL_ERR_ARGUMENT, scan.rows, x, x, b, b, over[:4], pool, s2, s2, starts, z=over[::2])
    refused(R.RL_ERR_ARGUMENT, scan.rows, x, x, b, b, b.view(-1, 8)[:4], pool, s2, s2, starts)
    refused(R.RL_ERR_CAPACITY, scan.rows, *(torch.cat([t, t]) for t in (x, x, b, b, y)), pool, s2, s2, starts)
    refused(R.RL_ERR_CAPACITY, scan.rows, x, x, b, b, y, pool, i32([0, 1, -1], device), i32([0, 1, -1], device), i32([0, 1, 2, 4], device))
    # Nothing to do is no error, and a call without rows passes states on.
    none = i32([], device)
    conv.rows(x[:0], y[:0], states, none, none)
    scan.rows(x[:0], x[:0], b[:0], b[:0], y[:0], pool, none, none)
    states[0], pool[0] = 5, 6
    a, c, zero = i32([0], device), i32([1], device), i32([0, 0], device)
    conv.rows(x[:0], y[:0], states, a, c, zero)
    scan.rows(x[:0], x[:0], b[:0], b[:0], y[:0], pool, a, c, zero)
    torch.cuda.synchronize()
    assert (states[1] == 5).all() and (pool[1] == 6).all()
