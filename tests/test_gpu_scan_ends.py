"""Steps of the state space scan at the ends of their types' range: the lowest value,
which a mask fills in, gives a step of 0 that leaves the state as it was, in each of the
forms that a call may take."""
import numpy as np
import pytest
import torch

import mixer_fixtures as F
import rl_mixers as M
from test_gpu_conv_scan import i32, scan_case

pytestmark = pytest.mark.gpu

# Rows of one sequence of few channels: token by token, as a whole, in pieces.
FORMS = [3, 40, 300]


@pytest.mark.parametrize("rows", FORMS)
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_steps_at_the_ends_of_the_range(device, dtype, rows):
    # One channel a value, every other token masked by the lowest value: the state is the step itself.
    low, big = torch.finfo(F.TYPES[dtype]).min, torch.finfo(F.TYPES[dtype]).max
    v = torch.tensor([low, big, -2.4e38, 2.4e38, -2.3e38, 2.3e38, float("-inf"), float("inf"), float("nan"), -1e30, 1e30, 1.0])
    v = v.to(F.TYPES[dtype]).to(device)
    channels = v.shape[0]
    for bias in (0.0, 0.5, -1.0):
        scan = M.DeviceScan(rows, 1, -torch.ones(channels, 16), dt_bias=torch.full((channels,), bias))
        dt = torch.full((rows, channels), low, dtype=v.dtype, device=device)
        dt[rows // 2] = v
        x, b = torch.ones_like(dt), torch.ones(rows, 1, 16, dtype=v.dtype, device=device)
        out, states = torch.empty_like(x), torch.zeros(1, channels, 16, device=device)
        scan.rows(x, dt, b, b, out, states, i32([-1], device), i32([0], device), i32([0, rows], device))
        torch.cuda.synchronize()
        want = np.logaddexp(0, F.as64(v) + bias)
        got = F.as64(states[0])
        assert np.array_equal(np.isnan(got[:, 0]), np.isnan(want)), (got[:, 0], want)
        for n in range(16):
            fine = np.isfinite(want)
            assert np.array_equal(got[~fine, n], want[~fine], equal_nan=True)
            assert np.all(np.abs(got[fine, n] - want[fine]) <= want[fine] * 10 * 2.0 ** -24), (got[:, n], want)


@pytest.mark.parametrize("rows", FORMS)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_masked_tokens_leave_the_state(device, dtype, rows):
    g = np.random.default_rng(rows)
    channels, state = 20, 20  # 20 values: lanes that have none
    t, w = scan_case(g, device, [rows], channels, 1, state, dtype, True, 0)
    scan = M.DeviceScan(rows, 1, w["a"], 1, w["skip"], w["dt_bias"])
    first = torch.randn(1, channels, state, device=device)
    slot = i32([0], device)

    def run(tokens, masked):
        # `masked` of the call's tokens hold the lowest value.
        p = {k: v[tokens].contiguous() for k, v in t.items()}
        p["dt"][masked] = torch.finfo(p["dt"].dtype).min
        states, out = first.clone(), torch.empty_like(p["x"])
        scan.rows(p["x"], p["dt"], p["b"], p["c"], out, states, slot, slot, i32([0, len(tokens)], device), z=p["z"],
                  most_rows=rows)
        torch.cuda.synchronize()
        return out, states

    every = torch.arange(rows, device=device)
    out, states = run(every, every)
    assert torch.equal(states, first)  # bit for bit
    y = F.as64(t["z"]) / (1 + np.exp(-F.as64(t["z"])))
    sums = np.einsum("cn,tn->tc", F.as64(first[0]), F.as64(t["c"][:, 0]))
    size = np.einsum("cn,tn->tc", np.abs(F.as64(first[0])), np.abs(F.as64(t["c"][:, 0])))
    skips = F.as64(w["skip"]) * F.as64(t["x"])
    want = (sums + skips) * y
    off = (size + np.abs(skips)) * np.abs(y) * (state + 16 + np.abs(F.as64(t["z"]))) * 2.0 ** -24
    assert np.all(np.abs(F.as64(out) - want) <= off + F.rounding(np.abs(want) + off, dtype))
    # Masked tokens among others: where no piece's bounds move, as if they were not there, bit for bit.
    masked = torch.tensor([0, rows // 2], device=device) if rows < 100 else torch.arange(rows // 2, rows, device=device)
    rest = every[~torch.isin(every, masked)]
    out, states = run(every, masked)
    assert torch.isfinite(out.float()).all() and torch.isfinite(states).all()
    if rows < 100:
        without, after = run(rest, rest[:0])
        assert torch.equal(out[rest], without) and torch.equal(states, after)
