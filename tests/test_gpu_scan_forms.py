"""The state space scan of prompts in each of its forms against a float64 statement of
its formula: whole sequences and pieces of several tiles of staged tokens and a
remainder, for every number of lanes that hold a channel. Bounds are those of the form:
what joins pieces is counted once at each of their borders, with the tokens of a piece."""
import numpy as np
import pytest
import torch

import mixer_fixtures as F
import rl_mixers as M
import step_fixtures as S
from test_gpu_conv_scan import i32, padded, scan_case

pytestmark = pytest.mark.gpu
E = S.E


def scan(x, dt, b, c, z, a, skip, bias, state, piece):
    """x, dt, z [rows][channels], b, c [rows][channels][n] of one sequence; `piece`
    tokens of a piece, or None. Outputs, the state after, and bounds of their f32 errors:
    of each step the decay's exponent and exponential, the products and the sum, as
    step_fixtures.scan counts them."""
    h, size, err = state.copy(), np.abs(state), np.zeros_like(state)
    out, off = np.zeros_like(x), np.zeros_like(x)
    passed, first = np.zeros(x.shape[1]), size  # of the piece: the sum of its steps, and the sizes it began with
    for t in range(len(x)):
        if piece and t and t % piece == 0:
            # The piece's first state goes by the exponential of the sum of its steps: `piece` roundings of the sum, two of
            # the exponent, the exponential's own, a product and a sum.
            e = np.exp(passed[:, None] * a)
            err = err + e * first * (np.abs(a) * passed[:, None] * (piece + 2) + 4) * E + size * E
            passed, first = np.zeros_like(passed), size
        v = dt[t] + bias
        s = np.logaddexp(0, v)
        passed = passed + s
        ds = np.abs(s) * 10 * E + np.abs(v) * E * np.exp(np.minimum(v, 0))  # the slope of softplus is at most e^v
        e, drive = np.exp(s[:, None] * a), (s * x[t])[:, None] * b[t]
        de = e * (np.abs(a) * (ds[:, None] + np.abs(s)[:, None] * 2 * E) + 4 * E)
        h = e * h + drive
        err = e * err + de * size + np.abs(drive) * 4 * E + (ds * np.abs(x[t]))[:, None] * np.abs(b[t])
        size = e * size + np.abs(drive)
        err = err + size * E
        y = (h * c[t]).sum(-1) + skip * x[t]
        o = (err * np.abs(c[t])).sum(-1) + ((size * np.abs(c[t])).sum(-1) + np.abs(skip * x[t])) * (a.shape[1] + 2) * E
        if z is not None:
            g = S.silu(z[t])
            o = o * np.abs(g) + np.abs(y) * S.silu_error(z[t], 0) + np.abs(y * g) * E
            y = y * g
        out[t], off[t] = y, o
    return out, h, off, err


FORMS = [
    # lens, channels, groups, state, type, gated, tokens of a piece (None: whole sequences)
    ([33, 40, 36, 38] * 4, 5120, 1, 16, "bf16", True, None),
    ([130, 0, 128, 129] * 5, 5120, 4, 16, "f32", True, None),
    ([50] * 20, 2600, 1, 32, "f32", True, None),
    ([47, 33] * 12, 2100, 3, 64, "f32", True, None),
    ([45, 1, 49] * 8, 1600, 1, 40, "f16", False, None),
    ([49, 34] * 6, 1040, 2, 8, "f32", True, None),
    ([37] * 9, 900, 1, 128, "bf16", True, None),
    ([41, 38] * 4, 520, 4, 252, "f32", True, None),
    ([3000, 5, 90], 40, 1, 16, "f32", True, 47),
    ([3000, 64, 0, 700], 36, 2, 32, "f32", True, 47),
    ([2600], 40, 4, 64, "f32", True, 41),
    ([3333, 1], 20, 1, 52, "bf16", True, 53),
    ([3200, 17], 24, 1, 4, "f16", False, 50),
    ([2900], 12, 1, 256, "f32", True, 46),
    ([1300], 10240, 1, 16, "bf16", True, 51),
    ([700, 400, 350], 6000, 2, 32, "f32", True, 68),
]


@pytest.mark.parametrize("case", range(len(FORMS)))
def test_forms(device, case):
    lens, channels, groups, state, dtype, gated, piece = FORMS[case]
    g = np.random.default_rng(500 + case)
    rows, n = sum(lens), len(lens)
    t, w = scan_case(g, device, lens, channels, groups, state, dtype, gated, 8 if case % 2 else 0)
    states = torch.from_numpy(g.standard_normal((n, channels, state)).astype(np.float32)).to(device)
    before = states.clone()
    out = padded(torch.full((rows, channels), 7.0, dtype=F.TYPES[dtype], device=device), 8 if case % 2 else 0)
    handle = M.DeviceScan(rows, n, w["a"], groups, w["skip"], w["dt_bias"])
    slots, starts = i32(range(n), device), i32([0] + list(np.cumsum(lens)), device)
    print("scan form", FORMS[case], flush=True)
    handle.rows(t["x"], t["dt"], t["b"], t["c"], out, states, slots, slots, starts, z=t["z"], most_rows=max(lens))
    torch.cuda.synchronize()
    # Channels are alike: the first and last of each workgroup's and group's share, and some between.
    some = sorted({0, channels - 1, channels // 2, channels // groups - 1, *g.integers(0, channels, 11)}
                  | {i for i in (15, 16, 63, 64, 127, 128, 255, 256) if i < channels})
    of = np.array(some) // (channels // groups)
    a, skip, bias = (F.as64(w[k])[some] for k in ("a", "skip", "dt_bias"))
    at = 0
    for i, m in enumerate(lens):
        x, dt, z = (None if t[k] is None else F.as64(t[k][at:at + m][:, some]) for k in ("x", "dt", "z"))
        b, c = (F.as64(t[k][at:at + m][:, of]) for k in ("b", "c"))
        want, after, off, err = scan(x, dt, b, c, z, a, skip, bias, F.as64(before[i, some]), piece)
        got = F.as64(out[at:at + m][:, some])
        slack = off + F.rounding(np.abs(want) + off, dtype)
        assert np.all(np.abs(got - want) <= slack), (i, np.max(np.abs(got - want) / slack))
        h = F.as64(states[i, some])
        assert np.all(np.abs(h - after) <= err + 2.0 ** -126), (i, np.max(np.abs(h - after) / (err + 1e-30)))
        at += m
    assert torch.isfinite(out.float()).all() and torch.isfinite(states).all()
    if t["x"].stride(0) > channels:
        assert torch.isnan(torch.as_strided(out, (rows, 8), (out.stride(0), 1), out.storage_offset() + channels)).all()
    handle.close()
