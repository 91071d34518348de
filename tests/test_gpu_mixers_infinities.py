"""Infinities that attention has in sight: what they may reach, and what not."""
import numpy as np
import pytest
import torch

import mixer_fixtures as F
import rl_mixers as M
from test_gpu_mixers import attend_check, randn

pytestmark = pytest.mark.gpu


def one_row(device, fmt, dtype, n, spoil):
    g = np.random.default_rng(60)
    cache = M.DeviceCache(8, 32, 1, 48, fmt)
    k, v = (randn(g, (n, 1, 48), fmt, device) for _ in range(2))
    q = randn(g, (1, 4, 48), dtype, device)
    spoil(q, k, v)
    cache.write(k, v, torch.arange(n, device=device))
    out, lse = torch.empty_like(q), torch.empty(1, 4, device=device)
    att = M.DeviceAttention(1, 4, 1, 48, 256)
    att.rows(cache, q, out, torch.tensor([n], dtype=torch.int32, device=device),
             torch.arange(8, dtype=torch.int32, device=device)[None], lse=lse)
    torch.cuda.synchronize()
    return q, out, lse, k, v


@pytest.mark.parametrize("fmt,dtype", [("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32")])
@pytest.mark.parametrize("n,at", [(1, 0), (40, 39), (40, 3), (250, 100)])
def test_an_infinite_value_stays_in_its_column(device, fmt, dtype, n, at):
    def spoil(q, k, v):
        v[at, 0, 7] = float("inf")
    q, out, lse, k, v = one_row(device, fmt, dtype, n, spoil)
    got = F.as64(out)
    assert not np.isfinite(got[..., 7]).any()  # an infinity, or NaN
    out[..., 7] = 0  # every other column as without it
    values = F.as64(v)
    values[..., 7] = 0
    attend_check(q, out, lse, [n], [1], [(F.as64(k), values)], fmt, dtype, 0, 48)


@pytest.mark.parametrize("fmt", ["bf16", "f16"])
def test_a_score_of_minus_infinity_has_no_weight(device, fmt):
    # 16-bit queries: an infinite key that gives minus infinity takes no part.
    def spoil(q, k, v):
        q[..., 3] = q[..., 3].abs() + 0.1
        k[5, 0, 3] = float("-inf")
    q, out, lse, k, v = one_row(device, fmt, fmt, 40, spoil)
    rest = [i for i in range(40) if i != 5]
    attend_check(q, out, lse, [39], [1], [(F.as64(k)[rest], F.as64(v)[rest])], fmt, fmt, 0, 48)
