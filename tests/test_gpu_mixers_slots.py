"""Slots that one call of the cache write gives to several rows: what they hold is
promised to nobody, but no other slot is touched, and the next write mends them."""
import numpy as np
import pytest
import torch

import mixer_fixtures as F
import rl_mixers as M
from test_gpu_mixers import randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["bf16", "f16", "i8", "f8"])
def test_a_slot_given_twice_spoils_no_other(device, fmt):
    g = np.random.default_rng(50)
    rows, heads, dim, page = 600, 2, 80, 24
    cache = M.DeviceCache(30, page, heads, dim, fmt)
    k, v = (randn(g, (rows, heads, dim), "f32", device) for _ in range(2))
    slots = g.permutation(30 * page)[:rows]
    shared, alone = slots[::3].copy(), np.ones(rows, bool)
    slots[1::3] = shared  # every third slot is given to two rows
    alone[0::3] = alone[1::3] = False
    dev = torch.from_numpy(slots).to(device)
    cache.write(k, v, dev)
    every = torch.arange(30 * page, device=device)
    ko, vo = (torch.empty(30 * page, heads, dim, device=device) for _ in range(2))
    cache.read(every, ko, vo)
    torch.cuda.synchronize()
    for got, x in ((F.as64(ko), k), (F.as64(vo), v)):
        assert np.array_equal(got[slots[alone]], F.encode(F.as64(x)[alone], fmt))
        untouched = np.setdiff1d(np.arange(30 * page), slots)
        assert not got[untouched].any()
        assert np.isfinite(got).all()
    cache.write(k[::3], v[::3], dev[::3].contiguous())
    cache.read(every, ko, vo)
    torch.cuda.synchronize()
    for got, x in ((F.as64(ko), k), (F.as64(vo), v)):
        assert np.array_equal(got[slots[::3]], F.encode(F.as64(x)[::3], fmt))
        assert np.array_equal(got[slots[alone]], F.encode(F.as64(x)[alone], fmt))
