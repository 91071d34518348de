"""The token mixers without a GPU: what the library refuses before it selects a
device, the packed tensor layout, and the float64 statements the GPU tests use."""
import ctypes

import numpy as np
import pytest
import torch

import mixer_fixtures as F
import rl_mixers as M
import rl_sampler as R


def test_rotary_specs_that_are_refused():
    h = ctypes.c_void_p()
    good = dict(dims=64, layout=0, scaling=3, original=4096, base=1e4, factor=4.0)

    def code(**kw):
        return M.lib().rl_rotary_create(0, ctypes.byref(M.RotarySpec(**dict(good, **kw))), ctypes.byref(h))

    for kw in (dict(dims=0), dict(dims=63), dict(dims=514), dict(layout=2), dict(scaling=4), dict(base=1.0),
               dict(base=float("inf")), dict(base=float("nan")), dict(factor=0.5), dict(factor=float("nan")),
               dict(original=0), dict(beta_fast=1.0, beta_slow=2.0), dict(beta_slow=-1.0), dict(magnitude=-1.0),
               dict(scaling=2, dims=2)):
        assert code(**kw) == R.RL_ERR_ARGUMENT, kw
    assert M.lib().rl_rotary_create(0, None, ctypes.byref(h)) == R.RL_ERR_ARGUMENT
    assert M.lib().rl_rotary_create(0, ctypes.byref(M.RotarySpec(**good)), None) == R.RL_ERR_ARGUMENT


def test_handles_that_are_refused():
    L, h = M.lib(), ctypes.c_void_p()
    for a in ((0, 16, 1, 64, 1), (1, 0, 1, 64, 1), (1, 16, 0, 64, 1), (1, 16, 1, 0, 1), (1, 16, 1, 24, 1),
              (1, 16, 1, 272, 1), (1, 16, 1, 64, 0), (1, 16, 1, 64, 5)):
        assert L.rl_kv_cache_create(0, *a, ctypes.byref(h)) == R.RL_ERR_ARGUMENT, a
    assert L.rl_kv_cache_create(0, 2 ** 31, 2 ** 31, 1, 64, 1, ctypes.byref(h)) == R.RL_ERR_CAPACITY
    for a in ((0, 4, 2, 64, 9), (1, 0, 1, 64, 9), (1, 3, 2, 64, 9), (1, 4, 0, 64, 9), (1, 4, 2, 40, 9), (1, 4, 2, 64, 0)):
        assert L.rl_attention_create(0, *a, ctypes.byref(h)) == R.RL_ERR_ARGUMENT, a
    assert L.rl_attention_create(0, 1, 4, 2, 64, 2 ** 31, ctypes.byref(h)) == R.RL_ERR_CAPACITY
    for a in ((0, 1, 1, 1, 64, 64), (1, 0, 1, 1, 64, 64), (1, 1, 2, 3, 64, 64), (1, 1, 1, 1, 72, 64), (1, 1, 1, 1, 64, 288)):
        assert L.rl_delta_create(0, *a, ctypes.byref(h)) == R.RL_ERR_ARGUMENT, a
    assert L.rl_rotary_rows(None, None, 1, None, None, 1, 0, None) == R.RL_ERR_ARGUMENT
    assert L.rl_kv_cache_write(None, None, None, None, 1, None, None, None) == R.RL_ERR_ARGUMENT
    assert L.rl_kv_cache_read(None, None, 1, None, None, None) == R.RL_ERR_ARGUMENT
    assert L.rl_attention_rows(None, None, None, None, None, 1, None, None, 1, None, 1, 1.0, 0, 0, 0,
                               None) == R.RL_ERR_ARGUMENT
    assert L.rl_delta_rows(None, None, None, None, None, None, 1, None, 1, None, 1, None, None, None, 1, 1, 1.0, 1.0, 0,
                           None) == R.RL_ERR_ARGUMENT
    assert L.rl_kv_cache_bytes(None) == 0
    for name in ("rl_rotary_destroy", "rl_kv_cache_destroy", "rl_attention_destroy", "rl_delta_destroy"):
        getattr(L, name)(None)  # accepted


def test_packed_tensors_match_the_header():
    x = torch.zeros(3, 5, 8, dtype=torch.bfloat16)[:, 1:4, :6]
    data, rows, heads, n, dim, dtype, _ = M._HEADS.unpack(M._heads(x))
    assert (data, rows, heads, n, dim, dtype) == (x.data_ptr(), 40, 8, 3, 6, 2) and M._HEADS.size == 40
    with pytest.raises(ValueError):
        M._heads(x.transpose(1, 2))
    with pytest.raises(ValueError):
        M._heads(torch.zeros(1, 1, 4, dtype=torch.float64))


def test_the_statements_agree_with_other_forms():
    g = np.random.default_rng(0)
    # Turning by p and then by -p gives the input back; pairs keep their length.
    x = g.standard_normal((3, 2, 12))
    for layout in ("half", "interleaved"):
        f, _ = F.frequencies(8, 1e4)
        y = F.turn(x, [1, 50, 7], f, 1.0, layout)
        assert np.allclose(F.turn(y, [1, 50, 7], f, 1.0, layout, -1.0), x)
        assert np.allclose((y ** 2).sum(-1), (x ** 2).sum(-1)) and np.array_equal(y[..., 8:], x[..., 8:])
    # Attention against torch's softmax.
    q, k, v = g.standard_normal((2, 4, 8)), g.standard_normal((9, 2, 8)), g.standard_normal((9, 2, 8))
    out, lse, _, _ = F.attention(q, k, v, 0.3, 9)
    kk, vv = (torch.from_numpy(t).repeat_interleave(2, 1).movedim(1, 0) for t in (k, v))
    s = 0.3 * torch.from_numpy(q).movedim(1, 0) @ kk.transpose(1, 2)
    s[:, 0, 8:] = -np.inf
    assert np.allclose((torch.softmax(s, -1) @ vv).movedim(0, 1), out) and np.allclose(torch.logsumexp(s, -1).T, lse)
    # The delta rule as one product of the step's matrix: S <- e^g (1 - beta k k') S + beta k v'.
    q, k, v = g.standard_normal((6, 1, 4)), g.standard_normal((6, 1, 4)), g.standard_normal((6, 1, 3))
    gate, beta, s0 = -g.random((6, 1)), g.random((6, 1)), g.standard_normal((1, 4, 3))
    out, state = F.delta(q, k, v, gate, beta, s0, 0.5, -1.0)
    s = s0[0]
    for t in range(6):
        s = np.exp(gate[t, 0]) * (np.eye(4) - beta[t, 0] * np.outer(k[t, 0], k[t, 0])) @ s + beta[t, 0] * np.outer(k[t, 0], v[t, 0])
        assert np.allclose(0.5 * q[t, 0] @ s, out[t, 0])
    assert np.allclose(s, state[0])
    # Codes: the largest value is the largest code, halves go to even.
    assert np.array_equal(F.encode(np.array([[127.0, 0.5, 1.5, -2.5]]), "i8"), [[127.0, 0.0, 2.0, -2.0]])
    assert np.array_equal(F.encode(np.array([[448.0, 1.0625, -3.0]]), "f8"), [[448.0, 1.0, -3.0]])


def test_host_tensors_are_refused():
    # Before any call: a kernel could not read them.
    x, at = torch.zeros(2, 1, 8), torch.zeros(2, dtype=torch.int64)
    r = M.DeviceRotary.__new__(M.DeviceRotary)
    r.h = ctypes.c_void_p()
    with pytest.raises(ValueError, match="device"):
        r.apply(x, at)
