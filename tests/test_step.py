"""The convolution, the scan, shared prefixes and the verification of drafts without a
GPU: what the library and its bindings refuse, and the float64 statements that the GPU
tests use."""
import ctypes

import numpy as np
import pytest
import torch

import rl_drafts as D
import rl_mixers as M
import rl_sampler as R
import step_fixtures as S
from test_mixers_devices import On1, Reached, handle, no_library, tensor  # noqa: F401


def test_handles_that_are_refused():
    L, h = M.lib(), ctypes.c_void_p()
    D.lib()
    w = (ctypes.c_float * 64)()
    for a in ((0, 4, w, None, 0), (4, 1, w, None, 0), (4, 9, w, None, 0), (4, 4, None, None, 0), (4, 4, w, None, 2)):
        assert L.rl_conv_create(0, *a, ctypes.byref(h)) == R.RL_ERR_ARGUMENT, a
    assert L.rl_conv_create(0, 2 ** 20 + 1, 2, w, None, 0, ctypes.byref(h)) == R.RL_ERR_CAPACITY
    assert L.rl_conv_create(0, 4, 4, w, None, 0, None) == R.RL_ERR_ARGUMENT
    for a in ((0, 1, 4, 1, 4, w), (1, 0, 4, 1, 4, w), (1, 1, 0, 1, 4, w), (1, 1, 4, 0, 4, w), (1, 1, 4, 3, 4, w),
              (1, 1, 4, 1, 0, w), (1, 1, 4, 1, 6, w), (1, 1, 4, 1, 260, w), (1, 1, 4, 1, 4, None)):
        assert L.rl_scan_create(0, *a, None, None, ctypes.byref(h)) == R.RL_ERR_ARGUMENT, a
    for a in ((1, 1, 2 ** 20 + 1, 1, 4, w), (2 ** 23 + 1, 1, 4, 1, 4, w), (1, 2 ** 23 + 1, 4, 1, 4, w)):
        assert L.rl_scan_create(0, *a, None, None, ctypes.byref(h)) == R.RL_ERR_CAPACITY, a
    for a in ((0, 4), (1, 0)):
        assert L.rl_drafts_create(0, *a, ctypes.byref(h)) == R.RL_ERR_ARGUMENT, a
    for a in ((2 ** 16 + 1, 4), (1, 2 ** 21 + 1)):
        assert L.rl_drafts_create(0, *a, ctypes.byref(h)) == R.RL_ERR_CAPACITY, a
    assert L.rl_conv_rows(None, None, None, None, 0, None, None, None, 1, 1, None) == R.RL_ERR_ARGUMENT
    assert L.rl_scan_rows(None, None, None, None, None, None, None, None, 0, None, None, None, 1, 1, 1, 0,
                          None) == R.RL_ERR_ARGUMENT
    assert L.rl_attention_shared(None, None, None, None, None, 1, None, None, 1, None, 1, None, None, 1, None, 1, 1.0, 0, 0,
                                 0, None) == R.RL_ERR_ARGUMENT
    assert L.rl_drafts_verify(None, None, None, None, None, None, None, 1, 1, None, None, None) == R.RL_ERR_ARGUMENT
    for name in ("rl_conv_destroy", "rl_scan_destroy", "rl_drafts_destroy"):
        getattr(L, name)(None)  # accepted


def calls():
    """(a call of each method, its tensors by name)."""
    i32 = torch.int32
    conv = handle(M.DeviceConv, state=(3, 16))
    scan = handle(M.DeviceScan, state=(16, 8))
    attention = handle(M.DeviceAttention, q_heads=2, scale=1.0)
    cache, drafts = handle(M.DeviceCache), handle(D.DeviceDrafts, vocab=9)
    x = lambda: tensor(3, 16)  # noqa: E731
    slots = lambda: tensor(2, t=i32)  # noqa: E731
    heads = lambda: tensor(3, 2, 16)  # noqa: E731
    return {
        "conv": (conv.rows, dict(x=x(), out=x(), states=tensor(4, 3, 16), slots_in=slots(), slots_out=slots(),
                                 starts=tensor(3, t=i32))),
        "scan": (scan.rows, dict(x=x(), dt=x(), b=tensor(3, 1, 8), c=tensor(3, 1, 8), out=x(), z=x(),
                                 states=tensor(4, 16, 8), slots_in=slots(), slots_out=slots(), starts=tensor(3, t=i32))),
        "shared": (lambda **kw: attention.shared(cache, **kw),
                   dict(q=heads(), out=heads(), lens=slots(), pages=tensor(2, 4, t=i32), groups=tensor(2, t=i32),
                        prefix_lens=tensor(1, t=i32), prefix_pages=tensor(1, 3, t=i32), starts=tensor(3, t=i32),
                        lse=tensor(3, 2))),
        "dense": (drafts.verify, dict(target=tensor(5, 9), drafted=tensor(3, t=i32), starts=tensor(3, t=i32),
                                      uniforms=tensor(3), draws=tensor(2), accepted=tensor(2, t=i32),
                                      tokens=tensor(5, t=i32), draft=tensor(3, 9))),
        "lists": (drafts.verify, dict(target=tensor(5, 4), drafted=tensor(3, t=i32), starts=tensor(3, t=i32),
                                      uniforms=tensor(3), draws=tensor(2), accepted=tensor(2, t=i32),
                                      tokens=tensor(5, t=i32), draft=tensor(3, 4), target_ids=tensor(5, 4, t=i32),
                                      target_kept=tensor(5, t=i32), draft_ids=tensor(3, 4, t=i32),
                                      draft_kept=tensor(3, t=i32))),
    }


@pytest.fixture
def no_drafts(monkeypatch, no_library):  # noqa: F811
    monkeypatch.setattr(D, "lib", M.lib)


@pytest.mark.parametrize("call", list(calls()))
def test_every_tensor_has_to_be_on_the_handles_device(no_drafts, call):
    f, tensors = calls()[call]
    with pytest.raises(Reached):
        f(**tensors)
    for name, x in tensors.items():
        for other in (torch.zeros(x.shape, dtype=x.dtype), torch.zeros(x.shape, dtype=x.dtype).as_subclass(On1)):
            with pytest.raises(ValueError, match="device"):
                f(**dict(tensors, **{name: other}))
                pytest.fail("%s passed" % name)


@pytest.mark.parametrize("call,name,other", [
    ("conv", "out", lambda: tensor(3, 15)), ("conv", "states", lambda: tensor(4, 2, 16)),
    ("conv", "states", lambda: tensor(4, 3, 16, t=torch.bfloat16)), ("conv", "x", lambda: tensor(16, 3).t()),
    ("conv", "starts", lambda: tensor(3, t=torch.int64)), ("conv", "slots_out", lambda: tensor(1, t=torch.int32)),
    ("scan", "dt", lambda: tensor(2, 16)), ("scan", "z", lambda: tensor(4, 16)), ("scan", "b", lambda: tensor(2, 1, 8)),
    ("scan", "states", lambda: tensor(4, 8, 16)), ("scan", "c", lambda: tensor(3, 8, 1).transpose(1, 2)[:, :, ::2]),
    ("shared", "groups", lambda: tensor(1, t=torch.int32)), ("shared", "prefix_lens", lambda: tensor(0, t=torch.int32)),
    ("dense", "target", lambda: tensor(4, 9)), ("dense", "target", lambda: tensor(5, 8)),
    ("dense", "draft", lambda: tensor(3, 10)), ("dense", "tokens", lambda: tensor(4, t=torch.int32)),
    ("dense", "draws", lambda: tensor(1)), ("dense", "drafted", lambda: tensor(3, t=torch.int64)),
    ("lists", "target_kept", lambda: None), ("lists", "draft_ids", lambda: tensor(3, 5, t=torch.int32)),
    ("lists", "target_ids", lambda: tensor(5, 8, t=torch.int32)[:, ::2]),
])
def test_tensors_that_do_not_fit_are_refused(no_drafts, call, name, other):
    f, tensors = calls()[call]
    with pytest.raises(ValueError):
        f(**dict(tensors, **{name: other()}))


def test_weights_that_do_not_fit_are_refused(no_library):  # noqa: F811
    with pytest.raises(ValueError):
        M.DeviceConv(torch.zeros(4, 3), bias=torch.zeros(3))
    for kw in (dict(skip=torch.zeros(5)), dict(dt_bias=torch.zeros(4, 1))):
        with pytest.raises(ValueError):
            M.DeviceScan(8, 1, torch.zeros(4, 8), **kw)


def test_the_statements_agree_with_other_forms():
    g = np.random.default_rng(0)
    x, w, bias = g.standard_normal((9, 5)), g.standard_normal((5, 4)), g.standard_normal(5)
    y, after, _ = S.conv(x, np.zeros((3, 5)), w, bias, "silu")
    t = torch.nn.functional.conv1d(torch.from_numpy(x.T)[None], torch.from_numpy(w)[:, None], torch.from_numpy(bias),
                                   padding=3, groups=5)[0, :, :9]
    assert np.allclose(torch.nn.functional.silu(t).numpy().T, y) and np.array_equal(after, x[-3:])
    a, b, _ = S.conv(x[:4], np.zeros((3, 5)), w, bias, "none")
    c, d, _ = S.conv(x[4:], b, w, bias, "none")
    assert np.allclose(np.concatenate([a, c]), S.conv(x, np.zeros((3, 5)), w, bias, "none")[0]) and np.array_equal(d, x[-3:])
    # The scan as one sum over the tokens before.
    dt, bb, cc = g.standard_normal((9, 4)), g.standard_normal((9, 2, 3)), g.standard_normal((9, 2, 3))
    x, a, skip, bias = g.standard_normal((9, 4)), -g.random((4, 3)), g.standard_normal(4), g.standard_normal(4)
    y, h, _, _ = S.scan(x, dt, bb, cc, None, a, skip, bias, np.zeros((4, 3)))
    s = np.log(1 + np.exp(dt + bias))
    for t in (0, 5, 8):
        want = skip * x[t]
        for j in range(t + 1):
            decay = np.exp(a * s[j + 1:t + 1].sum(0)[:, None])
            want = want + (np.repeat(cc[t] * bb[j], 2, 0) * decay).sum(-1) * s[j] * x[j]
        assert np.allclose(want, y[t])


def test_verified_tokens_are_distributed_as_the_targets():
    # The first token of a sequence with one draft from q, over a grid of uniforms: p, whatever q is.
    p, q = np.array([0.1, 0.5, 0.0, 0.4]), np.array([0.4, 0.3, 0.3, 0.0])
    ids, n = np.arange(4), 400
    u = (np.arange(n) + 0.5) / n
    share = np.zeros(4)
    for d in range(3):
        for x in u:
            accepted = x * q[d] < p[d]
            for draw in ((0.5,) if accepted else u):
                k, tokens = S.verify([(ids, p), (ids, p)], [(ids, q)], [d], [x], draw)
                assert k == int(accepted)
                share[tokens[0]] += q[d] / n / (1 if accepted else n)
    assert np.abs(share - p).max() <= 3.0 / n
