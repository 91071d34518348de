"""What the token mixers' binding accepts and refuses before the library is called:
every tensor has to be on the handle's device (a kernel would fault on another
address), and only strides that are used are looked at. No GPU: host tensors that
say where they are take the place of the device's."""
import ctypes

import pytest
import torch

import rl_mixers as M


class On0(torch.Tensor):
    """A tensor that says it is on device 0."""

    def get_device(self):
        return 0


class On1(torch.Tensor):
    def get_device(self):
        return 1


def tensor(*shape, t=torch.float32):
    return torch.zeros(*shape, dtype=t).as_subclass(On0)


def handle(cls, **fields):
    h = cls.__new__(cls)
    h.h, h.device = ctypes.c_void_p(), 0
    for name, x in fields.items():
        setattr(h, name, x)
    return h


def calls():
    """(a call of each method, its tensors by name)."""
    i32, i64 = torch.int32, torch.int64
    rotary = handle(M.DeviceRotary)
    cache = handle(M.DeviceCache)
    attention = handle(M.DeviceAttention, q_heads=2, scale=1.0)
    delta = handle(M.DeviceDelta, scale=1.0, state=(2, 16, 16))
    x = lambda: tensor(3, 2, 16)  # noqa: E731
    gates = lambda: tensor(3, 2)  # noqa: E731
    slots = lambda: tensor(3, t=i64)  # noqa: E731
    return {
        "rotary": (rotary.apply, dict(x=x(), positions=slots(), out=x(), second=x(), second_out=x())),
        "write": (lambda **kw: cache.write(rotary=rotary, **kw), dict(keys=x(), values=x(), slots=slots(), positions=slots())),
        "read": (cache.read, dict(slots=slots(), keys=x(), values=x())),
        "attention": (lambda **kw: attention.rows(cache, **kw),
                      dict(q=x(), out=x(), lens=tensor(2, t=i32), pages=tensor(2, 4, t=i32), starts=tensor(3, t=i32), lse=gates())),
        "delta": (delta.rows, dict(q=x(), k=x(), v=x(), g=gates(), beta=gates(), out=x(), states=tensor(4, 2, 16, 16),
                                   slots_in=tensor(2, t=i32), slots_out=tensor(2, t=i32), starts=tensor(3, t=i32))),
    }


class Reached(Exception):
    pass


class Library:
    def __getattr__(self, name):
        def call(*arguments):
            raise Reached
        return call


@pytest.fixture
def no_library(monkeypatch):
    monkeypatch.setattr(M, "lib", Library)
    # Without a GPU there is no current stream to ask for.
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: 0, raising=False)


@pytest.mark.parametrize("call", ["rotary", "write", "read", "attention", "delta"])
def test_every_tensor_has_to_be_on_the_handles_device(no_library, call):
    f, tensors = calls()[call]
    with pytest.raises(Reached):
        f(**tensors)
    for name, x in tensors.items():
        for other in (torch.zeros(x.shape, dtype=x.dtype), torch.zeros(x.shape, dtype=x.dtype).as_subclass(On1)):
            with pytest.raises(ValueError, match="device"):
                f(**dict(tensors, **{name: other}))
                pytest.fail("%s passed" % name)


def test_gates_of_one_head_have_any_head_stride(no_library):
    delta = handle(M.DeviceDelta, scale=1.0, state=(1, 16, 16))
    x, slots, starts = tensor(3, 1, 16), tensor(2, t=torch.int32), tensor(3, t=torch.int32)
    call = lambda g, beta: delta.rows(x, x, x, g, beta, x, tensor(4, 1, 16, 16), slots, slots, starts)  # noqa: E731
    turned = tensor(1, 3).t()  # [3][1] with strides (1, 3): a row a token, as the library reads it
    assert turned.stride() == (1, 3)
    with pytest.raises(Reached):
        call(turned, turned)
    delta.state = (2, 16, 16)
    x = tensor(3, 2, 16)
    with pytest.raises(ValueError, match="contiguous"):
        call(tensor(2, 3).t(), tensor(3, 2))
